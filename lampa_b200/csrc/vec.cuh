// Vectors of row elements, 16 bytes or four elements, for the kernels that stream rows.
#pragma once
#include "common.cuh"

namespace lampa {

template <int DT> struct Vec16;     // 16 bytes of channels
template <> struct Vec16<LAMPA_F32> { static constexpr int N = 4; };
template <> struct Vec16<LAMPA_BF16> { static constexpr int N = 8; };
template <> struct Vec16<LAMPA_F16> { static constexpr int N = 8; };

template <int DT>
__device__ __forceinline__ void unpack_vec(const uint4& u, float (&x)[Vec16<DT>::N]) {
    if (DT == LAMPA_F32) {
        x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
    } else {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 f;
            if (DT == LAMPA_BF16) f = unpack_bf16x2(w[j]);
            else f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            x[2 * j] = f.x; x[2 * j + 1] = f.y;
        }
    }
}
template <int DT>
__device__ __forceinline__ void store_vec(void* p, size_t elem, const float (&x)[Vec16<DT>::N]) {
    uint4 u;
    if (DT == LAMPA_F32) {
        u = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    } else if (DT == LAMPA_BF16) {
        u = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    } else {
        __half2 h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
        u = *reinterpret_cast<const uint4*>(h);
    }
    *reinterpret_cast<uint4*>((char*)p + elem * (DT == LAMPA_F32 ? 4 : 2)) = u;
}

// Four channels of one token: 8 bytes of bf16 / fp16, 16 bytes of fp32.
template <int DT> struct Raw4 { using T = uint2; };
template <> struct Raw4<LAMPA_F32> { using T = uint4; };
template <int DT>
__device__ __forceinline__ typename Raw4<DT>::T ldg4(const void* p, size_t elem) {
    return __ldg(reinterpret_cast<const typename Raw4<DT>::T*>((const char*)p + elem * (DT == LAMPA_F32 ? 4 : 2)));
}
__device__ __forceinline__ void unpack4(const uint4& u, float (&x)[4], int) {
    x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack4(const uint2& u, float (&x)[4], int dt) {
    float2 a, b;
    if (dt == LAMPA_BF16) { a = unpack_bf16x2(u.x); b = unpack_bf16x2(u.y); }
    else { a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)); b = __half22float2(*reinterpret_cast<const __half2*>(&u.y)); }
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}
template <int DT>
__device__ __forceinline__ void store4(void* p, size_t elem, const float (&x)[4]) {
    if (DT == LAMPA_F32) {
        *reinterpret_cast<uint4*>((char*)p + elem * 4) =
            make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    } else if (DT == LAMPA_BF16) {
        *reinterpret_cast<uint2*>((char*)p + elem * 2) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    } else {
        const __half2 h0 = __floats2half2_rn(x[0], x[1]), h1 = __floats2half2_rn(x[2], x[3]);
        *reinterpret_cast<uint2*>((char*)p + elem * 2) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
    }
}

}  // namespace lampa
