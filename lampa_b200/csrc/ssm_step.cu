// One token per row through the short convolution and the selective recurrence, in place:
//   cache <- (cache[1:], u);  v = act(b + sum_w cache_w weight_w) = [x | B | C];
//   h <- exp(A d) h + d x B^T;   y = (h C + D x) silu(z).
//
// Bound by the state, which is read and written once (8 bytes per element in fp32; everything else is a few hundred bytes per
// state row of a head).  The CTAs of a cluster share the P x N states of one row's heads of one group; each finds the group's B and C
// for itself (2 N channels) and the x of its own state rows.  The caches of x have one owner; those of B and C are read by all, so that
// one CTA moves them on once everybody has passed the cluster's barrier.  A state row lies over up to 32 lanes, 16 bytes each, and the
// first rows of a warp are asked for before the convolution starts.
#include "act.cuh"
#include "common.cuh"
#include "profile.cuh"

#include <algorithm>

namespace lampa {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_W = 8;
constexpr int ROWS = THREADS;         // state rows whose inputs are kept at a time

struct StepArgsS {
    const void* u; const void* dt; void* cache; float* state;
    const void* w; const void* bias; const float* A; const float* D; const void* z; const float* dt_bias;
    void* y;
    int64_t u_row, dt_row, z_row, z_head;
    int H, P, N, G, W, dt_dt, w_dt, softplus, silu;
    int rows;                         // state rows of a CTA
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;\n" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctaid.x;\n" : "=r"(r)); return r; }

// The inputs of a channel's convolution (the cache's last W - 1 and the new one) and its weights.  All loads of a channel come before
// its stores; four taps of 16-bit types (T4) are one load each, and stay packed.
template <int DT, bool T4>
struct Channel {
    float v[MAX_W], w[MAX_W], b;
    __device__ __forceinline__ void load(const StepArgsS& a, int64_t row, int ch, int channels) {
        const size_t at = ((size_t)row * channels + ch) * a.W;
        b = a.bias ? load_as_float(a.bias, ch, a.w_dt) : 0.f;
        const float u = Elem<DT>::ld(a.u, (size_t)(row * a.u_row + ch));
#pragma unroll
        for (int i = 0; i < MAX_W; ++i)
            if (i < a.W) {
                v[i] = i == a.W - 1 ? u : Elem<DT>::ld(a.cache, at + i + 1);
                w[i] = load_as_float(a.w, (size_t)ch * a.W + i, a.w_dt);
            }
    }
    __device__ __forceinline__ float result(const StepArgsS& a) const {
        float acc = b;
#pragma unroll
        for (int i = 0; i < MAX_W; ++i)
            if (i < a.W) acc = fmaf(v[i], w[i], acc);
        return a.silu ? acc / (1.f + expf(-acc)) : acc;
    }
    __device__ __forceinline__ void move(const StepArgsS& a, int64_t row, int ch, int channels) const {
        const size_t at = ((size_t)row * channels + ch) * a.W;
#pragma unroll
        for (int i = 0; i < MAX_W; ++i)
            if (i < a.W) Elem<DT>::st(a.cache, at + i, v[i]);
    }
};
template <int DT>
struct Channel<DT, true> {
    uint2 c, k;                       // c: the cache as it was
    uint16_t u, b;
    // (no branch and no use of a loaded value in here, so that all loads of a thread are on their way at once)
    __device__ __forceinline__ void load(const StepArgsS& a, int64_t row, int ch, int channels) {
        c = reinterpret_cast<const uint2*>(a.cache)[(size_t)row * channels + ch];
        k = __ldg(reinterpret_cast<const uint2*>(a.w) + ch);
        b = __ldg((const uint16_t*)(a.bias ? a.bias : a.w) + ch);
        u = __ldg((const uint16_t*)a.u + row * a.u_row + ch);
    }
    __device__ __forceinline__ uint2 moved() const { return make_uint2(c.x >> 16 | c.y << 16, c.y >> 16 | (uint32_t)u << 16); }
    __device__ __forceinline__ static float2 pair(uint32_t x, bool bf) { return bf ? unpack_bf16x2(x) : __half22float2(*reinterpret_cast<const __half2*>(&x)); }
    __device__ __forceinline__ float result(const StepArgsS& a) const {
        const bool bf = a.w_dt == LAMPA_BF16;
        const uint2 m = moved();
        const float2 v0 = pair(m.x, DT == LAMPA_BF16), v1 = pair(m.y, DT == LAMPA_BF16), w0 = pair(k.x, bf), w1 = pair(k.y, bf);
        const float acc = fmaf(v1.y, w1.y, fmaf(v1.x, w1.x, fmaf(v0.y, w0.y, fmaf(v0.x, w0.x, a.bias ? pair(b, bf).x : 0.f))));
        return a.silu ? acc / (1.f + expf(-acc)) : acc;
    }
    __device__ __forceinline__ void move(const StepArgsS& a, int64_t row, int ch, int channels) const {
        reinterpret_cast<uint2*>(a.cache)[(size_t)row * channels + ch] = moved();
    }
};

// What a row's heads of one group need beside their states
template <int DT, bool T4>
struct StepInputs {
    const StepArgsS& a;
    int b, grp, total, channels;
    // a group's B (i < N) and C channels
    __device__ __forceinline__ int bc_channel(int i) const { return a.H * a.P + grp * a.N + (i < a.N ? i : a.G * a.N + i - a.N); }
    __device__ __forceinline__ void put_bc(int i, const Channel<DT, T4>& k, float* sB, float* sC) const { (i < a.N ? sB[i] : sC[i - a.N]) = k.result(a); }
    // a state row's x and what else its head has
    struct Row { Channel<DT, T4> x; uint32_t d, z; float bias, A, D; };
    __device__ __forceinline__ void load_x(int r, Row& k) const {
        const int h = grp * (a.H / a.G) + r / a.P, p = r % a.P;
        k.x.load(a, b, h * a.P + p, channels);
        const int64_t at = b * a.dt_row + h, az = a.z ? b * a.z_row + h * a.z_head + p : 0;
        k.d = a.dt_dt == LAMPA_F32 ? __ldg((const uint32_t*)a.dt + at) : __ldg((const uint16_t*)a.dt + at);
        k.z = DT == LAMPA_F32 ? __ldg((const uint32_t*)(a.z ? a.z : a.u) + az) : __ldg((const uint16_t*)(a.z ? a.z : a.u) + az);
        k.bias = __ldg((a.dt_bias ? a.dt_bias : a.A) + h);
        k.A = __ldg(a.A + h);
        k.D = __ldg((a.D ? a.D : a.A) + h);
    }
    __device__ __forceinline__ void put_x(int r, float4& to, const Row& k) const {
        k.x.move(a, b, grp * total + r, channels);
        const float x = k.x.result(a), z = Elem<DT>::ld(&k.z, 0);
        float d = load_as_float(&k.d, 0, a.dt_dt) + (a.dt_bias ? k.bias : 0.f);
        if (a.softplus) d = fmaxf(d, 0.f) + log1pf(expf(-fabsf(d)));
        to = make_float4(d * x, expf(d * k.A), a.D ? k.D * x : 0.f, a.z ? z / (1.f + expf(-z)) : 1.f);      // d x, exp(A d), D x, gate
    }
};

// What bounds it.  One stream: the launch and one chain of loads (4.5 us a call, among others).  64 streams, 16 heads of 64 x 128 (67 MB): 17.3 us,
// of which the rows alone take 13.9 (4.8 TB/s with the launch); the rest is the first loads' round trip, in all CTAs at once.  18.4 with the rows' loads in
// front of them, 26 with 102 registers (two CTAs to an SM), 21.6 with clusters of four; the rows through a ring of bulk copies: 17.7 - 29.
template <int DT, int VEC, int NV, bool T4>    // NV vectors of VEC state elements per lane
__global__ void __launch_bounds__(THREADS, T4 && VEC * NV == 4 ? 4 : 1) ssm_step_kernel(StepArgsS a) {
    constexpr int UNR = NV * VEC <= 4 ? 4 : 2;
    __shared__ __align__(16) float sB[256], sC[256];
    __shared__ float4 sRow[ROWS];     // d x, exp(A d), D x, gate
    if (chain_wait()) return;
    const uint32_t cs = cluster_size(), rank = cluster_rank();
    const int bg = blockIdx.x / cs, b = bg / a.G, grp = bg - b * a.G;
    const int hpg = a.H / a.G, total = hpg * a.P, channels = a.H * a.P + 2 * a.G * a.N;
    const int r_begin = min(total, (int)rank * a.rows), r_end = min(total, r_begin + a.rows);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int lpr = 1;                      // lanes to a state row
    while (lpr < 32 && lpr * VEC * NV < a.N) lpr <<= 1;
    const int rpw = 32 / lpr, sub = lane / lpr, l = lane % lpr;
    float* const state = a.state + ((size_t)b * a.H + grp * hpg) * a.P * a.N;

    float s[UNR][NV * VEC];           // rows of a warp in flight: as soon as one is done, the one a pass further on is asked for
    auto load_row = [&](int k, int r, int end) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int n = (l + lpr * v) * VEC;
            const bool ok = r < end && n < a.N;
            const float* p = state + (size_t)r * a.N + n;
            if constexpr (VEC == 4) {
                const float4 f = ok ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
                s[k][4 * v] = f.x; s[k][4 * v + 1] = f.y; s[k][4 * v + 2] = f.z; s[k][4 * v + 3] = f.w;
            } else {
                s[k][v] = ok ? *p : 0.f;
            }
        }
    };
    const int step = (THREADS / 32) * rpw * UNR;                   // rows of one pass of the CTA
    const StepInputs<DT, T4> in{a, b, grp, total, channels};
    Channel<DT, T4> bc;
    typename StepInputs<DT, T4>::Row own;
    const bool has_bc = threadIdx.x < 2 * a.N;
    bc.load(a, b, in.bc_channel(min((int)threadIdx.x, 2 * a.N - 1)), channels);
    in.load_x(min(r_begin + (int)threadIdx.x, total - 1), own);    // (ROWS is the number of threads)
#pragma unroll
    for (int k = 0; k < UNR; ++k) load_row(k, r_begin + (warp * UNR + k) * rpw + sub, min(r_end, r_begin + ROWS));
    if (has_bc) in.put_bc(threadIdx.x, bc, sB, sC);
    for (int i = threadIdx.x + THREADS; i < 2 * a.N; i += THREADS) {
        bc.load(a, b, in.bc_channel(i), channels);
        in.put_bc(i, bc, sB, sC);
    }
    cluster_arrive();                                              // the caches of B and C have been read
    cluster_wait();
    if (rank == 0)                                                 // everybody has read the caches of B and C: they move on
        for (int i = threadIdx.x; i < 2 * a.N; i += THREADS) {
            if (2 * a.N > THREADS) bc.load(a, b, in.bc_channel(i), channels);
            bc.move(a, b, in.bc_channel(i), channels);
        }
    float Bv[NV * VEC], Cv[NV * VEC];
    for (int c0 = r_begin; c0 < r_end; c0 += ROWS) {
        const int c1 = min(r_end, c0 + ROWS), r = c0 + threadIdx.x;
        if (c0 != r_begin) {
            __syncthreads();
            if (r < c1) in.load_x(r, own);
        }
        if (r < c1) in.put_x(r, sRow[threadIdx.x], own);
        __syncthreads();
        if (c0 == r_begin) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int n = (l + lpr * v) * VEC + e;
                    Bv[v * VEC + e] = n < a.N ? sB[n] : 0.f;
                    Cv[v * VEC + e] = n < a.N ? sC[n] : 0.f;
                }
        }
        const int base0 = c0 + warp * rpw * UNR + sub;
        if (c0 != r_begin)
#pragma unroll
            for (int k = 0; k < UNR; ++k) load_row(k, base0 + k * rpw, c1);
#pragma unroll 1
        for (int base = base0; base - sub < c1; base += step)
#pragma unroll
            for (int k = 0; k < UNR; ++k) {
                const int r = base + k * rpw;
                const bool ok = r < c1;
                const float4 row = ok ? sRow[r - c0] : make_float4(0.f, 0.f, 0.f, 0.f);
                float (&x)[NV * VEC] = s[k];
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < NV * VEC; ++i) {
                    x[i] = fmaf(row.y, x[i], row.x * Bv[i]);
                    dot = fmaf(x[i], Cv[i], dot);
                }
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const int n = (l + lpr * v) * VEC;
                    if (!ok || n >= a.N) continue;
                    float* p = state + (size_t)r * a.N + n;
                    if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(x[4 * v], x[4 * v + 1], x[4 * v + 2], x[4 * v + 3]);
                    else *p = x[v];
                }
                load_row(k, r + step, c1);
                for (int o = lpr >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                if (ok && l == 0) Elem<DT>::st(a.y, (size_t)b * a.H * a.P + (size_t)grp * total + r, (dot + row.z) * row.w);
            }
    }
}

template <typename K>
int launch(K kernel, const StepArgsS& a, int cs, int ctas, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[2];
    at[0] = chained_attribute();
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cs; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? LAMPA_OK : LAMPA_ERR_CUDA;
}

template <int DT, bool T4>
int launch_dt(const StepArgsS& a, int cs, int ctas, cudaStream_t st) {
    if (a.N % 4 || ((uintptr_t)a.state & 15)) return launch(ssm_step_kernel<DT, 1, 8, T4>, a, cs, ctas, st);
    if (a.N <= 128) return launch(ssm_step_kernel<DT, 4, 1, T4>, a, cs, ctas, st);
    return launch(ssm_step_kernel<DT, 4, 2, T4>, a, cs, ctas, st);
}

}  // namespace
}  // namespace lampa

using namespace lampa;

extern "C" int lampa_ssm_step(const lampa_ssm_desc* d, const void* xbc, int64_t xbc_row, const void* dt, int64_t dt_row, void* conv_cache,
                              const void* conv_weight, const void* conv_bias, int32_t taps, int32_t w_dtype, int32_t silu, const float* A,
                              const float* D, const void* z, int64_t z_row, int64_t z_head, const float* dt_bias, float* state, void* y,
                              void* stream) {
    if (!d || d->B < 0 || d->H <= 0 || d->P <= 0 || d->N <= 0 || d->G <= 0 || d->H % d->G) return LAMPA_ERR_ARG;
    if (d->dtype < LAMPA_BF16 || d->dtype > LAMPA_F32 || d->dt_dtype < LAMPA_BF16 || d->dt_dtype > LAMPA_F32 || w_dtype < LAMPA_BF16 || w_dtype > LAMPA_F32)
        return LAMPA_ERR_ARG;
    if (d->N > 256 || taps < 2 || taps > MAX_W) return LAMPA_ERR_UNSUPPORTED;
    if (d->B == 0) return LAMPA_OK;
    if (!xbc || !dt || !conv_cache || !conv_weight || !A || !state || !y) return LAMPA_ERR_ARG;
    // State rows per CTA: as few as a warp takes in one pass while the GPU has room for the CTAs, and no cluster above the portable 8
    const int64_t total = (int64_t)(d->H / d->G) * d->P, groups = (int64_t)d->B * d->G;
    if (total > (1 << 30) || groups * 8 > INT32_MAX) return LAMPA_ERR_UNSUPPORTED;
    int cs = 1;
    while (cs < 8 && total > 16 * cs) cs <<= 1;
    StepArgsS a = {xbc, dt, conv_cache, state, conv_weight, conv_bias, A, D, z, dt_bias, y, xbc_row, dt_row, z_row, z_head,
                   d->H, d->P, d->N, d->G, taps, d->dt_dtype, w_dtype, d->dt_softplus, silu, (int)((total + cs - 1) / cs)};
    cudaStream_t st = (cudaStream_t)stream;
    ProfScope prof("ssm_step", st);
    const int ctas = (int)groups * cs;
    const bool t4 = taps == 4 && w_dtype != LAMPA_F32 && (((uintptr_t)conv_cache | (uintptr_t)conv_weight) & 7) == 0;
    if (d->dtype == LAMPA_BF16) return t4 ? launch_dt<LAMPA_BF16, true>(a, cs, ctas, st) : launch_dt<LAMPA_BF16, false>(a, cs, ctas, st);
    if (d->dtype == LAMPA_F16) return t4 ? launch_dt<LAMPA_F16, true>(a, cs, ctas, st) : launch_dt<LAMPA_F16, false>(a, cs, ctas, st);
    return launch_dt<LAMPA_F32, false>(a, cs, ctas, st);
}
