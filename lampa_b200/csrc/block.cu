// Kernels around the mixer of a state space block: the short convolution of a prompt that continues from a cache, and the norms
// before and after the block with its gate, residual scale and residual.  Both stream their rows once and are bound by HBM;
// arithmetic is fp32 whatever the storage type.
#include "act.cuh"
#include "common.cuh"
#include "profile.cuh"
#include "vec.cuh"

#include <algorithm>

namespace lampa {
namespace {

bool dt_ok(int dt) { return dt >= LAMPA_BF16 && dt <= LAMPA_F32; }

// -------------------------------------------------------------------------------------------------
// y[t, d] = act(bias[d] + sum_i w[d, i] x[t - (W-1) + i, d]); what lies before a sequence's first token is its cache's last slots
// (zero without a cache).  cache[n, d, :] becomes the last W inputs of the sequence, those before it included.
// A thread takes VEC channels of RUN consecutive tokens with the window in registers.  The thread that has a sequence's first
// token has all tokens that look back into the cache (W - 1 at most, also where they lie in the next run) and, knowing all of x,
// writes the cache as well: nobody else touches these slots, so one launch suffices.
// -------------------------------------------------------------------------------------------------
constexpr int RUN = 16;               // tokens per thread, at least the largest W - 1

struct ConvArgsR {
    const void* x; const void* w; const void* bias; const int64_t* cu; void* cache; void* y; int32_t* status;
    int64_t n_tok, T, x_tok;
    int nseq, D, W, silu, w_dt, write;
};

template <int DT> struct Bits { using T = uint16_t; };
template <> struct Bits<LAMPA_F32> { using T = uint32_t; };

template <int DT, int VEC>
__device__ __forceinline__ void load_row(const void* x, int64_t at, float (&v)[VEC]) {
    if constexpr (VEC == 1) v[0] = Elem<DT>::ld(x, (size_t)at);
    else unpack_vec<DT>(__ldg(reinterpret_cast<const uint4*>((const typename Elem<DT>::T*)x + at)), v);
}

template <int DT, int VEC, int MW>    // MW: compile-time bound on the number of taps
__global__ void __launch_bounds__(128) conv_resume_kernel(ConvArgsR a) {
    if (chain_wait()) return;
    using E = typename Bits<DT>::T;
    if (a.cu && blockIdx.x == 0 && blockIdx.y == 0) check_offsets(a.cu, a.nseq, a.n_tok, a.status, 51);
    const int d0 = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    const int64_t t_begin = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * RUN;
    if (d0 >= a.D || t_begin >= a.n_tok) return;
    const int W = a.W;
    float wt[MW][VEC], bs[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        bs[j] = a.bias ? load_as_float(a.bias, d0 + j, a.w_dt) : 0.f;
#pragma unroll
        for (int i = 0; i < MW; ++i) wt[i][j] = i < W ? load_as_float(a.w, (size_t)(d0 + j) * W + i, a.w_dt) : 0.f;
    }
    int seq;                          // sequence of the first token; nseq: behind the last one
    int64_t bos, eos;
    auto bounds = [&]() {
        if (a.cu) {
            bos = a.cu[seq];
            eos = seq < a.nseq ? a.cu[seq + 1] : a.n_tok;
        } else {
            bos = (int64_t)seq * a.T;
            eos = bos + a.T;
        }
        return bos >= 0 && bos <= eos && eos <= a.n_tok;          // reported above
    };
    if (a.cu) {
        int hi = a.nseq + 1;
        seq = 0;
        while (hi - seq > 1) {
            const int mid = (seq + hi) >> 1;
            if (a.cu[mid] <= t_begin) seq = mid; else hi = mid;
        }
    } else {
        seq = (int)(t_begin / a.T);
    }
    if (!bounds() || t_begin < bos) return;
    float win[MW][VEC];               // win[i]: input W - 1 - i tokens back, i < W - 1
    const int64_t t_end = min(t_begin + RUN, a.n_tok);
    int64_t t_stop = t_end;
    // inputs before token t of this sequence; its first token opens it
    auto history = [&](int64_t t) {
        E* const slots = a.cache && seq < a.nseq ? (E*)a.cache + ((size_t)seq * a.D + d0) * W : nullptr;
#pragma unroll
        for (int i = 0; i < MW - 1; ++i)
            if (i < W - 1) {
                const int64_t tt = t - (W - 1) + i;
                if (tt >= bos) load_row<DT, VEC>(a.x, tt * a.x_tok + d0, win[i]);
                else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) win[i][j] = slots ? Elem<DT>::ld(slots, (size_t)j * W + W + (int)(tt - bos)) : 0.f;
                }
            }
        if (t != bos) return;
        t_stop = max(t_end, min(eos, bos + W - 1));                // those that look back into the cache are this thread's
        if (!slots || !a.write) return;
        const int64_t len = eos - bos;
        for (int w = 0; w < W; ++w) {                              // ascending: a slot that moves comes from further on
            const int64_t tt = len - W + w;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                slots[j * W + w] = tt >= 0 ? ((const E*)a.x)[(bos + tt) * a.x_tok + d0 + j] : slots[j * W + w + (int)len];
        }
    };
    // tokens that look back into the cache of a sequence of an earlier run are that run's
    const int64_t t_first = bos < t_begin ? max(t_begin, min(eos, bos + W - 1)) : t_begin;
    if (t_first < eos) history(t_first);
    constexpr int AHEAD = 8;          // rows that are asked for before the first of them is used
#pragma unroll 1
    for (int64_t t0 = t_first; t0 < t_stop; t0 += AHEAD) {
        float cur[AHEAD][VEC];
        uint4 raw[VEC > 1 ? AHEAD : 1];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int64_t at = min(t0 + k, a.n_tok - 1) * a.x_tok + d0;
            if constexpr (VEC > 1) raw[k] = __ldg(reinterpret_cast<const uint4*>((const typename Elem<DT>::T*)a.x + at));
            else cur[k][0] = Elem<DT>::ld(a.x, (size_t)at);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int64_t t = t0 + k;
            if (t >= t_stop) break;
            if constexpr (VEC > 1) unpack_vec<DT>(raw[k], cur[k]);
            if (t >= eos) {                                        // the next sequence that has tokens, or what lies behind the last
                do { ++seq; } while (seq < a.nseq && a.cu && a.cu[seq + 1] <= t);
                if (!bounds() || bos != t) return;
                history(t);
            }
            float out[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float acc = bs[j];
#pragma unroll
                for (int i = 0; i < MW - 1; ++i)
                    if (i < W - 1) acc = fmaf(win[i][j], wt[i][j], acc);
#pragma unroll
                for (int i = 0; i < MW; ++i)
                    if (i == W - 1) acc = fmaf(cur[k][j], wt[i][j], acc);
                if (a.silu) acc *= sigmoidf_(acc);
                out[j] = seq < a.nseq ? acc : 0.f;
            }
            if constexpr (VEC == 1) Elem<DT>::st(a.y, (size_t)t * a.D + d0, out[0]);
            else store_vec<DT>(a.y, (size_t)t * a.D + d0, out);
#pragma unroll
            for (int i = 0; i < MW - 1; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (i < W - 2) win[i][j] = win[i + 1 < MW ? i + 1 : i][j];
                    else if (i == W - 2) win[i][j] = cur[k][j];
        }
    }
}

template <int DT, int VEC>
int launch_conv(const ConvArgsR& a, cudaStream_t st) {
    const int groups = (a.D + VEC - 1) / VEC;
    int bx = 1;
    while (bx < groups && bx < 128) bx <<= 1;
    const dim3 block(bx, 128 / bx);
    const int64_t runs = (a.n_tok + RUN - 1) / RUN, gx = (runs + block.y - 1) / block.y;
    if (gx > INT32_MAX) return LAMPA_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)gx, (groups + bx - 1) / bx);
    if (grid.y > 65535) return LAMPA_ERR_UNSUPPORTED;
    const auto kernel = a.W <= 4 ? conv_resume_kernel<DT, VEC, 4> : conv_resume_kernel<DT, VEC, 8>;
    return launch_chained(kernel, grid, block, 0, st, a) == cudaSuccess ? LAMPA_OK : LAMPA_ERR_CUDA;
}

// -------------------------------------------------------------------------------------------------
// Norms around a block, on its fp32 residual stream:
//   n = delta rsqrt(mean(delta^2) + eps) post;   v = res + scale act(gate) n;   res = v;   y = v rsqrt(mean(v^2) + eps) pre.
// A row lies over TPR threads (lanes of a warp, or the whole CTA for wide rows) in vectors of VEC elements, VPT per thread, and stays
// in registers between its two sums.
// -------------------------------------------------------------------------------------------------
constexpr int NORM_THREADS = 256;

struct NormArgs {
    float* res; const void* delta; const void* gate; const float* post; const float* pre; const float* scale; const int64_t* cu;
    void* y; int32_t* status;
    int64_t rows, delta_row, gate_row;
    float scale1, eps;
    int D, nseq, delta_dt, gate_dt, y_dt, post_norm, act, lpr;
};

template <int VEC>
__device__ __forceinline__ void load_vec(const void* p, int64_t at, int dt, bool ok, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = ok ? load_as_float(p, (size_t)at, dt) : 0.f;
    } else if (!ok) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 0.f;
    } else if (dt == LAMPA_F32) {
#pragma unroll
        for (int q = 0; q < VEC / 4; ++q) {
            const float4 f = __ldg(reinterpret_cast<const float4*>((const float*)p + at) + q);
            v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
        }
    } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>((const uint16_t*)p + at));
        const uint32_t w[2] = {u.x, u.y};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const float2 f = dt == LAMPA_BF16 ? unpack_bf16x2(w[q]) : __half22float2(*reinterpret_cast<const __half2*>(&w[q]));
            v[2 * q] = f.x; v[2 * q + 1] = f.y;
        }
    }
}
template <int VEC>
__device__ __forceinline__ void put_vec(void* p, int64_t at, int dt, const float (&v)[VEC]) {
    if constexpr (VEC == 1) store_from_float(p, (size_t)at, v[0], dt);
    else if (dt == LAMPA_F32) *reinterpret_cast<float4*>((float*)p + at) = make_float4(v[0], v[1], v[2], v[3]);
    else if (dt == LAMPA_BF16) *reinterpret_cast<uint2*>((uint16_t*)p + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    else {
        const __half2 h0 = __floats2half2_rn(v[0], v[1]), h1 = __floats2half2_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>((uint16_t*)p + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
    }
}

// Sum over the threads of a row.  WIDE: the row's CTA, through one of two sets of words in turn (one barrier per sum).
template <bool WIDE>
__device__ __forceinline__ float row_sum(float v, int lpr, float (*words)[NORM_THREADS / 32], int& turn) {
    for (int o = (WIDE ? 32 : lpr) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (!WIDE) return v;
    float* const w = words[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) w[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NORM_THREADS / 32; ++i) v += w[i];
    return v;
}

template <int VEC, int VPT, bool WIDE>
__global__ void __launch_bounds__(NORM_THREADS) block_norm_kernel(NormArgs a) {
    if (chain_wait()) return;
    __shared__ float words[2][NORM_THREADS / 32];
    if (a.cu && blockIdx.x == 0) check_offsets(a.cu, a.nseq, a.rows, a.status, 52);
    int turn = 0;
    const int lpr = WIDE ? NORM_THREADS : a.lpr, rpc = NORM_THREADS / lpr;        // rows a CTA holds
    const int l = threadIdx.x % lpr;
    const int nvec = a.D / VEC;
    const float inv_d = 1.f / (float)a.D;
    for (int64_t base = (int64_t)blockIdx.x * rpc; base < a.rows; base += (int64_t)gridDim.x * rpc) {
        const int64_t row = base + threadIdx.x / lpr;
        const bool in = row < a.rows;
        int64_t grow = row;                                        // row of the gate, or -1: no sequence, no gate
        if (a.gate && a.cu && in) {
            int lo = 0, hi = a.nseq + 1;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.cu[mid] <= row) lo = mid; else hi = mid;
            }
            grow = lo < a.nseq && a.cu[lo] <= row && a.cu[lo + 1] > row ? lo : -1;
        }
        const bool add = a.delta && (!a.cu || !a.gate || grow >= 0);
        float r[VPT][VEC], d[VPT][VEC], g[VPT][VEC];
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = (l + lpr * v) * VEC;
            const bool ok = in && l + lpr * v < nvec;
            load_vec<VEC>(a.res, row * a.D + c, LAMPA_F32, ok, r[v]);
            if (a.delta) load_vec<VEC>(a.delta, row * a.delta_row + c, a.delta_dt, ok && add, d[v]);
            if (a.gate) load_vec<VEC>(a.gate, grow * a.gate_row + c, a.gate_dt, ok && add, g[v]);
        }
        if (a.delta) {
            float rstd = 1.f;
            if (a.post_norm) {
                float ss = 0.f;
#pragma unroll
                for (int v = 0; v < VPT; ++v)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ss = fmaf(d[v][j], d[v][j], ss);
                rstd = 1.f / sqrtf(row_sum<WIDE>(ss, lpr, words, turn) * inv_d + a.eps);
            }
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = (l + lpr * v) * VEC;
                const bool ok = l + lpr * v < nvec;
                float w[VEC], s[VEC];
                if (a.post) load_vec<VEC>(a.post, c, LAMPA_F32, ok, w);
                if (a.scale) load_vec<VEC>(a.scale, c, LAMPA_F32, ok, s);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float x = d[v][j] * rstd;
                    if (a.post) x *= w[j];
                    if (a.gate) {
                        const float gv = g[v][j];
                        x *= a.act == 0 ? gv : a.act == 1 ? sigmoidf_(gv) : gv * sigmoidf_(gv);
                    }
                    x *= a.scale ? s[j] : a.scale1;
                    if (add) r[v][j] += x;
                }
                if (ok && in && add) put_vec<VEC>(a.res, row * a.D + c, LAMPA_F32, r[v]);
            }
        }
        if (!a.y) continue;
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int j = 0; j < VEC; ++j) ss = fmaf(r[v][j], r[v][j], ss);
        const float rstd = 1.f / sqrtf(row_sum<WIDE>(ss, lpr, words, turn) * inv_d + a.eps);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = (l + lpr * v) * VEC;
            const bool ok = l + lpr * v < nvec;
            float w[VEC], out[VEC];
            if (a.pre) load_vec<VEC>(a.pre, c, LAMPA_F32, ok, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) out[j] = r[v][j] * rstd * (a.pre ? w[j] : 1.f);
            if (ok && in) put_vec<VEC>(a.y, row * a.D + c, a.y_dt, out);
        }
    }
}

template <int VEC>
int launch_norm(NormArgs a, cudaStream_t st) {
    const int nvec = a.D / VEC;
    const bool wide = nvec > 128;
    int lpr = 1;
    while (lpr < nvec && lpr < 32) lpr <<= 1;
    a.lpr = lpr;
    const int tpr = wide ? NORM_THREADS : lpr, vpt = (nvec + tpr - 1) / tpr, rpc = NORM_THREADS / tpr;
    const unsigned grid = (unsigned)std::min<int64_t>((a.rows + rpc - 1) / rpc, (int64_t)sm_count() * 16);
    void (*kernel)(NormArgs);
    if (wide) {
        if (vpt == 1) kernel = block_norm_kernel<VEC, 1, true>;
        else if (vpt == 2) kernel = block_norm_kernel<VEC, 2, true>;
        else if (vpt <= 4) kernel = block_norm_kernel<VEC, 4, true>;
        else if (vpt <= 8) kernel = block_norm_kernel<VEC, 8, true>;
        else if (VEC == 1 && vpt <= 32) kernel = block_norm_kernel<VEC, VEC == 1 ? 32 : 8, true>;
        else return LAMPA_ERR_UNSUPPORTED;
    } else {
        if (vpt == 1) kernel = block_norm_kernel<VEC, 1, false>;
        else if (vpt == 2) kernel = block_norm_kernel<VEC, 2, false>;
        else kernel = block_norm_kernel<VEC, 4, false>;
    }
    return launch_chained(kernel, dim3(grid), dim3(NORM_THREADS), 0, st, a) == cudaSuccess ? LAMPA_OK : LAMPA_ERR_CUDA;
}

}  // namespace
}  // namespace lampa

using namespace lampa;

extern "C" int lampa_short_conv_resume(const void* x, int64_t x_row, const void* weight, const void* bias, const int64_t* cu_seqlens,
                                       int32_t nseq, int64_t n_tok, int32_t D, int32_t W, int32_t dtype, int32_t w_dtype, int32_t silu,
                                       void* cache, int32_t write_cache, void* y, int32_t* status, void* stream) {
    if (nseq <= 0 || n_tok < 0 || D <= 0 || !dt_ok(dtype) || !dt_ok(w_dtype)) return LAMPA_ERR_ARG;
    if (W < 2 || W > 8) return LAMPA_ERR_UNSUPPORTED;
    if (n_tok == 0) return LAMPA_OK;
    if (!x || !weight || !y || (write_cache && !cache) || (!cu_seqlens && n_tok % nseq)) return LAMPA_ERR_ARG;
    const ConvArgsR a = {x, weight, bias, cu_seqlens, cache, y, status, n_tok, n_tok / nseq, x_row, nseq, D, W, silu, w_dtype, write_cache};
    cudaStream_t st = (cudaStream_t)stream;
    ProfScope prof("short_conv_resume", st);
    const int eb = dtype_bytes(dtype), nv = 16 / eb;
    const bool vec = D % nv == 0 && (x_row * eb) % 16 == 0 && (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    if (dtype == LAMPA_BF16) return vec ? launch_conv<LAMPA_BF16, 8>(a, st) : launch_conv<LAMPA_BF16, 1>(a, st);
    if (dtype == LAMPA_F16) return vec ? launch_conv<LAMPA_F16, 8>(a, st) : launch_conv<LAMPA_F16, 1>(a, st);
    return vec ? launch_conv<LAMPA_F32, 4>(a, st) : launch_conv<LAMPA_F32, 1>(a, st);
}

extern "C" int lampa_block_norm(float* res, const void* delta, int64_t delta_row, int32_t delta_dtype, const void* gate, int64_t gate_row,
                                int32_t gate_dtype, int32_t gate_act, const int64_t* cu_seqlens, int32_t nseq, int64_t rows, int32_t D,
                                const float* post_weight, int32_t post_norm, const float* scale, float scale_all, const float* pre_weight,
                                float eps, void* y, int32_t y_dtype, int32_t* status, void* stream) {
    if (rows < 0 || D <= 0 || gate_act < 0 || gate_act > 2 || (cu_seqlens && nseq <= 0)) return LAMPA_ERR_ARG;
    if (rows == 0) return LAMPA_OK;
    if (!res || (!delta && (!y || gate)) || (delta && !dt_ok(delta_dtype)) || (gate && !dt_ok(gate_dtype)) || (y && !dt_ok(y_dtype))) return LAMPA_ERR_ARG;
    const NormArgs a = {res, delta, gate, post_weight, pre_weight, scale, cu_seqlens, y, status, rows, delta_row, gate_row, scale_all, eps,
                        D, nseq, delta_dtype, gate_dtype, y_dtype, post_norm, gate_act, 0};
    cudaStream_t st = (cudaStream_t)stream;
    ProfScope prof("block_norm", st);
    auto rows_of_four = [](const void* p, int64_t row, int dt) {   // four elements at a time
        const uintptr_t m = dt == LAMPA_F32 ? 15 : 7;
        return !p || ((((uintptr_t)p) & m) == 0 && row % 4 == 0);
    };
    const bool vec = D % 4 == 0 && rows_of_four(res, D, LAMPA_F32) && rows_of_four(delta, delta_row, delta_dtype) &&
                     rows_of_four(gate, gate_row, gate_dtype) && rows_of_four(y, D, y_dtype) && rows_of_four(post_weight, 0, LAMPA_F32) &&
                     rows_of_four(pre_weight, 0, LAMPA_F32) && rows_of_four(scale, 0, LAMPA_F32);
    if (vec && D > 32 * NORM_THREADS) return LAMPA_ERR_UNSUPPORTED;
    if (!vec && D > 32 * NORM_THREADS) return LAMPA_ERR_UNSUPPORTED;
    return vec ? launch_norm<4>(a, st) : launch_norm<1>(a, st);
}
