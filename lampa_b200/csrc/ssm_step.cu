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
constexpr int ROWS = 64;              // state rows whose inputs are kept at a time

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

// Convolution of channel ch of row b; MOVE: the cache moves on too
template <int DT, bool MOVE>
__device__ __forceinline__ float conv_channel(const StepArgsS& a, int b, int ch, int channels) {
    const size_t at = ((size_t)b * channels + ch) * a.W;
    const float u = Elem<DT>::ld(a.u, (size_t)(b * a.u_row + ch));
    float acc = a.bias ? load_as_float(a.bias, ch, a.w_dt) : 0.f;
#pragma unroll
    for (int i = 0; i < MAX_W; ++i) {
        if (i >= a.W) break;
        const float v = i == a.W - 1 ? u : Elem<DT>::ld(a.cache, at + i + 1);
        if (MOVE) Elem<DT>::st(a.cache, at + i, v);
        acc = fmaf(v, load_as_float(a.w, (size_t)ch * a.W + i, a.w_dt), acc);
    }
    return a.silu ? acc / (1.f + expf(-acc)) : acc;
}

template <int DT, int VEC, int NV>    // NV vectors of VEC state elements per lane
__global__ void __launch_bounds__(THREADS) ssm_step_kernel(StepArgsS a) {
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

    float s[UNR][NV * VEC];
    auto load_rows = [&](int base, int end) {
#pragma unroll
        for (int k = 0; k < UNR; ++k)
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int r = base + k * rpw + sub, n = (l + lpr * v) * VEC;
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
    const int first = r_begin + warp * rpw * UNR;
    load_rows(first, min(r_end, r_begin + ROWS));

    for (int i = threadIdx.x; i < 2 * a.N; i += THREADS) {
        const bool c = i >= a.N;
        const int n = c ? i - a.N : i;
        const float v = conv_channel<DT, false>(a, b, a.H * a.P + (c ? a.G * a.N : 0) + grp * a.N + n, channels);
        (c ? sC : sB)[n] = v;
    }
    cluster_arrive();                                              // the caches of B and C have been read
    float Bv[NV * VEC], Cv[NV * VEC];
    for (int c0 = r_begin; c0 < r_end; c0 += ROWS) {
        const int c1 = min(r_end, c0 + ROWS);
        __syncthreads();
        for (int r = c0 + threadIdx.x; r < c1; r += THREADS) {
            const int h = grp * hpg + r / a.P, p = r % a.P;
            const float x = conv_channel<DT, true>(a, b, h * a.P + p, channels);
            float d = load_as_float(a.dt, (size_t)(b * a.dt_row + h), a.dt_dt) + (a.dt_bias ? a.dt_bias[h] : 0.f);
            if (a.softplus) d = fmaxf(d, 0.f) + log1pf(expf(-fabsf(d)));
            float gate = 1.f;
            if (a.z) {
                const float zv = Elem<DT>::ld(a.z, (size_t)(b * a.z_row + h * a.z_head + p));
                gate = zv / (1.f + expf(-zv));
            }
            sRow[r - c0] = make_float4(d * x, expf(d * a.A[h]), a.D ? a.D[h] * x : 0.f, gate);
        }
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
        for (int base = c0 + warp * rpw * UNR; base < c1; base += step) {
            if (base != first) load_rows(base, c1);
#pragma unroll
            for (int k = 0; k < UNR; ++k) {
                const int r = base + k * rpw + sub;
                const bool ok = r < c1;
                const float4 in = ok ? sRow[r - c0] : make_float4(0.f, 0.f, 0.f, 0.f);
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < NV * VEC; ++i) {
                    s[k][i] = fmaf(in.y, s[k][i], in.x * Bv[i]);
                    dot = fmaf(s[k][i], Cv[i], dot);
                }
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const int n = (l + lpr * v) * VEC;
                    if (!ok || n >= a.N) continue;
                    float* p = state + (size_t)r * a.N + n;
                    if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(s[k][4 * v], s[k][4 * v + 1], s[k][4 * v + 2], s[k][4 * v + 3]);
                    else *p = s[k][v];
                }
                for (int o = lpr >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                if (ok && l == 0) Elem<DT>::st(a.y, (size_t)b * a.H * a.P + (size_t)grp * total + r, (dot + in.z) * in.w);
            }
        }
    }
    cluster_wait();
    if (rank == 0)
        for (int i = threadIdx.x; i < 2 * a.N; i += THREADS)
            conv_channel<DT, true>(a, b, a.H * a.P + (i >= a.N ? a.G * a.N + i - a.N : i) + grp * a.N, channels);
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

template <int DT>
int launch_dt(const StepArgsS& a, int cs, int ctas, cudaStream_t st) {
    if (a.N % 4 || ((uintptr_t)a.state & 15)) return launch(ssm_step_kernel<DT, 1, 8>, a, cs, ctas, st);
    if (a.N <= 128) return launch(ssm_step_kernel<DT, 4, 1>, a, cs, ctas, st);
    return launch(ssm_step_kernel<DT, 4, 2>, a, cs, ctas, st);
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
    if (d->dtype == LAMPA_BF16) return launch_dt<LAMPA_BF16>(a, cs, ctas, st);
    if (d->dtype == LAMPA_F16) return launch_dt<LAMPA_F16>(a, cs, ctas, st);
    return launch_dt<LAMPA_F32>(a, cs, ctas, st);
}
