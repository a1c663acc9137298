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
// A thread takes VEC channels of `run` consecutive tokens with the window in registers.  The thread that has a sequence's first
// token has all tokens that look back into the cache (W - 1 at most, also where they lie in the next run) and, knowing all of x,
// writes the cache as well: nobody else touches these slots, so one launch suffices.
// -------------------------------------------------------------------------------------------------
constexpr int RUN_MIN = 16;           // tokens per thread, at least the largest W - 1

struct ConvArgsR {
    const void* x; const void* w; const void* bias; const int64_t* cu; void* cache; void* y; int32_t* status;
    int64_t n_tok, T, x_tok;
    int nseq, D, W, silu, w_dt, write, groups, run;
};

__device__ __forceinline__ float exp2_approx(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }

template <int DT> struct Bits { using T = uint16_t; };
template <> struct Bits<LAMPA_F32> { using T = uint32_t; };

// A row's channels of a thread as they lie in memory: four, or one where rows do not allow it
template <int DT, int VEC> struct RawRow { using T = uint2; };
template <> struct RawRow<LAMPA_F32, 4> { using T = uint4; };
template <int DT> struct RawRow<DT, 1> { using T = typename Bits<DT>::T; };
template <int DT, int VEC>
__device__ __forceinline__ typename RawRow<DT, VEC>::T load_raw(const void* x, int64_t at) {
    return __ldg(reinterpret_cast<const typename RawRow<DT, VEC>::T*>((const typename Elem<DT>::T*)x + at));
}
template <int DT, int VEC>
__device__ __forceinline__ void to_float(const typename RawRow<DT, VEC>::T& raw, float (&v)[VEC]) {
    if constexpr (VEC == 1) v[0] = Elem<DT>::ld(&raw, 0);
    else unpack4(raw, v, DT);
}

// 61 440 x 1 280 in bf16 (315 MB): 69 us, 69 % of the measured bandwidth (SiLU alone takes the special function unit 36).  Eight channels to a
// thread: 129 us, one weight to a load: 211.
template <int DT, int VEC, int MW, bool EXACT>    // MW: compile-time bound on the number of taps; EXACT: it is their number, four, and weights are 16-bit
__global__ void __launch_bounds__(128) conv_resume_kernel(ConvArgsR a) {
    if (chain_wait()) return;
    if (a.cu && blockIdx.x == 0) check_offsets(a.cu, a.nseq, a.n_tok, a.status, 51);
    using E = typename Bits<DT>::T;
    using Raw = typename RawRow<DT, VEC>::T;
    const int64_t item = (int64_t)blockIdx.x * 128 + threadIdx.x, no = item / a.groups;
    const int d0 = (int)(item - no * a.groups) * VEC;
    const int64_t t_begin = no * a.run;
    if (t_begin >= a.n_tok) return;
    const int W = EXACT ? MW : a.W;
    const int64_t t_end = min(t_begin + a.run, a.n_tok);
    // Rows come in batches of four through a ring of this thread's own in shared memory (registers for three batches in flight would halve
    // the threads, and with one in flight the loads bound it: 84 us); single channels, which are too small to copy that way, through registers.
    constexpr int AHEAD = 4, RING = VEC > 1 ? 4 : 1;
    __shared__ Raw ring[RING][AHEAD][VEC > 1 ? 128 : 1];
    auto ask = [&](int slot, int64_t t0, int64_t end) {
        if constexpr (VEC > 1) {
            if (t0 < end)
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const void* src = (const typename Elem<DT>::T*)a.x + min(t0 + k, a.n_tok - 1) * a.x_tok + d0;
                    if constexpr (sizeof(Raw) == 16) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;\n" :: "r"(smem_u32(&ring[slot][k][threadIdx.x])), "l"(src) : "memory");
                    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" :: "r"(smem_u32(&ring[slot][k][threadIdx.x])), "l"(src) : "memory");
                }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        }
    };
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
    // tokens that look back into the cache of a sequence of an earlier run are that run's
    const int64_t t_first = bos < t_begin ? max(t_begin, min(eos, bos + W - 1)) : t_begin;
    // (a sequence that opens in the last batch may move the end by W - 1)
    const int64_t ask_end = t_end + W - 1;
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) ask(i, t_first + i * AHEAD, ask_end);

    float wt[MW][VEC], bs[VEC];
    if constexpr (EXACT && VEC == 4) {             // a thread's weights are 4 MW neighbours
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[4];
            unpack4(__ldg(reinterpret_cast<const uint2*>((const uint16_t*)a.w + (size_t)(d0 + j) * MW)), f, a.w_dt);
#pragma unroll
            for (int i = 0; i < 4; ++i) wt[i][j] = f[i];
            bs[j] = 0.f;
        }
        if (a.bias) unpack4(__ldg(reinterpret_cast<const uint2*>((const uint16_t*)a.bias + d0)), bs, a.w_dt);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            bs[j] = a.bias ? load_as_float(a.bias, d0 + j, a.w_dt) : 0.f;
#pragma unroll
            for (int i = 0; i < MW; ++i) wt[i][j] = i < W ? load_as_float(a.w, (size_t)(d0 + j) * W + i, a.w_dt) : 0.f;
        }
    }
    float win[MW][VEC];               // win[i]: input W - 1 - i tokens back, i < W - 1
    int64_t t_stop = t_end;
    // inputs before token t of this sequence; its first token opens it
    auto history = [&](int64_t t) {
        E* const slots = a.cache && seq < a.nseq ? (E*)a.cache + ((size_t)seq * a.D + d0) * W : nullptr;
#pragma unroll
        for (int i = 0; i < MW - 1; ++i)
            if (i < W - 1) {
                const int64_t tt = t - (W - 1) + i;
                if (tt >= bos) to_float<DT, VEC>(load_raw<DT, VEC>(a.x, tt * a.x_tok + d0), win[i]);
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
    if (t_first < eos) history(t_first);
    // output of the token whose row is `row`, and on with the window
    auto token = [&](const Raw& row, int64_t at, bool inside) {
        float cur[VEC], out[VEC];
        to_float<DT, VEC>(row, cur);
        if constexpr (VEC == 4) {                                  // two channels to an instruction
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                F2 acc = f2(bs[j], bs[j + 1]);
#pragma unroll
                for (int i = 0; i < MW - 1; ++i)
                    if (i < W - 1) acc = fma2(f2(win[i][j], win[i][j + 1]), f2(wt[i][j], wt[i][j + 1]), acc);
#pragma unroll
                for (int i = 0; i < MW; ++i)
                    if (i == W - 1) acc = fma2(f2(cur[j], cur[j + 1]), f2(wt[i][j], wt[i][j + 1]), acc);
                if (a.silu) {
                    float e0, e1;
                    f2_get(mul2(acc, f2(-1.4426950408889634f)), e0, e1);
                    f2_get(add2(f2(exp2_approx(e0), exp2_approx(e1)), f2(1.f)), e0, e1);
                    acc = mul2(acc, f2(rcp_approx(e0), rcp_approx(e1)));
                }
                f2_get(acc, out[j], out[j + 1]);
            }
        } else
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float acc = bs[j];
#pragma unroll
            for (int i = 0; i < MW - 1; ++i)
                if (i < W - 1) acc = fmaf(win[i][j], wt[i][j], acc);
#pragma unroll
            for (int i = 0; i < MW; ++i)
                if (i == W - 1) acc = fmaf(cur[j], wt[i][j], acc);
            out[j] = acc;
        }
        if (VEC == 1 && a.silu) out[0] *= sigmoid_fast(out[0]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = inside ? out[j] : 0.f;
        if constexpr (VEC == 1) Elem<DT>::st(a.y, (size_t)at, out[0]);
        else store4<DT>(a.y, (size_t)at, out);
#pragma unroll
        for (int i = 0; i < MW - 1; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (i < W - 2) win[i][j] = win[i + 1 < MW ? i + 1 : i][j];
                else if (i == W - 2) win[i][j] = cur[j];
    };
    int slot = 0;
#pragma unroll 1
    for (int64_t t0 = t_first; t0 < t_stop; t0 += AHEAD, slot = (slot + 1) % RING) {
        Raw raw[AHEAD];
        if constexpr (VEC > 1) {
            ask((slot + RING - 1) % RING, t0 + (RING - 1) * AHEAD, ask_end);
            asm volatile("cp.async.wait_group %0;\n" :: "n"(RING - 1) : "memory");
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) raw[k] = ring[slot][k][threadIdx.x];
        } else {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) raw[k] = load_raw<DT, VEC>(a.x, min(t0 + k, a.n_tok - 1) * a.x_tok + d0);
        }
        if (t0 + AHEAD <= min(eos, t_stop) && seq < a.nseq) {              // a whole batch of one sequence
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) token(raw[k], (t0 + k) * a.D + d0, true);
            continue;
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int64_t t = t0 + k;
            if (t >= t_stop) break;
            if (t >= eos) {                                        // the next sequence that has tokens, or what lies behind the last
                do { ++seq; } while (seq < a.nseq && a.cu && a.cu[seq + 1] <= t);
                if (!bounds() || bos != t) t_stop = t;             // (bad offsets: nothing more)
                if (t >= t_stop) break;
                history(t);
            }
            token(raw[k], t * a.D + d0, seq < a.nseq);
        }
    }
    if constexpr (VEC > 1) asm volatile("cp.async.wait_all;\n" ::: "memory");
}

template <int DT, int VEC>
int launch_conv(ConvArgsR a, bool vec_w, cudaStream_t st) {
    a.groups = (a.D + VEC - 1) / VEC;
    // 64 or 32 tokens where that leaves every SM a thousand threads (fewer weights and earlier rows to a token: 64 instead of 67 us with 64
    // instead of 32 for 61 440 x 1 280 in bf16), else 16 (7.7 instead of 9.6 us with 32 for 6 007 x 640)
    a.run = RUN_MIN;
    while (a.run < 64 && a.n_tok * a.groups / (2 * a.run) >= (int64_t)sm_count() * 1024) a.run *= 2;
    const int64_t runs = (a.n_tok + a.run - 1) / a.run, grid = (runs * a.groups + 127) / 128;
    if (grid > INT32_MAX) return LAMPA_ERR_UNSUPPORTED;
    auto kernel = conv_resume_kernel<DT, VEC, 8, false>;
    if (a.W == 4 && vec_w && VEC == 4) kernel = conv_resume_kernel<DT, VEC, 4, true>;
    else if (a.W <= 4) kernel = conv_resume_kernel<DT, VEC, 4, false>;
    return launch_chained(kernel, dim3((unsigned)grid), dim3(128), 0, st, a) == cudaSuccess ? LAMPA_OK : LAMPA_ERR_CUDA;
}

// -------------------------------------------------------------------------------------------------
// Norms around a block, on its fp32 residual stream:
//   n = delta rsqrt(mean(delta^2) + eps) post;   v = res + scale act(gate) n;   res = v;   y = v rsqrt(mean(v^2) + eps) pre.
// A row lies over some lanes of a warp, or over the whole CTA where it has more than 1 024 elements, in vectors of VEC elements, VPT
// per thread, and stays in registers between its two sums.  All of a row is asked for before the first use, its gate's sequence is
// looked up meanwhile.  61 440 x 1 024 with a CTA to a row and the types looked at load by load: 260 us.
// -------------------------------------------------------------------------------------------------
constexpr int NORM_THREADS = 256;

struct NormArgs {
    float* res; const void* delta; const void* gate; const float* post; const float* pre; const float* scale; const int64_t* cu;
    void* y; int32_t* status;
    int64_t rows, delta_row, gate_row;
    float scale1, eps;
    int D, nseq, delta_dt, gate_dt, y_dt, post_norm, act, lpr;
};

// VEC elements of a type (NONE: no such input) as they lie in memory, and as floats
constexpr int NONE = -1;
template <int VEC, int DT> struct RawV { uint32_t w[VEC == 1 || DT == NONE ? 1 : DT == LAMPA_F32 ? VEC : VEC / 2]; };
template <int VEC, int DT>
__device__ __forceinline__ void load_v(RawV<VEC, DT>& r, const char* p, bool ok) {
    if constexpr (DT == NONE) return;
    else if constexpr (VEC == 4 && DT == LAMPA_F32) {
        const uint4 u = ok ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
        r.w[0] = u.x; r.w[1] = u.y; r.w[2] = u.z; r.w[3] = u.w;
    } else if constexpr (VEC == 4) {
        const uint2 u = ok ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0u, 0u);
        r.w[0] = u.x; r.w[1] = u.y;
    } else if constexpr (DT == LAMPA_F32) r.w[0] = ok ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
    else r.w[0] = ok ? __ldg(reinterpret_cast<const uint16_t*>(p)) : (uint16_t)0;
}
template <int VEC, int DT>
__device__ __forceinline__ void floats(const RawV<VEC, DT>& r, float (&x)[VEC]) {
    if constexpr (DT == NONE) return;
    else if constexpr (DT == LAMPA_F32) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = __uint_as_float(r.w[j]);
    } else if constexpr (VEC == 1) x[0] = Elem<DT>::ld(r.w, 0);
    else {
#pragma unroll
        for (int q = 0; q < VEC / 2; ++q) {
            const float2 f = DT == LAMPA_BF16 ? make_float2(__uint_as_float(r.w[q] << 16), __uint_as_float(r.w[q] & 0xffff0000u))
                                              : __half22float2(*reinterpret_cast<const __half2*>(&r.w[q]));
            x[2 * q] = f.x; x[2 * q + 1] = f.y;
        }
    }
}
template <int VEC>
__device__ __forceinline__ void load_w(const float* p, int c, bool ok, float (&v)[VEC]) {
    if constexpr (VEC == 4) {
        const float4 f = ok ? __ldg(reinterpret_cast<const float4*>(p + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
        v[0] = ok ? __ldg(p + c) : 0.f;
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

template <int VEC, int VPT, bool WIDE, int DD, int GD>             // types of delta and gate
__global__ void __launch_bounds__(NORM_THREADS) block_norm_kernel(NormArgs a) {
    if (chain_wait()) return;
    constexpr int DB = DD == NONE ? 0 : DD == LAMPA_F32 ? 4 : 2, GB = GD == NONE ? 0 : GD == LAMPA_F32 ? 4 : 2;
    __shared__ float words[2][NORM_THREADS / 32];
    if (GB && a.cu && blockIdx.x == 0) check_offsets(a.cu, a.nseq, a.rows, a.status, 52);
    int turn = 0;
    const int lpr = WIDE ? NORM_THREADS : VPT > 1 ? 32 : a.lpr, rpc = NORM_THREADS / lpr;      // lanes to a row, rows a CTA holds
    const int l = threadIdx.x % lpr, c0 = l * VEC, cs = lpr * VEC; // vector v of this thread begins at column c0 + v cs
    const float inv_d = 1.f / (float)a.D;
    for (int64_t base = (int64_t)blockIdx.x * rpc; base < a.rows; base += (int64_t)gridDim.x * rpc) {
        const int64_t row = base + threadIdx.x / lpr;
        const int cols = row < a.rows ? a.D - c0 : 0;              // vector v is there if v cs < cols
        char* const pr = (char*)a.res + (row * a.D + c0) * 4;
        const char* const pd = (const char*)a.delta + (row * a.delta_row + c0) * DB;
        RawV<VEC, LAMPA_F32> rr[VPT];
        RawV<VEC, DD> dd[VPT];
        RawV<VEC, GD> gg[VPT];
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            load_v<VEC, LAMPA_F32>(rr[v], pr + (int64_t)v * cs * 4, v * cs < cols);
            load_v<VEC, DD>(dd[v], pd + (int64_t)v * cs * DB, v * cs < cols);
        }
        bool add = DB > 0;                                         // a row of no sequence has no gate: its residual stays
        if (GB) {
            int64_t grow = row;
            if (a.cu && cols > 0) {
                int lo = 0, hi = a.nseq + 1;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (__ldg(a.cu + mid) <= row) lo = mid; else hi = mid;
                }
                grow = lo;
                add = lo < a.nseq && __ldg(a.cu + lo) <= row && __ldg(a.cu + lo + 1) > row;
            }
            const char* const pg = (const char*)a.gate + (grow * a.gate_row + c0) * GB;
#pragma unroll
            for (int v = 0; v < VPT; ++v) load_v<VEC, GD>(gg[v], pg + (int64_t)v * cs * GB, add && v * cs < cols);
        }
        if (DB) {
            float rstd = 1.f;
            if (a.post_norm) {
                float ss = 0.f;
#pragma unroll
                for (int v = 0; v < VPT; ++v) {
                    float x[VEC];
                    floats<VEC, DD>(dd[v], x);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ss = fmaf(x[j], x[j], ss);
                }
                rstd = 1.f / sqrtf(row_sum<WIDE>(ss, lpr, words, turn) * inv_d + a.eps);
            }
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const bool ok = v * cs < cols;
                float x[VEC], w[VEC];
                floats<VEC, DD>(dd[v], x);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[j] *= rstd;
                if (a.post) {
                    load_w<VEC>(a.post, c0 + v * cs, ok, w);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) x[j] *= w[j];
                }
                if (GB) {
                    float g[VEC];
                    floats<VEC, GD>(gg[v], g);
                    if (a.act == 1) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) g[j] = sigmoidf_(g[j]);
                    } else if (a.act == 2) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) g[j] *= sigmoidf_(g[j]);
                    }
#pragma unroll
                    for (int j = 0; j < VEC; ++j) x[j] *= g[j];
                }
                if (a.scale) load_w<VEC>(a.scale, c0 + v * cs, ok, w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[j] = fmaf(x[j], a.scale ? w[j] : a.scale1, __uint_as_float(rr[v].w[j]));
                if (add) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) rr[v].w[j] = __float_as_uint(x[j]);
                    if (ok) put_vec<VEC>(pr + (int64_t)v * cs * 4, 0, LAMPA_F32, x);
                }
            }
        }
        if (!a.y) continue;
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int j = 0; j < VEC; ++j) ss = fmaf(__uint_as_float(rr[v].w[j]), __uint_as_float(rr[v].w[j]), ss);
        const float rstd = 1.f / sqrtf(row_sum<WIDE>(ss, lpr, words, turn) * inv_d + a.eps);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const bool ok = v * cs < cols;
            float w[VEC], out[VEC];
            if (a.pre) load_w<VEC>(a.pre, c0 + v * cs, ok, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) out[j] = __uint_as_float(rr[v].w[j]) * rstd * (a.pre ? w[j] : 1.f);
            if (ok) put_vec<VEC>(a.y, row * a.D + c0 + v * cs, a.y_dt, out);
        }
    }
}

template <int VEC, int DD, int GD>
int launch_norm(NormArgs a, cudaStream_t st) {
    const int nvec = a.D / VEC;
    const bool wide = nvec > 256;
    int lpr = 1;
    while (lpr < nvec && lpr < 32) lpr <<= 1;
    a.lpr = lpr;
    const int tpr = wide ? NORM_THREADS : lpr, vpt = (nvec + tpr - 1) / tpr, rpc = NORM_THREADS / tpr;
    const unsigned grid = (unsigned)std::min<int64_t>((a.rows + rpc - 1) / rpc, (int64_t)sm_count() * 16);
    void (*kernel)(NormArgs);
    if (wide) {
        if (vpt <= 2) kernel = block_norm_kernel<VEC, 2, true, DD, GD>;
        else if (vpt <= 8) kernel = block_norm_kernel<VEC, 8, true, DD, GD>;
        else kernel = block_norm_kernel<VEC, VEC == 1 ? 32 : 8, true, DD, GD>;
    } else {
        if (vpt == 1) kernel = block_norm_kernel<VEC, 1, false, DD, GD>;
        else if (vpt == 2) kernel = block_norm_kernel<VEC, 2, false, DD, GD>;
        else if (vpt <= 4) kernel = block_norm_kernel<VEC, 4, false, DD, GD>;
        else kernel = block_norm_kernel<VEC, 8, false, DD, GD>;
    }
    return launch_chained(kernel, dim3(grid), dim3(NORM_THREADS), 0, st, a) == cudaSuccess ? LAMPA_OK : LAMPA_ERR_CUDA;
}
template <int VEC, int DD>
int launch_norm_gate(const NormArgs& a, cudaStream_t st) {         // a gate is of delta's type or fp32
    if (!a.gate) return launch_norm<VEC, DD, NONE>(a, st);
    if (a.gate_dt == LAMPA_F32) return launch_norm<VEC, DD, LAMPA_F32>(a, st);
    return a.gate_dt == DD ? launch_norm<VEC, DD, DD>(a, st) : LAMPA_ERR_UNSUPPORTED;
}
template <int VEC>
int launch_norm_types(const NormArgs& a, cudaStream_t st) {
    if (!a.delta) return launch_norm<VEC, NONE, NONE>(a, st);
    if (a.delta_dt == LAMPA_BF16) return launch_norm_gate<VEC, LAMPA_BF16>(a, st);
    return a.delta_dt == LAMPA_F16 ? launch_norm_gate<VEC, LAMPA_F16>(a, st) : launch_norm_gate<VEC, LAMPA_F32>(a, st);
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
    const ConvArgsR a = {x, weight, bias, cu_seqlens, cache, y, status, n_tok, n_tok / nseq, x_row, nseq, D, W, silu, w_dtype, write_cache, 0, 0};
    cudaStream_t st = (cudaStream_t)stream;
    ProfScope prof("short_conv_resume", st);
    const int eb = dtype_bytes(dtype);
    const bool vec = D % 4 == 0 && x_row % 4 == 0 && (((uintptr_t)x | (uintptr_t)y) & (4 * eb - 1)) == 0;
    const bool vec_w = w_dtype != LAMPA_F32 && (((uintptr_t)weight | (uintptr_t)bias) & 7) == 0;
    if (dtype == LAMPA_BF16) return vec ? launch_conv<LAMPA_BF16, 4>(a, vec_w, st) : launch_conv<LAMPA_BF16, 1>(a, false, st);
    if (dtype == LAMPA_F16) return vec ? launch_conv<LAMPA_F16, 4>(a, vec_w, st) : launch_conv<LAMPA_F16, 1>(a, false, st);
    return vec ? launch_conv<LAMPA_F32, 4>(a, false, st) : launch_conv<LAMPA_F32, 1>(a, false, st);
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
    if (D > 32 * NORM_THREADS) return LAMPA_ERR_UNSUPPORTED;
    return vec ? launch_norm_types<4>(a, st) : launch_norm_types<1>(a, st);
}
