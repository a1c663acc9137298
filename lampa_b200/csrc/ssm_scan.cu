// Selective state space scan over whole sequences, mma.sync form: any head dims, bf16 and fp16.
//
// Inside a chunk of 64 tokens, with G_i the running sum of A d, the output is a masked matrix product,
//   y_i = sum_{j <= i} (C_i . B_j) e^{G_i - G_j} d_j x_j + e^{G_i} S C_i,        S <- e^{G_last} S + sum_j e^{G_last - G_j} d_j x_j B_j^T,
// so a CTA that walks through a block of chunks keeps one P x N state in registers (fp32) and reads every token once.  One sequence
// has few heads, so its tokens are cut into blocks as well: a first kernel finds what each block makes of an empty state, a second
// runs over the blocks, a third walks through the tokens again from the states that enter the blocks.
//
// Accuracy.  Operands of the tensor cores are bf16; fp16 inputs are taken as two bf16 pieces, exactly.  What a caller sees in 16
// bits (y) has one rounding of the scores, or of the state, to the input's precision before its own.  States are seen in fp32: their
// updates take d x e^{..} in three bf16 pieces (24 bits), and chunk sums are added in fp32 arithmetic.
//
// A token whose x is not finite must not reach the rows in front of it through a zero of the mask (0 * NaN): such elements are taken
// out of the tile, and from their row on the column is NaN, as the recurrence has it.
//
// What bounds it: instructions (24 001 packed tokens in fp16, 6 heads of 32 x 16, 58 us in all; between events output 35 us, issue slots 45 %, tensor
// pipe 12 %, DRAM 0.7 TB/s; states 21, pass 15), most of them spent on splitting fp16 into pieces and on the gate, in four warps a CTA whose phases
// follow one another.  With an exponential for every pair of tokens 61 us, with tiles and steps loaded just before their use 107, with the weighted
// pieces made from the tile in shared memory 68.  61 440 bf16 tokens, 16 heads of 64 x 128, take 895 us here and 215 in the tcgen05 form (one call after
// another on the same inputs).
#include "profile.cuh"
#include "ssm.cuh"

#include <algorithm>

namespace lampa {
namespace {

constexpr int Q = SSM_Q;
constexpr int THREADS = 128;

template <int DT, int NP, int PT>
struct Sm {
    static constexpr int XP = DT == LAMPA_F16 ? 2 : 1;                 // bf16 pieces of an input
    static constexpr int LN = NP + 8, LP = PT + 8;                     // row pitches: 16 bytes more than a power of two
    static constexpr int STATE_BYTES = XP * Q * LN * 2 + 3 * Q * LP * 2 + 2 * Q * 4 + 2 * 4 * 4;     // up to and without C: all that ssm_state_kernel uses
    __nv_bfloat16 B[XP][Q * LN];
    __nv_bfloat16 wx[3][Q * LP];                                       // d x e^{G_last - G}
    float w[2][Q], sum[2][4];                                          // by chunk parity; sums of A d of 16 tokens each
    // (the output's alone)
    __nv_bfloat16 C[XP][Q * LN];
    __nv_bfloat16 S[XP][PT * LN];                                      // state as the right operand of C S^T
    __nv_bfloat16 x[XP][Q * LP];
    SsmExp G[2][Q];                                                    // sums of A d from the first of the token's 16 on
    float d[2][Q], cf[2][Q];                                           // cf = d e^{what follows in the token's 16}
    int bad[PT], any_bad;                                              // first row of the column that is not finite, or Q; whether there is one
};

// Rows [0, n) of a matrix of 16-bit elements as COLS-wide tile pieces of 16 bytes in a thread's registers, zero beyond n rows and `cols`
// columns: asked for a chunk ahead where that takes few registers (tiles up to 64 wide), just before use otherwise.
template <int COLS> struct Piece { static constexpr int N = Q * (COLS / 8) / THREADS; };
template <int DT, int COLS>
__device__ __forceinline__ void fetch(uint4 (&u)[Piece<COLS>::N], const void* base, int64_t off, int64_t pitch, int n, int cols, bool vec) {
    const uint16_t* src = (const uint16_t*)base + off;
#pragma unroll
    for (int k = 0; k < Piece<COLS>::N; ++k) {
        const int i = threadIdx.x + THREADS * k, r = i / (COLS / 8), c = (i % (COLS / 8)) * 8;
        u[k] = make_uint4(0u, 0u, 0u, 0u);
        if (r >= n || c >= cols) continue;
        const uint16_t* p = src + (int64_t)r * pitch + c;
        if (vec) u[k] = __ldg(reinterpret_cast<const uint4*>(p));      // cols is a multiple of 8 then
        else {
            uint32_t e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = c + j < cols ? __ldg(p + j) : (uint16_t)0;
            u[k] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
    }
}
// Two 16-bit values as floats
template <int DT>
__device__ __forceinline__ float2 pair_of(uint32_t w) { return DT == LAMPA_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&w)) : unpack_bf16x2(w); }
// ... into XP bf16 pieces.
template <int DT, int XP, int COLS>
__device__ __forceinline__ void put(__nv_bfloat16* dst, int piece, int ld, const uint4 (&u)[Piece<COLS>::N]) {
#pragma unroll
    for (int k = 0; k < Piece<COLS>::N; ++k) {
        const int i = threadIdx.x + THREADS * k, at = i / (COLS / 8) * ld + (i % (COLS / 8)) * 8;
        if (XP == 1) {                                                 // bf16 as it is
            *reinterpret_cast<uint4*>(dst + at) = u[k];
            continue;
        }
        const uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = pair_of<DT>(w[j]);
            hi[j] = pack_bf16x2(f.x, f.y);
            const float2 h = unpack_bf16x2(hi[j]);
            lo[j] = pack_bf16x2(f.x - h.x, f.y - h.y);
        }
        *reinterpret_cast<uint4*>(dst + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(dst + piece + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}
// x: as it is (KEEP; elements that are not finite become zero there and leave their row in bad[]), and as `pieces` pieces of w x
template <int DT, int NP, int PT, bool KEEP>
__device__ __forceinline__ void put_x(Sm<DT, NP, PT>& s, int buf, uint4 (&u)[Piece<PT>::N], int pieces) {
    using S = Sm<DT, NP, PT>;
    constexpr uint32_t EXP = DT == LAMPA_F16 ? 0x7c007c00u : 0x7f807f80u, ONE = DT == LAMPA_F16 ? 0x04000400u : 0x00800080u;
#pragma unroll
    for (int k = 0; k < Piece<PT>::N; ++k) {
        const int i = threadIdx.x + THREADS * k, r = i / (PT / 8), c = (i % (PT / 8)) * 8, at = r * S::LP + c;
        uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
        const float wr = s.w[buf][r];
        float2 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = pair_of<DT>(w[j]);
            v[j].x *= wr; v[j].y *= wr;
        }
        if (KEEP && ((((w[0] & EXP) + ONE) | ((w[1] & EXP) + ONE) | ((w[2] & EXP) + ONE) | ((w[3] & EXP) + ONE)) & 0x80008000u)) {
            s.any_bad = 1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if ((((w[j] & EXP) + ONE) & 0x8000u)) { atomicMin(&s.bad[c + 2 * j], r); w[j] &= 0xffff0000u; }
                if ((((w[j] & EXP) + ONE) & 0x80000000u)) { atomicMin(&s.bad[c + 2 * j + 1], r); w[j] &= 0xffffu; }
            }
            u[k] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        for (int p = 0; p < pieces; ++p) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = pack_bf16x2(v[j].x, v[j].y);
                const float2 h = unpack_bf16x2(o[j]);
                v[j].x -= h.x; v[j].y -= h.y;
            }
            *reinterpret_cast<uint4*>(&s.wx[p][at]) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    if (KEEP) put<DT, S::XP, PT>(s.x[0], Q * S::LP, S::LP, u);
}

// d and w = d e^{G_last - G} of a chunk's n tokens (tokens beyond them have d = 0), and FULL: what the decays between two of them are made
// from, by the first warp, two tokens to a lane: raw steps a chunk ahead, the rest while the other warps, which have more scores to work on,
// are busy.  Every exponent is a sum of what lies between its two tokens, or exact but for its rest (SsmExp), so that its error is one of its own size, not of G's.
__device__ __forceinline__ void raw_steps(const SsmArgs& a, int64_t t0, int n, int h, float (&raw)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = 2 * (threadIdx.x & 31) + k;
        raw[k] = i < n ? load_as_float(a.dt, (size_t)((t0 + i) * a.dt_tok + h), a.dt_dt) : 0.f;
    }
}
template <bool FULL, typename SM>
__device__ __forceinline__ void chunk_steps(const SsmArgs& a, SM& s, int buf, const float (&raw)[2], int n, float A, float bias) {
    const int l = threadIdx.x & 31;
    float d[2], g[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        d[k] = 2 * l + k < n ? ssm_step_size(raw[k] + bias, a.softplus) : 0.f;
        g[k] = 2 * l + k < n ? d[k] * A : 0.f;
    }
    float down = g[0] + g[1];                      // to the end of its 16 tokens, which eight lanes hold
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const float v = __shfl_down_sync(0xffffffffu, down, o, 8);
        if ((l & 7) + o < 8) down += v;
    }
    const float next = __shfl_down_sync(0xffffffffu, down, 1, 8), after = (l & 7) < 7 ? next : 0.f;
    float sum[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) sum[b] = __shfl_sync(0xffffffffu, down, 8 * b);
    float e = 0.f;                                 // of the 16-token blocks behind this one
#pragma unroll
    for (int b = 3; b > 0; --b) e += l < 8 * b ? sum[b] : 0.f;
    e += after;
    s.w[buf][2 * l] = d[0] * expf(e + g[1]);
    s.w[buf][2 * l + 1] = d[1] * expf(e);
    if (l < 4) s.sum[buf][l] = l < 2 ? l == 0 ? sum[0] : sum[1] : l == 2 ? sum[2] : sum[3];
    if constexpr (FULL) {
        const SsmExp g0 = ssm_split(g[0]), g1 = ssm_split(g[1]);
        SsmExp up = {g0.whole + g1.whole, g0.rest + g1.rest};
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            const float u = __shfl_up_sync(0xffffffffu, up.whole, o, 8), r = __shfl_up_sync(0xffffffffu, up.rest, o, 8);
            if ((l & 7) >= o) { up.whole += u; up.rest += r; }
        }
        const float bw = __shfl_up_sync(0xffffffffu, up.whole, 1, 8), br = __shfl_up_sync(0xffffffffu, up.rest, 1, 8);
        s.G[buf][2 * l] = {((l & 7) ? bw : 0.f) + g0.whole, ((l & 7) ? br : 0.f) + g0.rest};
        s.G[buf][2 * l + 1] = up;
        s.d[buf][2 * l] = d[0]; s.d[buf][2 * l + 1] = d[1];
        s.cf[buf][2 * l] = d[0] * __expf(after + g[1]);
        s.cf[buf][2 * l + 1] = d[1] * __expf(after);
    }
}
template <typename SM>
__device__ __forceinline__ float chunk_sum(const SM& s, int buf) { return (s.sum[buf][0] + s.sum[buf][1]) + (s.sum[buf][2] + s.sum[buf][3]); }

// The state of a CTA: PT x NP, warp w holds rows 16 (w % RS) .. +15 and columns of 16 (cg + CG i)
template <int NP, int PT>
struct StateMap {
    static constexpr int RS = PT / 16, CG = 4 / RS;
    static constexpr int CT = NP / 16 >= CG ? NP / 16 / CG : 1;
};

// S <- dec S + sum_j wx_j B_j^T.  Every chunk sum starts from zero and is added in fp32 arithmetic (an MMA that accumulates onto a
// long sum rounds it towards zero each time); smallest pieces first.
template <int DT, int NP, int PT>
__device__ __forceinline__ void update_state(float (&st)[StateMap<NP, PT>::CT][2][4], const Sm<DT, NP, PT>& s, float dec, int pieces) {
    using M = StateMap<NP, PT>;
    using S = Sm<DT, NP, PT>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, p0 = 16 * (warp % M::RS), cg = warp / M::RS;
#pragma unroll
    for (int i = 0; i < M::CT; ++i) {
        const int n0 = 16 * (cg + M::CG * i);
        if (n0 >= NP) continue;
        float c[2][4] = {};
#pragma unroll 1
        for (int p = pieces - 1; p >= 0; --p)
#pragma unroll
            for (int bp = S::XP - 1; bp >= 0; --bp)
#pragma unroll
                for (int k = 0; k < Q; k += 16) {
                    uint32_t av[4], bv[4];
                    load_a_t(av, s.wx[p], S::LP, p0, k, lane);
                    load_b_t(bv, s.B[bp], S::LN, n0, k, lane);
                    mma16816(c[0], av, bv[0], bv[1]);
                    mma16816(c[1], av, bv[2], bv[3]);
                }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q) st[i][t][q] = fmaf(dec, st[i][t][q], c[t][q]);
    }
}

// f(p, n, value) over the state elements of this thread
template <int NP, int PT, typename F>
__device__ __forceinline__ void each_state(float (&st)[StateMap<NP, PT>::CT][2][4], F f) {
    using M = StateMap<NP, PT>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, p0 = 16 * (warp % M::RS), cg = warp / M::RS;
#pragma unroll
    for (int i = 0; i < M::CT; ++i) {
        const int n0 = 16 * (cg + M::CG * i);
        if (n0 >= NP) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q) f(p0 + (lane >> 2) + 8 * (q >> 1), n0 + 8 * t + 2 * (lane & 3) + (q & 1), st[i][t][q]);
    }
}

// What every block makes of an empty state.  A block that is its whole sequence needs no such state.
template <int DT, int NP, int PT>
__global__ void __launch_bounds__(THREADS) ssm_state_kernel(SsmArgs a) {
    if (chain_wait()) return;
    extern __shared__ __align__(16) char smem[];
    Sm<DT, NP, PT>& s = *reinterpret_cast<Sm<DT, NP, PT>*>(smem);
    SsmUnit u;
    const int h = blockIdx.y, p0 = blockIdx.z * PT;
    if (!ssm_unit(a, blockIdx.x, u) || u.outside || u.single(a.bl)) return;
    using SMT = Sm<DT, NP, PT>;
    constexpr bool AHEAD = NP <= 128;
    const int grp = h / (a.H / a.G);
    const float A = a.A[h], bias = a.dt_bias ? a.dt_bias[h] : 0.f;
    float st[StateMap<NP, PT>::CT][2][4] = {};
    float log_dec = 0.f, raw[2];
    uint4 ub[Piece<NP>::N], ux[Piece<PT>::N];
    auto tokens = [&](int64_t t) { return (int)max((int64_t)0, min((int64_t)Q, u.t1 - t)); };
    auto ask = [&](int64_t t) {
        fetch<DT, NP>(ub, a.B, t * a.b_tok + grp * a.b_grp, a.b_tok, tokens(t), a.N, a.vec);
        fetch<DT, PT>(ux, a.x, t * a.x_tok + h * a.x_head + p0, a.x_tok, tokens(t), a.P - p0, a.vec);
    };
    if (threadIdx.x < 32) raw_steps(a, u.t0, tokens(u.t0), h, raw);
    if (AHEAD) ask(u.t0);
    if (threadIdx.x < 32) {
        chunk_steps<false>(a, s, 0, raw, tokens(u.t0), A, bias);
        raw_steps(a, u.t0 + Q, tokens(u.t0 + Q), h, raw);
    }
    int buf = 0;
    for (int64_t t = u.t0; t < u.t1; t += Q, buf ^= 1) {
        if (!AHEAD) ask(t);
        __syncthreads();
        put<DT, SMT::XP, NP>(s.B[0], Q * SMT::LN, SMT::LN, ub);
        put_x<DT, NP, PT, false>(s, buf, ux, 3);
        __syncthreads();
        if (AHEAD) ask(t + Q);
        if (threadIdx.x < 32) {
            chunk_steps<false>(a, s, buf ^ 1, raw, tokens(t + Q), A, bias);
            raw_steps(a, t + 2 * Q, tokens(t + 2 * Q), h, raw);
        }
        const float g = chunk_sum(s, buf);
        update_state(st, s, expf(g), 3);
        log_dec += g;
    }
    float* out = a.blk + (u.slot * a.H + h) * a.P * a.N;
    each_state<NP, PT>(st, [&](int p, int n, float v) {
        if (p0 + p < a.P && n < a.N) out[(int64_t)(p0 + p) * a.N + n] = v;
    });
    if (threadIdx.x == 0 && blockIdx.z == 0) a.blk_dec[u.slot * a.H + h] = log_dec;
}

// Over the blocks of a sequence: what enters each of them takes the place of what it makes of an empty state.  Also the final state,
// but for sequences of one block, whose only CTA writes it (in the output pass, or the block kernel of the tcgen05 form).  V state elements to a thread, AHEAD blocks asked for before the first is used
// (one by one: 27 us instead of 5 for 18 blocks of 16 heads of 64 x 128).
template <int V, int AHEAD>
__global__ void __launch_bounds__(256) ssm_pass_kernel(SsmArgs a) {
    if (chain_wait()) return;
    struct alignas(4 * V) Vec { float v[V]; };
    const int pn = a.P * a.N, slabs = (pn / V + 255) / 256, seq = blockIdx.x / slabs, h = blockIdx.y;
    const int e = ((blockIdx.x - seq * slabs) * 256 + threadIdx.x) * V;
    int64_t bos = (int64_t)seq * a.T, eos = bos + a.T, u0 = (int64_t)seq * a.nb;
    if (a.cu) {
        if (a.n_tok == 0 && blockIdx.x == 0 && blockIdx.y == 0) check_offsets(a.cu, a.nseq, 0, a.status, 50);      // (there is no output kernel)
        bos = a.cu[seq]; eos = a.cu[seq + 1];
        if (bos < 0 || eos < bos || eos > a.n_tok) return;         // reported by the output kernel
        u0 = ssm_block_of(a, bos, a.bl / 2);
    }
    if (e >= pn) return;
    const int64_t len = eos - bos, out = ((int64_t)seq * a.H + h) * pn + e;
    Vec s = {};
    if (a.h0) s = *reinterpret_cast<const Vec*>(a.h0 + out);
    if (len > a.bl) {
        const int nb = (int)((len + a.bl - 1) / a.bl);
        float* p = a.blk + (u0 * a.H + h) * pn + e;
        const float* dec = a.blk_dec + u0 * a.H + h;
        const int64_t step = (int64_t)a.H * pn;
        for (int b = 0; b < nb; b += AHEAD) {
            Vec part[AHEAD];
            float d[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                if (b + k < nb) {
                    part[k] = *reinterpret_cast<const Vec*>(p + (b + k) * step);
                    d[k] = dec[(int64_t)(b + k) * a.H];
                }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                if (b + k < nb) {
                    *reinterpret_cast<Vec*>(p + (b + k) * step) = s;
                    const float x = expf(d[k]);
#pragma unroll
                    for (int i = 0; i < V; ++i) s.v[i] = fmaf(x, s.v[i], part[k].v[i]);
                }
        }
    } else if (len > 0) return;
    if (a.ht) *reinterpret_cast<Vec*>(a.ht + out) = s;
}

template <int DT, int NP, int PT>
__global__ void __launch_bounds__(THREADS, NP * PT <= 512 && (DT == LAMPA_BF16 || NP == 16) ? 4 : 0) ssm_out_kernel(SsmArgs a) {     // (four: 128 registers, where that spills nothing)
    using SMT = Sm<DT, NP, PT>;
    constexpr int XP = SMT::XP, LN = SMT::LN, LP = SMT::LP;
    if (chain_wait()) return;
    extern __shared__ __align__(16) char smem[];
    SMT& s = *reinterpret_cast<SMT*>(smem);
    SsmUnit u;
    const int h = blockIdx.y, p0 = blockIdx.z * PT, grp = h / (a.H / a.G);
    if (a.cu && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_offsets(a.cu, a.nseq, a.n_tok, a.status, 50);
    if (!ssm_unit(a, blockIdx.x, u)) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t2 = 2 * (lane & 3);
    if (u.outside) {                                               // rows of no sequence read as zero
        for (int64_t i = threadIdx.x; i < (u.t1 - u.t0) * PT; i += THREADS) {
            const int p = p0 + (int)(i % PT);
            if (p < a.P) Elem<DT>::st(a.y, (size_t)(((u.t0 + i / PT) * a.H + h) * a.P + p), 0.f);
        }
        return;
    }
    const bool single = u.single(a.bl);
    const int pieces = single && a.ht ? 3 : XP;
    const int64_t pn = (int64_t)a.P * a.N;
    const float* enter = single ? (a.h0 ? a.h0 + ((int64_t)u.seq * a.H + h) * pn : nullptr) : a.blk + (u.slot * a.H + h) * pn;
    constexpr bool AHEAD = NP <= 64;
    const float Dh = a.D ? a.D[h] : 0.f, A = a.A[h], bias = a.dt_bias ? a.dt_bias[h] : 0.f;
    for (int i = threadIdx.x; i < PT; i += THREADS) s.bad[i] = Q;
    if (threadIdx.x == 0) s.any_bad = 0;
    float raw[2];
    uint4 ub[Piece<NP>::N], uc[Piece<NP>::N], ux[Piece<PT>::N];
    auto tokens = [&](int64_t t) { return (int)max((int64_t)0, min((int64_t)Q, u.t1 - t)); };
    auto ask = [&](int64_t t) {
        fetch<DT, NP>(ub, a.B, t * a.b_tok + grp * a.b_grp, a.b_tok, tokens(t), a.N, a.vec);
        fetch<DT, NP>(uc, a.C, t * a.c_tok + grp * a.c_grp, a.c_tok, tokens(t), a.N, a.vec);
        fetch<DT, PT>(ux, a.x, t * a.x_tok + h * a.x_head + p0, a.x_tok, tokens(t), a.P - p0, a.vec);
    };
    if (warp == 0) raw_steps(a, u.t0, tokens(u.t0), h, raw);
    if (AHEAD) ask(u.t0);
    float st[StateMap<NP, PT>::CT][2][4];
    each_state<NP, PT>(st, [&](int p, int n, float& v) { v = enter && p0 + p < a.P && n < a.N ? enter[(int64_t)(p0 + p) * a.N + n] : 0.f; });
    if (warp == 0) {
        chunk_steps<true>(a, s, 0, raw, tokens(u.t0), A, bias);
        raw_steps(a, u.t0 + Q, tokens(u.t0 + Q), h, raw);
    }

    int buf = 0;
    for (int64_t t = u.t0; t < u.t1; t += Q, buf ^= 1) {
        const int n = tokens(t);
        const bool last = t + Q >= u.t1;
        if (!AHEAD) ask(t);
        __syncthreads();
        put<DT, XP, NP>(s.B[0], Q * LN, LN, ub);
        put<DT, XP, NP>(s.C[0], Q * LN, LN, uc);
        put_x<DT, NP, PT, true>(s, buf, ux, !last || a.ht ? pieces : 0);
        each_state<NP, PT>(st, [&](int p, int nn, float v) {
            const __nv_bfloat16 hi = __float2bfloat16_rn(v);
            s.S[0][p * LN + nn] = hi;
            if (XP > 1) s.S[XP - 1][p * LN + nn] = __float2bfloat16_rn(v - __bfloat162float(hi));
        });
        __syncthreads();
        if (AHEAD) ask(t + Q);
        // gates of this thread's outputs, two neighbours at a time
        uint32_t zr[PT / 8][2];
        if (a.z)
#pragma unroll
            for (int j = 0; j < PT / 8; ++j)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int i = 16 * warp + g + 8 * k, p = p0 + 8 * j + t2;
                    const uint16_t* src = (const uint16_t*)a.z + (t + i) * a.z_tok + h * a.z_head + p;
                    zr[j][k] = 0u;
                    if (i >= n || p >= a.P) continue;
                    if (a.z_pair) zr[j][k] = __ldg(reinterpret_cast<const uint32_t*>(src));
                    else zr[j][k] = __ldg(src) | (p + 1 < a.P ? (uint32_t)__ldg(src + 1) << 16 : 0u);
                }
        // rows 16 warp .. +15: what the state gives them, e^{G_i} C_i S^T
        const int m0 = 16 * warp;
        const SsmExp gi[2] = {s.G[buf][m0 + g], s.G[buf][m0 + g + 8]};
        float from[2] = {gi[0].whole + gi[0].rest, gi[1].whole + gi[1].rest};      // sums from the start of the 16 columns behind the tile's
        float acc[PT / 8][4] = {};
#pragma unroll
        for (int cp = XP - 1; cp >= 0; --cp)
#pragma unroll
            for (int sp = XP - 1 - cp; sp >= 0; --sp)
                warp_gemm<PT / 8, NP, false, false>(acc, s.C[cp], LN, m0, s.S[sp], LN, 0, lane);
        {
            float before = 0.f;
#pragma unroll
            for (int b = 0; b < 3; ++b) before += b < warp ? s.sum[buf][b] : 0.f;
            const float e0 = __expf(before + from[0]), e1 = __expf(before + from[1]);
#pragma unroll
            for (int j = 0; j < PT / 8; ++j) { acc[j][0] *= e0; acc[j][1] *= e0; acc[j][2] *= e1; acc[j][3] *= e1; }
        }
        // and the tokens of the chunk up to their own: 16 columns of scores at a time, their own 16 first.  In front of those e^{G_i - G_j} is
        // a row's factor to the 16 columns' end and a column's from there
#pragma unroll 1
        for (int j0 = m0; j0 >= 0; j0 -= 16) {
            float sc[2][4] = {};
#pragma unroll
            for (int cp = XP - 1; cp >= 0; --cp)
#pragma unroll
                for (int bp = XP - 1 - cp; bp >= 0; --bp)
                    warp_gemm<2, NP, false, false>(sc, s.C[cp], LN, m0, s.B[bp], LN, j0, lane);
            float dec[2][4];
            if (j0 == m0) {
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int j = m0 + 8 * c + t2 + k;
                        const SsmExp gj = s.G[buf][j];
                        const float d = s.d[buf][j];
#pragma unroll
                        for (int r = 0; r < 2; ++r) dec[c][2 * r + k] = __expf((gi[r].whole - gj.whole) + (gi[r].rest - gj.rest)) * d;
                    }
            } else {
                const float r0 = __expf(from[0]), r1 = __expf(from[1]), sum = s.sum[buf][j0 / 16];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float2 cf = *reinterpret_cast<const float2*>(&s.cf[buf][j0 + 8 * c + t2]);
                    dec[c][0] = r0 * cf.x; dec[c][1] = r0 * cf.y; dec[c][2] = r1 * cf.x; dec[c][3] = r1 * cf.y;
                }
                from[0] += sum; from[1] += sum;
            }
            uint32_t pa[XP][4];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float v[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        v[k] = j0 < m0 || 8 * c + t2 + k <= g + 8 * r ? sc[c][2 * r + k] * dec[c][2 * r + k] : 0.f;
                    const uint32_t w = pack_bf16x2(v[0], v[1]);
                    pa[0][2 * c + r] = w;
                    if (XP > 1) {
                        const float2 f = unpack_bf16x2(w);
                        pa[XP - 1][2 * c + r] = pack_bf16x2(v[0] - f.x, v[1] - f.y);
                    }
                }
#pragma unroll
            for (int nt = 0; nt < PT / 8; nt += 2)
#pragma unroll
                for (int xp = XP - 1; xp >= 0; --xp) {
                    uint32_t b[4];
                    load_b_t(b, s.x[xp], LP, 8 * nt, j0, lane);
#pragma unroll
                    for (int pp = XP - 1 - xp; pp >= 0; --pp) {
                        mma16816(acc[nt], pa[pp], b[0], b[1]);
                        mma16816(acc[nt + 1], pa[pp], b[2], b[3]);
                    }
                }
        }
        // D x, gate, store
        const bool odd = s.any_bad;
#pragma unroll
        for (int j = 0; j < PT / 8; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int i = m0 + g + 8 * k, p = 8 * j + t2;
                if (i >= n || p0 + p >= a.P) continue;
                float2 xv = unpack_bf16x2(*reinterpret_cast<const uint32_t*>(&s.x[0][i * LP + p]));
                if (XP > 1) {
                    const float2 lo = unpack_bf16x2(*reinterpret_cast<const uint32_t*>(&s.x[XP - 1][i * LP + p]));
                    xv.x += lo.x; xv.y += lo.y;
                }
                float2 v = make_float2(fmaf(Dh, xv.x, acc[j][2 * k]), fmaf(Dh, xv.y, acc[j][2 * k + 1]));
                if (odd) {
                    if (i >= s.bad[p]) v.x = __int_as_float(0x7fc00000);
                    if (i >= s.bad[p + 1]) v.y = __int_as_float(0x7fc00000);
                }
                if (a.z) {
                    const float2 z = DT == LAMPA_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&zr[j][k])) : unpack_bf16x2(zr[j][k]);
                    v.x *= z.x * sigmoidf_(z.x);
                    v.y *= z.y * sigmoidf_(z.y);
                }
                const size_t at = (size_t)(((t + i) * a.H + h) * a.P + p0 + p);
                if (a.y_pair) {
                    if (DT == LAMPA_F16) *reinterpret_cast<__half2*>((__half*)a.y + at) = __floats2half2_rn(v.x, v.y);
                    else *reinterpret_cast<uint32_t*>((__nv_bfloat16*)a.y + at) = pack_bf16x2(v.x, v.y);
                } else {
                    Elem<DT>::st(a.y, at, v.x);
                    if (p0 + p + 1 < a.P) Elem<DT>::st(a.y, at + 1, v.y);
                }
            }
        if (warp == 0 && !last) {
            chunk_steps<true>(a, s, buf ^ 1, raw, tokens(t + Q), A, bias);
            raw_steps(a, t + 2 * Q, tokens(t + 2 * Q), h, raw);
        }
        if (last && !(single && a.ht)) break;
        __syncthreads();
        update_state(st, s, expf(chunk_sum(s, buf)), pieces);
        if (odd) each_state<NP, PT>(st, [&](int p, int, float& v) { if (s.bad[p] < Q) v = __int_as_float(0x7fc00000); });
    }
    if (single && a.ht) {
        float* out = a.ht + ((int64_t)u.seq * a.H + h) * pn;
        each_state<NP, PT>(st, [&](int p, int n, float v) {
            if (p0 + p < a.P && n < a.N) out[(int64_t)(p0 + p) * a.N + n] = v;
        });
    }
}

template <int DT, int NP, int PT>
int launch_np(const SsmArgs& a, int units, bool blocks, cudaStream_t st) {
    static std::atomic<uint64_t> ready_s{0}, ready_o{0};
    using SMT = Sm<DT, NP, PT>;
    const int smem = (int)sizeof(Sm<DT, NP, PT>), smem_s = (int)SMT::STATE_BYTES;
    static_assert(sizeof(Sm<DT, NP, PT>) <= MAX_SMEM, "tiles fit");
    static_assert(offsetof(SMT, C) == SMT::STATE_BYTES, "what the block kernel uses comes first");
    const dim3 grid(units, a.H, (a.P + PT - 1) / PT);
    if (blocks) {
        if (!allow_smem(ready_s, ssm_state_kernel<DT, NP, PT>, smem_s)) return LAMPA_ERR_CUDA;
        {
            ProfScope prof("ssm_state", st);
            if (launch_chained(ssm_state_kernel<DT, NP, PT>, grid, dim3(THREADS), smem_s, st, a) != cudaSuccess) return LAMPA_ERR_CUDA;
        }
    }
    if (blocks || (a.cu && a.ht)) {
        const int rc = launch_ssm_pass(a, st);
        if (rc != LAMPA_OK) return rc;
    }
    if (!allow_smem(ready_o, ssm_out_kernel<DT, NP, PT>, smem)) return LAMPA_ERR_CUDA;
    ProfScope prof("ssm_out", st);
    return launch_chained(ssm_out_kernel<DT, NP, PT>, grid, dim3(THREADS), smem, st, a) == cudaSuccess ? LAMPA_OK : LAMPA_ERR_CUDA;
}

template <int DT, int NP>
int launch_dt(const SsmArgs& a, int units, bool blocks, cudaStream_t st) {
    if (a.P <= 16) return launch_np<DT, NP, 16>(a, units, blocks, st);
    if (a.P <= 32 || NP == 256) return launch_np<DT, NP, 32>(a, units, blocks, st);
    if constexpr (NP < 256) return launch_np<DT, NP, 64>(a, units, blocks, st);
    return LAMPA_ERR_UNSUPPORTED;
}

template <int DT>
int launch_any(const SsmArgs& a, int units, bool blocks, cudaStream_t st) {
    if (a.N <= 16) return launch_dt<DT, 16>(a, units, blocks, st);
    if (a.N <= 32) return launch_dt<DT, 32>(a, units, blocks, st);
    if (a.N <= 64) return launch_dt<DT, 64>(a, units, blocks, st);
    if (a.N <= 128) return launch_dt<DT, 128>(a, units, blocks, st);
    return launch_dt<DT, 256>(a, units, blocks, st);
}

}  // namespace

int launch_ssm_pass(const SsmArgs& a, cudaStream_t st) {
    // four elements to a thread where every SM still has 128 threads (16 heads of 64 x 128: 3.3 instead of 5.2 us; 7 sequences of 6 heads of
    // 32 x 16: 9.3 instead of 7.3)
    const bool vec = (int64_t)a.P * a.N * a.nseq * a.H >= (int64_t)sm_count() * 512 && (int64_t)a.P * a.N % 4 == 0 && (((uintptr_t)a.h0 | (uintptr_t)a.ht) & 15) == 0;
    const int64_t slabs = ((int64_t)a.P * a.N / (vec ? 4 : 1) + 255) / 256;
    if (slabs * a.nseq > INT32_MAX) return LAMPA_ERR_UNSUPPORTED;
    ProfScope prof("ssm_pass", st);
    return launch_chained(vec ? ssm_pass_kernel<4, 8> : ssm_pass_kernel<1, 8>, dim3((unsigned)(slabs * a.nseq), a.H), dim3(256), 0, st, a) == cudaSuccess
               ? LAMPA_OK : LAMPA_ERR_CUDA;
}

int launch_ssm_scan_mma(const SsmArgs& a, int dtype, int units, bool blocks, cudaStream_t st) {
    return dtype == LAMPA_BF16 ? launch_any<LAMPA_BF16>(a, units, blocks, st) : launch_any<LAMPA_F16>(a, units, blocks, st);
}

}  // namespace lampa
