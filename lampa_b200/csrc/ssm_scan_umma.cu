// Selective state space scan on the 5th-generation tensor cores: bf16, head dims and state sizes that are multiples of 8, N up to 128.
//
// The algebra is ssm_scan.cu's with chunks of 128 tokens.  One CTA takes a block of chunks for TWO heads of a group, which share C, B and
// their scores.  Per chunk (heads a, b side by side in the columns; [token][column] bf16 tiles with 128-byte rows and swizzle, 64
// columns to a panel, serve as either operand of every product):
//   G   = C B^T                   128 x 128, K = N                        scores
//   Y   = C [S_a^T | S_b^T]       128 x 128, K = N                        what the entering states give; scaled by e^{G_i} in place
//   S  += B^T [wx_a | wx_b]       N x 128,   K = 128 tokens               what the chunk adds to the states, decayed before
//   Y_h += P_h x_h                128 x 64 each, K = 128                  P_h: masked, decayed scores, bf16, from tensor memory
// All accumulators are in tensor memory (G | P | Y | S, 128 columns each), the states S in fp32 among them.
//
// Sixteen warps do the element work, thread = (row or state row, head, half of the 64 columns).  Four more serve them.  One issues the
// products (and is held up while the tensor core's queue is full, so that it does nothing else).  One copies the tiles in (tiled TMA from
// three-dimensional maps, which fill what lies beyond the head's columns with zeros) and is the only one that polls for completions: it
// passes them on through hardware named barriers (30 cycles, where a poll costs 200 - 300).  Two, one to a head, turn the chunks'
// steps into decays a chunk ahead (one for both was slower than the products of a chunk).  Waits are bounded, and the helpers walk through all their barriers whether or not one ran out, so
// nobody can be left waiting; nor can anybody reach a barrier twice in one phase, because no warp is more than a chunk ahead of another.
#include "profile.cuh"
#include "ssm.cuh"
#include "tmap.cuh"
#include "umma.cuh"

#include <algorithm>

namespace lampa {
namespace {

constexpr int UQ = 128;                           // tokens per chunk
constexpr int CWARPS = 16, CT = CWARPS * 32;      // element warps
constexpr int W_MMA = CWARPS, W_CTL = CWARPS + 1, W_TAB = CWARPS + 2;     // products; copies and completions; steps of the two heads
constexpr int THREADS = CT + 128;
constexpr int TILE = 16384;                       // [128][64] bf16
constexpr float LOG2E = 1.4426950408889634f;

// tensor-memory columns
constexpr int TM_G = 0, TM_P = 128, TM_Y = 256, TM_S = 384;

// named barriers of the element warps with one helper (CC), with the copying and the step warps (CS), with everybody (ALL), and of two
// helpers (HH)
constexpr int CC = CT + 32, CS = CT + 96, ALL = THREADS, HH = 64;
template <int N> __device__ __forceinline__ void nb_sync(int id) { asm volatile("bar.sync %0, %1;\n" :: "r"(id), "n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void nb_arrive(int id) { asm volatile("bar.arrive %0, %1;\n" :: "r"(id), "n"(N) : "memory"); }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint64_t adv(uint64_t d, uint32_t bytes) { return d + (uint64_t)(bytes >> 4); }
__device__ __forceinline__ int swz(int r, int c16) { return r * 128 + ((c16 ^ (r & 7)) << 4); }
__device__ __forceinline__ F2 unpack2(uint32_t u) { return f2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack2(F2 v) { float lo, hi; f2_get(v, lo, hi); return pack_bf16x2(lo, hi); }

// [128 tokens][64 columns] of one head (or group) into a panel
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t t, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n"
                 :: "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(t), "r"(smem_u32(bar)) : "memory");
}

// Per head and chunk, by token: G (log2, from the start of its 32 tokens on), d, d e^{what follows in its 32}, d e^{G_last - G}; between[q][b]: log2
// of the decay of the 32-token blocks behind b and in front of q, [q][q] of all in front of q
struct Tab { float G[UQ], d[UQ], cf[UQ], w[UQ], between[4][4]; };

// One warp, four tokens to a lane, one head.  The steps are asked for a chunk ahead (raw); tokens from n on have d = 0.  Returns the logarithm of the
// chunk's decay.  Every exponent is a sum of what lies between its two tokens, so that its error is one of its own size.  Inside 32 tokens
// differences of G are taken, which is a sum of exact whole numbers and small rests (SsmExp), 32 x 128 at most and rounded once: a decay there is good to
// 2 x 2^-13 ln 2 < 2^-12, a sixteenth of a step of the bf16 that it becomes.  What lies between blocks, and w, has no such limit.
struct Steps {
    float A, bias;
    int h;
    bool has;
    uint32_t raw[4];
    __device__ __forceinline__ Steps(const SsmArgs& a, int h0, int x, bool there) : h(there ? h0 + x : h0), has(there) {
        A = a.A[h];
        bias = a.dt_bias ? a.dt_bias[h] : 0.f;
    }
    __device__ __forceinline__ void ask(const SsmArgs& a, int64_t t, int n) {      // n <= 0: there is no such chunk
        if (n <= 0) return;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t at = (t + min(4 * (int)(threadIdx.x & 31) + k, n - 1)) * a.dt_tok + h;
            raw[k] = a.dt_dt == LAMPA_F32 ? __ldg((const uint32_t*)a.dt + at) : __ldg((const uint16_t*)a.dt + at);
        }
    }
    template <bool FULL>
    __device__ __forceinline__ float make(const SsmArgs& a, float* ws, Tab* s, int n) const {
        const int l = threadIdx.x & 31;
        float d[4], g[4], down = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool in = 4 * l + k < n && has;
            d[k] = in ? ssm_step_size(load_as_float(&raw[k], 0, a.dt_dt) + bias, a.softplus) : 0.f;
            g[k] = in ? d[k] * A : 0.f;
            down += g[k];
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {          // to the end of its 32 tokens, which eight lanes hold
            const float v = __shfl_down_sync(0xffffffffu, down, o, 8);
            if ((l & 7) + o < 8) down += v;
        }
        const float next = __shfl_down_sync(0xffffffffu, down, 1, 8), after = (l & 7) < 7 ? next : 0.f;
        float sum[4], e = 0.f, w[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) sum[b] = __shfl_sync(0xffffffffu, down, 8 * b);
#pragma unroll
        for (int b = 3; b > 0; --b) e += l < 8 * b ? sum[b] : 0.f;
        e += after;
#pragma unroll
        for (int k = 3; k >= 0; --k) { w[k] = d[k] * expf(e); e += g[k]; }
        *reinterpret_cast<float4*>(ws + 4 * l) = make_float4(w[0], w[1], w[2], w[3]);
        if (FULL) {
            SsmExp G[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const SsmExp x = ssm_split(g[k] * LOG2E);
                G[k] = k ? SsmExp{G[k - 1].whole + x.whole, G[k - 1].rest + x.rest} : x;
            }
            SsmExp up = G[3];
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                const float u = __shfl_up_sync(0xffffffffu, up.whole, o, 8), r = __shfl_up_sync(0xffffffffu, up.rest, o, 8);
                if ((l & 7) >= o) { up.whole += u; up.rest += r; }
            }
            const float pw = __shfl_up_sync(0xffffffffu, up.whole, 1, 8), pr = __shfl_up_sync(0xffffffffu, up.rest, 1, 8);
            const SsmExp p = {(l & 7) ? pw : 0.f, (l & 7) ? pr : 0.f};
            float cf[4], f = after;
#pragma unroll
            for (int k = 3; k >= 0; --k) { cf[k] = d[k] * ex2(f * LOG2E); f += g[k]; }
            *reinterpret_cast<float4*>(&s->G[4 * l]) = make_float4((p.whole + G[0].whole) + (p.rest + G[0].rest), (p.whole + G[1].whole) + (p.rest + G[1].rest),
                                                                   (p.whole + G[2].whole) + (p.rest + G[2].rest), (p.whole + G[3].whole) + (p.rest + G[3].rest));
            *reinterpret_cast<float4*>(&s->d[4 * l]) = make_float4(d[0], d[1], d[2], d[3]);
            *reinterpret_cast<float4*>(&s->cf[4 * l]) = make_float4(cf[0], cf[1], cf[2], cf[3]);
            float t = 0.f;
            const int q = (l >> 2) & 3, b = l & 3;
#pragma unroll
            for (int m = 0; m < 3; ++m) t += m < q && (b == q || m > b) ? sum[m] : 0.f;
            if (l < 16) s->between[q][b] = t * LOG2E;
        }
        return (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
};

// State elements of a thread: row n and PC columns p0 ..  With N <= 64 the second half of dS's rows repeats the first (B's panel is there
// twice), and its warps take the other half of the columns.
template <int NPAN>
struct Own {
    static constexpr int PC = NPAN == 2 ? 32 : 16;
    int n, p0;
    __device__ __forceinline__ Own(int q, int half, int lane) {
        n = NPAN == 2 ? 32 * q + lane : 32 * (q & 1) + lane;
        p0 = 32 * half + (NPAN == 2 ? 0 : 16 * (q >> 1));
    }
};
template <int PC> __device__ __forceinline__ void tm_ld(float (&x)[PC], uint32_t t);
template <> __device__ __forceinline__ void tm_ld<32>(float (&x)[32], uint32_t t) { tmem_ld32(x, t); }
template <> __device__ __forceinline__ void tm_ld<16>(float (&x)[16], uint32_t t) { tmem_ld16(x, t); }
__device__ __forceinline__ void tm_st8(uint32_t t, const uint32_t (&w)[8]) {        // (waited for by tm_wait_st)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
                 :: "r"(t), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t t, const uint32_t (&w)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
                 :: "r"(t), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]),
                    "r"(w[8]), "r"(w[9]), "r"(w[10]), "r"(w[11]), "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15]) : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int32_t x, int32_t y, int32_t t, const void* src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n"
                 :: "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(t), "r"(smem_u32(src)) : "memory");
}

struct Maps { CUtensorMap x, B, C, z, y; };

// -------------------------------------------------------------------------------------------------
// What bounds it: shared memory, of which a chunk's 24 products read 192 KB and everything else moves as much again (3.1 k of the 4.1 k cycles
// of a chunk), and how the products' issue and the element work wait for one another: 61 440 tokens, 16 heads of 64 x 128: 64 us (67 between events), tensor pipe
// 35 %, issue slots 43 %, DRAM 34 % (2.2 TB/s).  One step warp for both heads: 75 us; the same warp polling and issuing: 98.
// What a block makes of an empty state.  Its products take d x e^{..} in three bf16 pieces where somebody will see the state (24 bits), in one
// where only y will.  Every chunk's sum starts from zero and is added to the states in fp32 arithmetic.
// -------------------------------------------------------------------------------------------------
// A_NEXT: a chunk's tiles and steps are there, and the place of its first half is free; A_F: that of its second half is; A_W: [half][chunk
// parity] tokens are in place; A_R: [chunk parity] the products of a chunk are issued; A_END: all of them are complete
enum { A_NEXT = 1, A_F, A_W, A_R = A_W + 4, A_END = A_R + 2 };
struct SmA {
    unsigned char wx[2][3][2][TILE / 2];          // [half of the tokens][piece][head]
    unsigned char B[2][2][TILE];                  // [chunk parity][panel]
    unsigned char x[2][2][TILE];                  // [chunk parity][head]
    float w[2][2][UQ];                            // [chunk parity][head]
    float tot[4][2];
    uint64_t bar[2], in[2], drain;
    uint32_t tslot;
};

template <int NPAN, int PIECES>
__global__ void __launch_bounds__(THREADS, 1) ssm_state_umma_kernel(SsmArgs a, const __grid_constant__ Maps maps) {
    if (chain_wait()) return;
    extern __shared__ __align__(1024) unsigned char raw[];
    SmA& s = *reinterpret_cast<SmA*>(raw);
    SsmUnit u;
    if (!ssm_unit(a, blockIdx.x, u) || u.outside || (u.single(a.bl) && !a.ht)) return;
    const bool single = PIECES == 3 && u.single(a.bl);             // the whole sequence: from the state that enters it to the final one
    const int hpg = a.H / a.G, pairs = (hpg + 1) / 2, grp = blockIdx.y / pairs, hl = 2 * (blockIdx.y % pairs), slab = blockIdx.z * 64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h0 = grp * hpg + hl;
    const int chunks = (int)((u.t1 - u.t0 + UQ - 1) / UQ);
    if (warp == W_MMA) {
        if (lane == 0) {
            mbar_init(&s.bar[0], 1); mbar_init(&s.bar[1], 1); mbar_init(&s.in[0], 1); mbar_init(&s.in[1], 1); mbar_init(&s.drain, 1);
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&s.tslot, 256);
    }
    tc_fence_before();
    nb_sync<ALL>(0);
    tc_fence_after();
    const uint32_t tm = s.tslot;

    if (warp == W_MMA) {
        constexpr uint32_t id = umma_idesc(128, 128, 1, 1);
        for (int c = 0; c < chunks; ++c) {
#pragma unroll 1
            for (int hf = 0; hf < 2; ++hf) {
                nb_sync<CC>(A_W + 2 * hf + (c & 1));
                if (lane == 0) {
                    tc_fence_after();
                    const uint64_t da = umma_desc_mn128(smem_u32(s.B[c & 1][0]) + hf * (TILE / 2), TILE);
#pragma unroll
                    for (int p = PIECES - 1; p >= 0; --p) {
                        const uint64_t db = umma_desc_mn128(smem_u32(s.wx[hf][p][0]), TILE / 2);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f16_ss(tm + 128 * (c & 1), adv(da, 2048 * k), adv(db, 2048 * k), id, hf || p < PIECES - 1 || k);
                    }
                    umma_commit(&s.bar[hf]);
                }
                __syncwarp();
            }
            nb_arrive<HH>(A_R + (c & 1));
        }
        if (lane == 0) {
            umma_commit(&s.drain);
            if (!mbar_drain(&s.drain, 0)) set_status(a.status, LAMPA_ERR_TIMEOUT, 53, 0);
        }
        __syncwarp();
        nb_sync<ALL>(0);
        tmem_dealloc(tm, 256);
        return;
    }
    if (warp == W_CTL) {
        bool dead = false;
        auto load = [&](int c) {                  // the second panel of a small state is its first again
            uint64_t* bar = &s.in[c & 1];
            const int32_t t = (int32_t)(u.t0 + (int64_t)c * UQ);
            mbar_expect_tx(bar, 4 * TILE);
            tma_load_3d(s.x[c & 1][0], &maps.x, slab, h0, t, bar);
            tma_load_3d(s.x[c & 1][1], &maps.x, slab, min(h0 + 1, a.H - 1), t, bar);
            tma_load_3d(s.B[c & 1][0], &maps.B, 0, grp, t, bar);
            tma_load_3d(s.B[c & 1][1], &maps.B, NPAN == 2 ? 64 : 0, grp, t, bar);
        };
        if (lane == 0) load(0);
        int loaded = 1;
        for (int c = 0; c < chunks; ++c) {
            if (c > 1) nb_sync<HH>(A_R + (c & 1));         // the products of chunk c - 2 are issued: nobody gets further ahead
            if (lane == 0) {
                mbar_wait(&s.in[c & 1], (c >> 1) & 1, dead, a.status, 53, a.poll_budget);
                if (c > 0) mbar_wait(&s.bar[0], (c - 1) & 1, dead, a.status, 53, a.poll_budget);
            }
            __syncwarp();
            tc_fence_before();
            nb_sync<CS>(A_NEXT);
            if (lane == 0) {
                // chunk c - 1 is taken in: its buffers are free
                if (c > 0) mbar_wait(&s.bar[1], (c - 1) & 1, dead, a.status, 53, a.poll_budget);
                if (c + 1 < chunks && !dead) { load(c + 1); loaded = c + 2; }
            }
            __syncwarp();
            tc_fence_before();
            nb_arrive<CC>(A_F);
        }
        if (lane == 0) {
            mbar_wait(&s.bar[0], (chunks - 1) & 1, dead, a.status, 53, a.poll_budget);
            mbar_wait(&s.bar[1], (chunks - 1) & 1, dead, a.status, 53, a.poll_budget);
        }
        __syncwarp();
        tc_fence_before();
        nb_arrive<CC>(A_END);
        if (lane == 0 && dead) {                  // copies that nobody has waited for
            bool ok = true;
            for (int c = max(0, loaded - 2); c < loaded; ++c) ok = mbar_drain(&s.in[c & 1], (c >> 1) & 1) && ok;
            if (!ok) set_status(a.status, LAMPA_ERR_TIMEOUT, 53, 1);
        }
        __syncwarp();
        for (int c = max(0, chunks - 2); c < chunks; ++c) nb_sync<HH>(A_R + (c & 1));
        nb_sync<ALL>(0);
        return;
    }
    if (warp >= W_TAB) {
        const int x = warp - W_TAB;
        Steps p(a, h0, x, hl + x < hpg);
        auto rows = [&](int c) { return (int)max((int64_t)0, min((int64_t)UQ, u.t1 - (u.t0 + (int64_t)c * UQ))); };
        float log_dec = 0.f;
        p.ask(a, u.t0, rows(0));
        for (int c = 0; c < chunks; ++c) {
            const float g = p.make<false>(a, s.w[c & 1][x], nullptr, rows(c));
            if (lane == 0) s.tot[c & 3][x] = expf(g);
            log_dec += g;
            p.ask(a, u.t0 + (int64_t)(c + 1) * UQ, rows(c + 1));
            nb_sync<CS>(A_NEXT);
        }
        if (p.has && lane == 0 && slab == 0 && !single) a.blk_dec[u.slot * a.H + h0 + x] = log_dec;
        nb_sync<ALL>(0);
        return;
    }

    const int q = warp & 3, hd = warp >> 3, half = (warp >> 2) & 1;
    const Own<NPAN> own(q, half, lane);
    constexpr int PC = Own<NPAN>::PC;
    const bool has = hl + hd < hpg;
    const int64_t pn = (int64_t)a.P * a.N;
    float st[PC];
    const float* const enter = single && a.h0 && has && own.n < a.N ? a.h0 + ((int64_t)u.seq * a.H + h0 + hd) * pn + own.n : nullptr;
#pragma unroll
    for (int i = 0; i < PC; ++i) st[i] = enter && slab + own.p0 + i < a.P ? enter[(int64_t)(slab + own.p0 + i) * a.N] : 0.f;
    auto take_in = [&](int c) {                   // states <- decay * states + dS of chunk c
        float ds[PC];
        tm_ld<PC>(ds, tm + ((uint32_t)(32 * q) << 16) + 128 * (c & 1) + 64 * hd + own.p0);
        const float dec = s.tot[c & 3][hd];
#pragma unroll
        for (int i = 0; i < PC; ++i) st[i] = fmaf(dec, st[i], ds[i]);
    };
    const int col = threadIdx.x & 7, r0 = (threadIdx.x >> 3) & 63;
    for (int c = 0; c < chunks; ++c) {
        const int n = (int)min((int64_t)UQ, u.t1 - (u.t0 + (int64_t)c * UQ));
        nb_sync<CS>(A_NEXT);
        tc_fence_after();
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if (hf) { nb_sync<CC>(A_F); tc_fence_after(); }
            const int row = 64 * hf + r0;
            if (n < UQ && hf == 0) {              // what follows the sequence's last token is not its own: zero
                for (int i = threadIdx.x; i < (UQ - n) * 16; i += CT)
                    *reinterpret_cast<uint4*>(s.B[c & 1][(i >> 3) & 1] + swz(n + (i >> 4), i & 7)) = make_uint4(0u, 0u, 0u, 0u);
            }
            F2 f[2][4];
            const F2 neg = f2(-1.f);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const F2 w2 = f2(s.w[c & 1][k][row]);
                uint4 v = *reinterpret_cast<const uint4*>(s.x[c & 1][k] + swz(row, col));
                if (row >= n) v = make_uint4(0u, 0u, 0u, 0u);
                f[k][0] = mul2(unpack2(v.x), w2); f[k][1] = mul2(unpack2(v.y), w2);
                f[k][2] = mul2(unpack2(v.z), w2); f[k][3] = mul2(unpack2(v.w), w2);
            }
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint4 o = make_uint4(pack2(f[k][0]), pack2(f[k][1]), pack2(f[k][2]), pack2(f[k][3]));
                    *reinterpret_cast<uint4*>(s.wx[hf][p][k] + swz(r0, col)) = o;
                    if (p + 1 == PIECES) continue;
                    f[k][0] = fma2(unpack2(o.x), neg, f[k][0]); f[k][1] = fma2(unpack2(o.y), neg, f[k][1]);
                    f[k][2] = fma2(unpack2(o.z), neg, f[k][2]); f[k][3] = fma2(unpack2(o.w), neg, f[k][3]);
                }
            fence_async_smem();
            tc_fence_before();
            nb_arrive<CC>(A_W + 2 * hf + (c & 1));
        }
        if (c > 0) take_in(c - 1);
    }
    nb_sync<CC>(A_END);
    tc_fence_after();
    take_in(chunks - 1);
    float* const out = single ? a.ht + ((int64_t)u.seq * a.H + h0 + hd) * pn : a.blk + (u.slot * a.H + h0 + hd) * pn;
    if (has && own.n < a.N)
#pragma unroll
        for (int i = 0; i < PC; ++i)
            if (slab + own.p0 + i < a.P) out[(int64_t)(slab + own.p0 + i) * a.N + own.n] = st[i];
    tc_fence_before();
    nb_sync<ALL>(0);
}

// -------------------------------------------------------------------------------------------------
// The output, walking through a block from the state that enters it.
// What bounds it: a chain of dependent phases of four warps to a scheduler, 10.2 k cycles a chunk of two heads for 3.4 k issue slots (wx 0.9 k,
// scores 2 - 3 k, states and the entering states' share 1.5 k, gates 2 k beside the products P x, output 0.7 k, hand-overs), and behind that shared
// memory (4.6 k cycles): 61 440 tokens, 16 heads of 64 x 128: 158 us between events, issue slots 39 %, tensor pipe 18 %,
// DRAM 37 % (2.4 TB/s).  (154 where an exponent between tokens is a difference of sums from the chunk's start, which is wrong behind a large step, and
// nobody looks at a barrier before arming it.)
// On the way: tiles by cp.async of the element warps 398 us (spills reach L2 here: shared memory leaves L1 nothing), TMA 198, states in tensor
// memory instead of registers 159, gates while P x runs 146.  All scores of a row loaded at once: 176 (spills).
// -------------------------------------------------------------------------------------------------
enum { C_NEXT = 1, C_WX, C_G, C_Y, C_P, C_DS, C_PX, C_YF };
template <int NPAN>
struct SmC {
    unsigned char C[NPAN][TILE], B[2][TILE], x[2][TILE], wx[2][TILE], z[2][TILE], S[2][NPAN * TILE / 2];
    Tab tab[2][2];                                // [chunk parity][head]
    float tot[2][2];
    int bad[2][64];                               // first row of the column that is not finite, or UQ
    int any_bad[2];
    uint64_t in_c, in_b, in_x, in_z, g, y, ds, px, drain;
    uint32_t tslot;
};
// Two warps wait in the output pass, and each arms barriers that only the other one waits on: z's (in_z) is armed by the product warp, C's and B's by
// the copying warp.  Behind C_NEXT their last phases are complete, unless the other one's wait has run out; a barrier must not be armed in an
// open phase, so whoever arms looks for itself, and gives up as well where it finds one.
__device__ __forceinline__ void complete_or_dead(uint64_t* bar, int c, bool& dead, int32_t* status) {
    if (dead || mbar_try_wait(bar, c & 1)) return;
    dead = true;
    set_status(status, LAMPA_ERR_TIMEOUT, 54, c & 1);
}

// z sigmoid(z) of two values.  With t = e^-|z| the denominator 1 + t lies in [1, 2], where its reciprocal is a cubic and one Newton step:
// 1 - v p(v) = T4(2v - 3) / T4(3) with the Chebyshev polynomial T4, 1 / 577 at most, squared by the step: 3e-6.  (Through the
// special function unit, which has a quarter of the issue rate, both the exponential and the reciprocal would bound the epilogue.)
// The numerator z e^min(z, 0) is the larger of z and z t.
__device__ __forceinline__ F2 silu2(F2 z) {
    float z0, z1, m0, m1;
    f2_get(z, z0, z1);
    const F2 t = f2(ex2(-LOG2E * fabsf(z0)), ex2(-LOG2E * fabsf(z1)));
    const F2 v = add2(t, f2(1.f));
    F2 p = fma2(v, f2(-128.f / 577.f), f2(768.f / 577.f));
    p = fma2(p, v, f2(-1696.f / 577.f));
    p = fma2(p, v, f2(1632.f / 577.f));
    p = mul2(p, fma2(mul2(v, p), f2(-1.f), f2(2.f)));
    f2_get(mul2(z, t), m0, m1);
    return mul2(f2(fmaxf(z0, m0), fmaxf(z1, m1)), p);
}

template <int NPAN>
__global__ void __launch_bounds__(THREADS, 1) ssm_out_umma_kernel(SsmArgs a, const __grid_constant__ Maps maps) {
    if (chain_wait()) return;
    extern __shared__ __align__(1024) unsigned char raw[];
    SmC<NPAN>& s = *reinterpret_cast<SmC<NPAN>*>(raw);
    SsmUnit u;
    const int hpg = a.H / a.G, pairs = (hpg + 1) / 2, grp = blockIdx.y / pairs, hl = 2 * (blockIdx.y % pairs), slab = blockIdx.z * 64;
    if (a.cu && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_offsets(a.cu, a.nseq, a.n_tok, a.status, 50);
    if (!ssm_unit(a, blockIdx.x, u)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h0 = grp * hpg + hl;
    if (u.outside) {                              // rows of no sequence read as zero
        for (int hd = 0; hd < 2 && hl + hd < hpg; ++hd)
            for (int64_t i = threadIdx.x; i < (u.t1 - u.t0) * 64; i += THREADS) {
                const int p = slab + (int)(i % 64);
                if (p < a.P) ((__nv_bfloat16*)a.y)[((u.t0 + i / 64) * a.H + h0 + hd) * a.P + p] = __float2bfloat16_rn(0.f);
            }
        return;
    }
    const int chunks = (int)((u.t1 - u.t0 + UQ - 1) / UQ);
    if (warp == W_MMA) {
        if (lane == 0) {
            mbar_init(&s.in_c, 1); mbar_init(&s.in_b, 1); mbar_init(&s.in_x, 1); mbar_init(&s.in_z, 1);
            mbar_init(&s.g, 1); mbar_init(&s.y, 1); mbar_init(&s.ds, 1); mbar_init(&s.px, 1); mbar_init(&s.drain, 1);
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&s.tslot, 512);
    }
    tc_fence_before();
    nb_sync<ALL>(0);
    tc_fence_after();
    const uint32_t tm = s.tslot;

    if (warp == W_MMA) {
        bool dead = false;
        const uint64_t dC = umma_desc_k128(smem_u32(s.C[0])), dBk = umma_desc_k128(smem_u32(s.B[0])), dBm = umma_desc_mn128(smem_u32(s.B[0]), TILE),
                       dS = umma_desc_mn128(smem_u32(s.S[0]), NPAN * TILE / 2), dW = umma_desc_mn128(smem_u32(s.wx[0]), TILE),
                       dX0 = umma_desc_mn128(smem_u32(s.x[0])), dX1 = umma_desc_mn128(smem_u32(s.x[1]));
        auto scores_and_states = [&](int c) {     // G of chunk c as soon as its tiles are there, Y when the last chunk's has been read
            if (lane == 0) {
                mbar_wait(&s.in_c, c & 1, dead, a.status, 54, a.poll_budget_products);
                mbar_wait(&s.in_b, c & 1, dead, a.status, 54, a.poll_budget_products);
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 4 * NPAN; ++k) {
                    const uint32_t at = (k >> 2) * TILE + (k & 3) * 32;
                    umma_f16_ss(tm + TM_G, adv(dC, at), adv(dBk, at), umma_idesc(128, 128, 0, 0), k > 0);
                }
                umma_commit(&s.g);
            }
            __syncwarp();
            nb_sync<CC>(C_YF);
            if (lane == 0) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 4 * NPAN; ++k)
                    umma_f16_ss(tm + TM_Y, adv(dC, (k >> 2) * TILE + (k & 3) * 32), adv(dS, 2048 * k), umma_idesc(128, 128, 0, 1), k > 0);
                umma_commit(&s.y);
            }
            __syncwarp();
        };
        const int h1 = min(h0 + 1, a.H - 1);
        int asked_z = 0;
        auto load_z = [&](int c) {
            const int32_t t = (int32_t)(u.t0 + (int64_t)c * UQ);
            mbar_expect_tx(&s.in_z, 2 * TILE);
            tma_load_3d(s.z[0], &maps.z, slab, h0, t, &s.in_z);
            tma_load_3d(s.z[1], &maps.z, slab, h1, t, &s.in_z);
            ++asked_z;
        };
        if (lane == 0 && a.z_vec) load_z(0);
        scores_and_states(0);
        for (int c = 0; c < chunks; ++c) {
            const bool last = c + 1 == chunks;
            nb_sync<ALL>(C_NEXT);
            if (lane == 0 && c > 0) {             // the last chunk's output lies in z's place; when it has been read, z may follow
                const int32_t t = (int32_t)(u.t0 + (int64_t)(c - 1) * UQ);
                tma_store_3d(&maps.y, slab, h0, t, s.z[0]);
                if (hl + 1 < hpg) tma_store_3d(&maps.y, slab, h1, t, s.z[1]);
                bulk_commit();
                if (a.z_vec) complete_or_dead(&s.in_z, c - 1, dead, a.status);
                bulk_wait_read();
                if (a.z_vec && !dead) load_z(c);
            }
            __syncwarp();
            nb_sync<CC>(C_WX);
            if (lane == 0 && !last) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 8; ++k) umma_f16_ss(tm + TM_S, adv(dBm, 2048 * k), adv(dW, 2048 * k), umma_idesc(128, 128, 1, 1), 1);
                umma_commit(&s.ds);
            }
            __syncwarp();
            nb_sync<CC>(C_P);
            if (lane == 0) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 8; ++k) umma_f16_ts(tm + TM_Y, tm + TM_P + 8 * k, adv(dX0, 2048 * k), umma_idesc(128, 64, 0, 1), 1);
#pragma unroll
                for (int k = 0; k < 8; ++k) umma_f16_ts(tm + TM_Y + 64, tm + TM_P + 64 + 8 * k, adv(dX1, 2048 * k), umma_idesc(128, 64, 0, 1), 1);
                umma_commit(&s.px);
            }
            __syncwarp();
            if (!last) scores_and_states(c + 1);
        }
        if (lane == 0) {
            umma_commit(&s.drain);
            bool ok = mbar_drain(&s.drain, 0);
            if (asked_z) ok = mbar_drain(&s.in_z, (asked_z - 1) & 1) && ok;
            if (!ok) set_status(a.status, LAMPA_ERR_TIMEOUT, 54, 0);
        }
        __syncwarp();
        nb_sync<ALL>(0);
        tmem_dealloc(tm, 512);
        return;
    }
    if (warp == W_CTL) {
        bool dead = false;
        const int h1 = min(h0 + 1, a.H - 1);
        auto tok = [&](int c) { return (int32_t)(u.t0 + (int64_t)c * UQ); };
        auto load_C = [&](int c) {
            mbar_expect_tx(&s.in_c, NPAN * TILE);
#pragma unroll
            for (int p = 0; p < NPAN; ++p) tma_load_3d(s.C[p], &maps.C, 64 * p, grp, tok(c), &s.in_c);
        };
        auto load_B = [&](int c) {                // the second panel of a small state is its first again
            mbar_expect_tx(&s.in_b, 2 * TILE);
            tma_load_3d(s.B[0], &maps.B, 0, grp, tok(c), &s.in_b);
            tma_load_3d(s.B[1], &maps.B, NPAN == 2 ? 64 : 0, grp, tok(c), &s.in_b);
        };
        auto load_x = [&](int c) {
            mbar_expect_tx(&s.in_x, 2 * TILE);
            tma_load_3d(s.x[0], &maps.x, slab, h0, tok(c), &s.in_x);
            tma_load_3d(s.x[1], &maps.x, slab, h1, tok(c), &s.in_x);
        };
        // A wait that ran out (`dead`), or one of the product warp's whose copy is not there yet, ends the loading; what was asked for is drained at the end.
        int asked_c = 1, asked_b = 1, asked_x = 1;
        if (lane == 0) { load_x(0); load_C(0); load_B(0); }
        __syncwarp();
        nb_arrive<CS>(C_DS);
        auto wait = [&](uint64_t* bar, int c) { mbar_wait(bar, c & 1, dead, a.status, 54, a.poll_budget); };
        for (int c = 0; c < chunks; ++c) {
            const bool more = c + 1 < chunks;
            if (lane == 0) wait(&s.in_x, c);
            __syncwarp();
            nb_sync<ALL>(C_NEXT);
            if (lane == 0) wait(&s.g, c);
            __syncwarp();
            tc_fence_before();
            nb_arrive<CC>(C_G);
            if (lane == 0) {
                if (more) {
                    complete_or_dead(&s.in_c, c, dead, a.status);
                    complete_or_dead(&s.in_b, c, dead, a.status);
                }
                wait(&s.y, c);
                if (more && !dead) { load_C(c + 1); ++asked_c; }
            }
            __syncwarp();
            if (more) {                           // the states' operand has been read, what the chunk adds to them is there
                if (lane == 0) {
                    wait(&s.ds, c);
                    if (!dead) { load_B(c + 1); ++asked_b; }
                }
                __syncwarp();
                tc_fence_before();
                nb_arrive<CS>(C_DS);
            }
            if (lane == 0 && a.z_vec) wait(&s.in_z, c);
            __syncwarp();
            tc_fence_before();
            nb_arrive<CC>(C_Y);
            if (lane == 0) {
                wait(&s.px, c);
                if (more && !dead) { load_x(c + 1); ++asked_x; }
            }
            __syncwarp();
            tc_fence_before();
            nb_arrive<CC>(C_PX);
        }
        if (lane == 0) {
            bool ok = mbar_drain(&s.in_c, (asked_c - 1) & 1);
            ok = mbar_drain(&s.in_b, (asked_b - 1) & 1) && ok;
            ok = mbar_drain(&s.in_x, (asked_x - 1) & 1) && ok;
            if (!ok) set_status(a.status, LAMPA_ERR_TIMEOUT, 54, 1);
        }
        __syncwarp();
        nb_sync<ALL>(0);
        return;
    }
    if (warp >= W_TAB) {
        const int x = warp - W_TAB;
        Steps p(a, h0, x, hl + x < hpg);
        auto rows = [&](int c) { return (int)max((int64_t)0, min((int64_t)UQ, u.t1 - (u.t0 + (int64_t)c * UQ))); };
        p.ask(a, u.t0, rows(0));
        for (int c = 0; c < chunks; ++c) {
            const float g = p.make<true>(a, s.tab[c & 1][x].w, &s.tab[c & 1][x], rows(c));
            if (lane == 0) s.tot[c & 1][x] = expf(g);
            p.ask(a, u.t0 + (int64_t)(c + 1) * UQ, rows(c + 1));
            __syncwarp();
            nb_arrive<CS>(C_DS);                  // the states that enter chunk c may be decayed for what it adds
            nb_sync<ALL>(C_NEXT);
        }
        nb_sync<ALL>(0);
        return;
    }

    const int q = warp & 3, hd = warp >> 3, half = (warp >> 2) & 1, row = 32 * q + lane;
    const Own<NPAN> own(q, half, lane);
    constexpr int PC = Own<NPAN>::PC;
    const int h = h0 + hd, len = (int)(u.t1 - u.t0);
    const bool has = hl + hd < hpg;
    const uint32_t tl = tm + ((uint32_t)(32 * q) << 16);
    if (threadIdx.x < 128) s.bad[threadIdx.x >> 6][threadIdx.x & 63] = UQ;
    if (threadIdx.x < 2) s.any_bad[threadIdx.x] = 0;
    // scores above the diagonal stay zero
    for (int b = q + 1; b < 4; ++b) {
        const uint32_t zero[8] = {};
        tm_st8(tl + TM_P + 64 * hd + 16 * b + 8 * half, zero);
    }
    tm_wait_st();
    // 16-byte pieces of this thread's row (and state row): piece k lies at the first one's offset with k in its bits 4 and up flipped
    const int at0 = swz(row, 4 * half), sat0 = swz(own.n, own.p0 / 8);
    // 16 state elements: as bf16 to the operand of the chunk's Y, decayed to the accumulator of what it adds
    auto put_state = [&](int k, const float (&v)[16], float dec) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint4*>(s.S[hd] + (sat0 ^ ((2 * k + i) << 4))) =
                make_uint4(pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                           pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i] * dec);
        tm_st16(tl + TM_S + 64 * hd + own.p0 + 16 * k, w);
    };
    {
        const bool single = u.single(a.bl);
        const int64_t pn = (int64_t)a.P * a.N;
        const float* enter = !has ? nullptr : single ? (a.h0 ? a.h0 + ((int64_t)u.seq * a.H + h) * pn : nullptr) : a.blk + (u.slot * a.H + h) * pn;
        nb_sync<CS>(C_DS);
        const float dec = s.tot[0][hd];
#pragma unroll
        for (int k = 0; k < PC / 16; ++k) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int p = slab + own.p0 + 16 * k + i;
                v[i] = enter && own.n < a.N && p < a.P ? enter[(int64_t)p * a.N + own.n] : 0.f;
            }
            put_state(k, v, dec);
        }
    }
    tm_wait_st();
    fence_async_smem();
    tc_fence_before();
    nb_arrive<CC>(C_YF);
    const F2 Dh = f2(has && a.D ? a.D[h] : 0.f);

    for (int c = 0; c < chunks; ++c) {
        const bool last = c + 1 == chunks;
        const int n = min(UQ, len - c * UQ);
        const Tab& t = s.tab[c & 1][hd];
        nb_sync<ALL>(C_NEXT);                     // x and the steps are there
        // ---- wx
        {
            const F2 w2 = f2(t.w[row]);
            float odd = 0.f;
            uint4 xr[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) xr[k] = *reinterpret_cast<const uint4*>(s.x[hd] + (at0 ^ (k << 4)));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const F2 f0 = unpack2(xr[k].x), f1 = unpack2(xr[k].y), f2_ = unpack2(xr[k].z), f3 = unpack2(xr[k].w);
                float m0, m1;
                f2_get(add2(add2(f0, f1), add2(f2_, f3)), m0, m1);
                odd = fmaf(m0, 0.f, odd); odd = fmaf(m1, 0.f, odd);            // NaN with any that is not finite
                *reinterpret_cast<uint4*>(s.wx[hd] + (at0 ^ (k << 4))) =
                    make_uint4(pack2(mul2(f0, w2)), pack2(mul2(f1, w2)), pack2(mul2(f2_, w2)), pack2(mul2(f3, w2)));
            }
            if (odd != 0.f || row >= n) {
                // Elements that are not finite may not reach the rows above through a zero score, and what follows the sequence's last
                // token is not its own: both become zero in the tile
#pragma unroll 1
                for (int e = 0; e < 32; ++e) {
                    uint16_t* p = reinterpret_cast<uint16_t*>(s.x[hd] + (at0 ^ ((e >> 3) << 4))) + (e & 7);
                    if (row >= n) *p = 0;
                    else if ((*p & 0x7f80) == 0x7f80) { *p = 0; atomicMin(&s.bad[hd][32 * half + e], row); s.any_bad[hd] = 1; }
                }
            }
        }
        fence_async_smem();
        nb_arrive<CC>(C_WX);
        // ---- decayed scores
        nb_sync<CC>(C_G);
        tc_fence_after();
        const float Gi = t.G[row];
        {
            // Sixteen columns of every 32-block up to the diagonal; the two warps of a row share the blocks.  Below the diagonal block
            // e^{G_i - G_j} is a row's factor to the block's end and a column's from there, both at most 1.
            const int j0 = 16 * half;
            float nx[16];
            tmem_ld16_issue(nx, tl + TM_G + j0);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (b > q) break;
                float sc[16];
                tmem_wait_ld();
                tmem_loaded(nx);
#pragma unroll
                for (int j = 0; j < 16; ++j) sc[j] = nx[j];
                if (b < q) tmem_ld16_issue(nx, tl + TM_G + 32 * (b + 1) + j0);
                uint32_t o[8];
                if (b < q) {
                    const F2 r = f2(ex2(Gi + t.between[q][b]));
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(&t.cf[32 * b + j0 + j]);
                        o[j / 2] = pack2(mul2(f2(sc[j], sc[j + 1]), mul2(F2{f.x}, r)));
                        o[j / 2 + 1] = pack2(mul2(f2(sc[j + 2], sc[j + 3]), mul2(F2{f.y}, r)));
                    }
                } else {
                    const int m = lane - j0;      // the last column that counts; what lies beyond is masked as bits, whatever it is
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 g = *reinterpret_cast<const float4*>(&t.G[32 * b + j0 + j]);
                        const ulonglong2 d = *reinterpret_cast<const ulonglong2*>(&t.d[32 * b + j0 + j]);
                        o[j / 2] = pack2(mul2(f2(sc[j], sc[j + 1]), mul2(F2{d.x}, f2(ex2(Gi - g.x), ex2(Gi - g.y)))));
                        o[j / 2 + 1] = pack2(mul2(f2(sc[j + 2], sc[j + 3]), mul2(F2{d.y}, f2(ex2(Gi - g.z), ex2(Gi - g.w)))));
                        o[j / 2] &= m > j ? 0xffffffffu : m == j ? 0xffffu : 0u;
                        o[j / 2 + 1] &= m > j + 2 ? 0xffffffffu : m == j + 2 ? 0xffffu : 0u;
                    }
                }
                tm_st8(tl + TM_P + 64 * hd + 16 * b + j0 / 2, o);
            }
        }
        // ---- states
        if (!last) {
            nb_sync<CS>(C_DS);
            tc_fence_after();
            const float dec = s.tot[(c + 1) & 1][hd];
            float v[PC / 16][16];
#pragma unroll
            for (int k = 0; k < PC / 16; ++k) tmem_ld16_issue(v[k], tl + TM_S + 64 * hd + own.p0 + 16 * k);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < PC / 16; ++k) {
                tmem_loaded(v[k]);
                put_state(k, v[k], dec);
            }
            fence_async_smem();
        }
        // ---- e^{G_i} C S^T + D x (elements that are not finite, zero by now, make no difference: their rows become NaN)
        nb_sync<CC>(C_Y);
        tc_fence_after();
        {
            const F2 r = f2(ex2(Gi + t.between[q][q]));
            float yv[2][16];
            tmem_ld16_issue(yv[0], tl + TM_Y + 64 * hd + 32 * half);
            tmem_ld16_issue(yv[1], tl + TM_Y + 64 * hd + 32 * half + 16);
            tmem_wait_ld();
            tmem_loaded(yv[0]);
            tmem_loaded(yv[1]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float (&y)[16] = yv[k];
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const uint4 x = *reinterpret_cast<const uint4*>(s.x[hd] + (at0 ^ ((2 * k + v) << 4)));
                    const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float& lo = y[8 * v + 2 * e];
                        float& hi = y[8 * v + 2 * e + 1];
                        f2_get(fma2(Dh, unpack2(xw[e]), mul2(f2(lo, hi), r)), lo, hi);
                    }
                }
                tm_st16(tl + TM_Y + 64 * hd + 32 * half + 16 * k, reinterpret_cast<const uint32_t (&)[16]>(y));
            }
        }
        tm_wait_st();
        tc_fence_before();
        fence_async_smem();                       // (zeroed elements of x)
        nb_arrive<CC>(C_P);
        // ---- gate, of the first half of the columns while the products run
        F2 gate[16];
        auto gates = [&](int k) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                uint32_t zw[4];
                if (a.z_vec) {
                    const uint4 z = *reinterpret_cast<const uint4*>(s.z[hd] + (at0 ^ ((2 * k + v) << 4)));
                    zw[0] = z.x; zw[1] = z.y; zw[2] = z.z; zw[3] = z.w;
                } else {                          // rows that do not begin on 16-byte boundaries
                    const int p = slab + 32 * half + 16 * k + 8 * v;
                    const uint16_t* src = (const uint16_t*)a.z + (u.t0 + (int64_t)c * UQ + row) * a.z_tok + h * a.z_head + p;
#pragma unroll
                    for (int e = 0; e < 4; ++e) zw[e] = has && row < n && p < a.P ? (uint32_t)__ldg(src + 2 * e) | (uint32_t)__ldg(src + 2 * e + 1) << 16 : 0u;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) gate[8 * k + 4 * v + e] = silu2(unpack2(zw[e]));
            }
        };
        if (a.z) { gates(0); gates(1); }
        // ---- output, into z's place
        nb_sync<CC>(C_PX);
        tc_fence_after();
        uint32_t o[16];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float y[16];
            tmem_ld16(y, tl + TM_Y + 64 * hd + 32 * half + 16 * k);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                F2 v = f2(y[2 * e], y[2 * e + 1]);
                if (a.z) v = mul2(v, gate[8 * k + e]);
                o[8 * k + e] = pack2(v);
            }
        }
        tm_wait_st();
        tc_fence_before();
        if (!last) nb_arrive<CC>(C_YF);           // the next chunk's Y may come
        if (s.any_bad[hd])
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if (row >= s.bad[hd][32 * half + e]) o[e >> 1] = (o[e >> 1] & (e & 1 ? 0xffffu : 0xffff0000u)) | (e & 1 ? 0x7fc00000u : 0x7fc0u);
        unsigned char* const stage = s.z[hd];
#pragma unroll
        for (int v = 0; v < 4; ++v) *reinterpret_cast<uint4*>(stage + (at0 ^ (v << 4))) = make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
        fence_async_smem();
        if (!last) continue;                      // (stored by the warp that issues the products)
        __syncwarp();
        {                                         // rows r and r + 4 together: their pieces lie in different banks
            const int r0 = 32 * q + ((lane >> 3) & 3) + (lane & 4), c16 = 4 * half + (lane & 3);
            const unsigned char* src = stage + swz(r0, c16);
            __nv_bfloat16* dst = (__nv_bfloat16*)a.y + ((u.t0 + (int64_t)c * UQ + r0) * a.H + h) * a.P + slab + c16 * 8;
            const int left = has && slab + c16 * 8 < a.P ? n - r0 : 0;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (8 * k < left) *reinterpret_cast<uint4*>(dst + (int64_t)(8 * k) * a.H * a.P) = *reinterpret_cast<const uint4*>(src + 1024 * k);
        }
    }
    tc_fence_before();
    nb_sync<ALL>(0);
}

// [n_tok][heads][cols] with the given distances (elements) as boxes of 64 columns of one head and 128 tokens; columns beyond the head's
// read as zero
bool make_map3(CUtensorMap* m, const void* base, int64_t n_tok, int heads, int cols, int64_t tok, int64_t head) {
    PFN_cuTensorMapEncodeTiled enc = tensor_map_encoder();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)heads, (cuuint64_t)n_tok};
    const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? head : 8) * 2, (cuuint64_t)(n_tok > 1 ? tok : 8) * 2};     // (those of one row are not used)
    const cuuint32_t box[3] = {64, 1, UQ}, estr[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NPAN>
int launch_pan(const SsmArgs& a, const Maps& maps, int units, bool blocks, cudaStream_t st) {
    static std::atomic<uint64_t> ready_s{0}, ready_1{0}, ready_o{0};
    static_assert(sizeof(SmA) <= MAX_SMEM && sizeof(SmC<NPAN>) <= MAX_SMEM, "tiles fit");
    const dim3 grid(units, (unsigned)(a.G * ((a.H / a.G + 1) / 2)), (a.P + 63) / 64);
    if (blocks || a.ht) {
        const auto kernel = a.ht ? ssm_state_umma_kernel<NPAN, 3> : ssm_state_umma_kernel<NPAN, 1>;
        if (!allow_smem(a.ht ? ready_s : ready_1, kernel, (int)sizeof(SmA))) return LAMPA_ERR_CUDA;
        {
            ProfScope prof("ssm_state", st);
            if (launch_chained(kernel, grid, dim3(THREADS), sizeof(SmA), st, a, maps) != cudaSuccess) return LAMPA_ERR_CUDA;
        }
    }
    if (blocks || (a.cu && a.ht)) {
        const int rc = launch_ssm_pass(a, st);
        if (rc != LAMPA_OK) return rc;
    }
    if (!allow_smem(ready_o, ssm_out_umma_kernel<NPAN>, (int)sizeof(SmC<NPAN>))) return LAMPA_ERR_CUDA;
    ProfScope prof("ssm_out", st);
    return launch_chained(ssm_out_umma_kernel<NPAN>, grid, dim3(THREADS), sizeof(SmC<NPAN>), st, a, maps) == cudaSuccess ? LAMPA_OK : LAMPA_ERR_CUDA;
}

}  // namespace

int launch_ssm_scan_umma(SsmArgs a, int units, bool blocks, cudaStream_t st) {
    Maps maps;
    if (!make_map3(&maps.x, a.x, a.n_tok, a.H, a.P, a.x_tok, a.x_head) || !make_map3(&maps.B, a.B, a.n_tok, a.G, a.N, a.b_tok, a.b_grp) ||
        !make_map3(&maps.C, a.C, a.n_tok, a.G, a.N, a.c_tok, a.c_grp)) return LAMPA_ERR_CUDA;
    maps.z = maps.x;
    if (!make_map3(&maps.y, a.y, a.n_tok, a.H, a.P, (int64_t)a.H * a.P, a.P)) return LAMPA_ERR_CUDA;
    a.z_vec = a.z_vec && make_map3(&maps.z, a.z, a.n_tok, a.H, a.P, a.z_tok, a.z_head);
    return a.N <= 64 ? launch_pan<1>(a, maps, units, blocks, st) : launch_pan<2>(a, maps, units, blocks, st);
}

}  // namespace lampa
