// Selective state space scan on the 5th-generation tensor cores: bf16, head dims and state sizes that are multiples of 8, N up to 128.
//
// The algebra is ssm_scan.cu's with chunks of 128 tokens.  One CTA takes a block of chunks for TWO heads of a group, which share C, B and
// their scores.  Per chunk (heads a, b side by side in the columns; [token][column] bf16 tiles with 128-byte rows and swizzle, 64
// columns to a panel, serve as either operand of every product):
//   G   = C B^T                   128 x 128, K = N                        scores
//   Y   = C [S_a^T | S_b^T]       128 x 128, K = N                        what the entering states give; scaled by e^{G_i} in place
//   dS  = B^T [wx_a | wx_b]       N x 128,   K = 128 tokens               what the chunk adds to the states
//   Y_h += P_h x_h                128 x 64 each, K = 128                  P_h: masked, decayed scores, bf16, from tensor memory
// All accumulators are in tensor memory (G | P | Y | dS, 128 columns each).  The states stay in registers in fp32.
//
// Sixteen warps do the element work, thread = (row or state row, head, half of the 64 columns); a control warp issues the products and is
// the only one that polls mbarriers: it passes completions on through hardware named barriers (30 cycles, where a poll costs 200 - 300).
// Its waits are bounded and it walks through all barriers whether or not one ran out, so nobody can be left waiting.
#include "profile.cuh"
#include "ssm.cuh"
#include "umma.cuh"

#include <algorithm>

namespace lampa {
namespace {

constexpr int UQ = 128;                           // tokens per chunk
constexpr int CWARPS = 16, CT = CWARPS * 32;      // element warps
constexpr int THREADS = CT + 32;
constexpr int TILE = 16384;                       // [128][64] bf16
constexpr float LOG2E = 1.4426950408889634f;

// tensor-memory columns
constexpr int TM_G = 0, TM_P = 128, TM_Y = 256, TM_S = 384;

__device__ __forceinline__ void nb_sync(int id) { asm volatile("bar.sync %0, %1;\n" :: "r"(id), "n"(THREADS) : "memory"); }
__device__ __forceinline__ void nb_arrive(int id) { asm volatile("bar.arrive %0, %1;\n" :: "r"(id), "n"(THREADS) : "memory"); }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" :: "r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_all;\n" ::: "memory"); }
__device__ __forceinline__ uint64_t adv(uint64_t d, uint32_t bytes) { return d + (uint64_t)(bytes >> 4); }
__device__ __forceinline__ int swz(int r, int c16) { return r * 128 + ((c16 ^ (r & 7)) << 4); }

// Per head and chunk, by token: G (log2), d, d e^{G_end(32-block) - G}, d e^{G_last - G}
struct Tab { float G[UQ], d[UQ], cf[UQ], w[UQ]; };

// One warp, four tokens to a lane.  Returns log2 of the chunk's decay.  The exponent of w is summed from the chunk's end, so
// that its error is one of its own size.
__device__ __forceinline__ void raw_steps(const SsmArgs& a, int64_t t, int64_t t1, int h, bool has, float (&v)[4]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t i = t + 4 * lane + k;
        v[k] = has && i < t1 ? load_as_float(a.dt, (size_t)(i * a.dt_tok + h), a.dt_dt) : 0.f;
    }
}
template <bool FULL>
__device__ __forceinline__ float make_tab(const SsmArgs& a, float* ws, Tab* s, const float (&raw)[4], int n, float A2, float bias) {
    const int l = threadIdx.x & 31;
    float d[4], g[4], up = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        d[k] = 4 * l + k < n ? ssm_step_size(raw[k] + bias, a.softplus) : 0.f;
        g[k] = 4 * l + k < n ? d[k] * A2 : 0.f;
        up += g[k];
    }
    float down = up;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float u = __shfl_up_sync(0xffffffffu, up, o), v = __shfl_down_sync(0xffffffffu, down, o);
        if (l >= o) up += u;
        if (l + o < 32) down += v;
    }
    const float before = __shfl_up_sync(0xffffffffu, up, 1), after = __shfl_down_sync(0xffffffffu, down, 1);
    float e = l < 31 ? after : 0.f, w[4];
#pragma unroll
    for (int k = 3; k >= 0; --k) { w[k] = d[k] * exp2f(e); e += g[k]; }
    *reinterpret_cast<float4*>(ws + 4 * l) = make_float4(w[0], w[1], w[2], w[3]);
    if (FULL) {
        float G[4], b = l ? before : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) { b += g[k]; G[k] = b; }
        const float end = __shfl_sync(0xffffffffu, G[3], l | 7);
        *reinterpret_cast<float4*>(&s->G[4 * l]) = make_float4(G[0], G[1], G[2], G[3]);
        *reinterpret_cast<float4*>(&s->d[4 * l]) = make_float4(d[0], d[1], d[2], d[3]);
        *reinterpret_cast<float4*>(&s->cf[4 * l]) = make_float4(d[0] * ex2(end - G[0]), d[1] * ex2(end - G[1]), d[2] * ex2(end - G[2]), d[3] * ex2(end - G[3]));
    }
    return __shfl_sync(0xffffffffu, up, 31);
}

// [128] rows of PAN * 64 columns into PAN panels, zero beyond n rows and `cols` columns; by the element warps
template <int PAN>
__device__ __forceinline__ void load_panels(uint32_t dst, const void* base, int64_t off, int64_t pitch, int n, int cols, bool twice) {
    const __nv_bfloat16* src = (const __nv_bfloat16*)base + off;
#pragma unroll
    for (int k = 0; k < UQ * 8 * PAN / CT; ++k) {
        const int i = threadIdx.x + CT * k, r = i / (8 * PAN), c = i % (8 * PAN);
        const bool ok = r < n && c * 8 < cols;
        const uint32_t at = dst + (c >> 3) * TILE + swz(r, c & 7);
        const void* p = ok ? src + (int64_t)r * pitch + c * 8 : src;
        cp16(at, p, ok);
        if (PAN == 1 && twice) cp16(at + TILE, p, ok);
    }
}

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
__device__ __forceinline__ void tm_st32f(uint32_t t, const float (&x)[32]) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(x);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n"
                 :: "r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                    "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
                    "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
                    "r"(r[30]), "r"(r[31]) : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}

// -------------------------------------------------------------------------------------------------
// What a block makes of an empty state.  Its products take d x e^{..} in three bf16 pieces where somebody will see the state (24 bits), in one
// where only y will.  Every chunk's sum starts from zero and is added to the states in fp32 arithmetic.
// -------------------------------------------------------------------------------------------------
enum { A_W0 = 1, A_W1, A_F0, A_F1 };
template <int NPAN>
struct SmA {
    unsigned char wx[2][3][2][TILE / 2];          // [half of the tokens][piece][head]
    unsigned char B[2][2][TILE];                  // [chunk parity][panel]
    float w[2][2][UQ];                            // [chunk parity][head]
    float tot[4][2];
    uint64_t bar[2], drain;
    uint32_t tslot;
};

template <int NPAN>
__global__ void __launch_bounds__(THREADS, 1) ssm_state_umma_kernel(SsmArgs a) {
    if (chain_wait()) return;
    extern __shared__ __align__(1024) unsigned char raw[];
    SmA<NPAN>& s = *reinterpret_cast<SmA<NPAN>*>(raw);
    SsmUnit u;
    if (!ssm_unit(a, blockIdx.x, u) || u.outside || (u.single(a.bl) && !a.ht)) return;
    const int hpg = a.H / a.G, pairs = (hpg + 1) / 2, grp = blockIdx.y / pairs, hl = 2 * (blockIdx.y % pairs), slab = blockIdx.z * 64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunks = (int)((u.t1 - u.t0 + UQ - 1) / UQ), pieces = a.ht ? 3 : 1;
    if (warp == CWARPS) {
        if (lane == 0) {
            mbar_init(&s.bar[0], 1); mbar_init(&s.bar[1], 1); mbar_init(&s.drain, 1);
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&s.tslot, 256);
    }
    tc_fence_before();
    nb_sync(0);
    tc_fence_after();
    const uint32_t tm = s.tslot;

    if (warp == CWARPS) {
        bool dead = false;
        constexpr uint32_t id = umma_idesc(128, 128, 1, 1);
        for (int c = 0; c < chunks; ++c)
#pragma unroll 1
            for (int hf = 0; hf < 2; ++hf) {
                if (c > 0) {                      // the tokens' half that was there before has been taken in
                    if (lane == 0) mbar_wait(&s.bar[hf], (c - 1) & 1, dead, a.status, 53, a.poll_budget);
                    __syncwarp();
                    nb_arrive(A_F0 + hf);
                }
                nb_sync(A_W0 + hf);
                if (lane == 0) {
                    tc_fence_after();
                    const uint64_t da = umma_desc_mn128(smem_u32(s.B[c & 1][0]) + hf * (TILE / 2), TILE);
                    for (int p = pieces - 1; p >= 0; --p) {
                        const uint64_t db = umma_desc_mn128(smem_u32(s.wx[hf][p][0]), TILE / 2);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f16_ss(tm + 128 * (c & 1), adv(da, 2048 * k), adv(db, 2048 * k), id, hf || p < pieces - 1 || k);
                    }
                    umma_commit(&s.bar[hf]);
                }
                __syncwarp();
            }
        if (lane == 0) {
            umma_commit(&s.drain);
            if (!mbar_drain(&s.drain, 0)) set_status(a.status, LAMPA_ERR_TIMEOUT, 53, 0);
        }
        __syncwarp();
        nb_arrive(A_F0);
        nb_sync(0);
        tmem_dealloc(tm, 256);
        return;
    }

    const int q = warp & 3, hd = warp >> 3, half = (warp >> 2) & 1;
    const Own<NPAN> own(q, half, lane);
    constexpr int PC = Own<NPAN>::PC;
    const int h0 = grp * hpg + hl;
    const bool step_warp = q == 0 && half == 1;   // of its head
    const bool has = hl + hd < hpg;
    float A2 = 0.f, bias = 0.f, dt[4], log_dec = 0.f;
    if (step_warp && has) { A2 = a.A[h0 + hd] * LOG2E; bias = a.dt_bias ? a.dt_bias[h0 + hd] : 0.f; }
    auto tab = [&](int c) {
        const float g = make_tab<false>(a, s.w[c & 1][hd], nullptr, dt, (int)min((int64_t)UQ, u.t1 - (u.t0 + (int64_t)c * UQ)), A2, bias);
        if (lane == 0) s.tot[c & 3][hd] = exp2f(g);
        log_dec += g;
    };
    // x of a half chunk: 16 bytes of (head, row, 8 columns), two per thread
    uint4 xr[2][2];
    auto load_x = [&](int c, int hf) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = threadIdx.x + CT * k, col = i & 7, r = 64 * hf + ((i >> 3) & 63), xh = k;
            const int64_t t = u.t0 + (int64_t)c * UQ + r;
            const bool ok = c < chunks && t < u.t1 && hl + xh < hpg && slab + col * 8 < a.P;
            xr[hf][k] = ok ? __ldg(reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.x + t * a.x_tok + (h0 + xh) * a.x_head + slab + col * 8)) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    auto load_B = [&](int c) {
        const int64_t t = u.t0 + (int64_t)c * UQ;
        load_panels<NPAN>(smem_u32(s.B[c & 1][0]), a.B, t * a.b_tok + grp * a.b_grp, a.b_tok, (int)min((int64_t)UQ, u.t1 - t), a.N, true);
    };
    load_B(0);
    load_x(0, 0);
    load_x(0, 1);
    if (step_warp) {
        raw_steps(a, u.t0, u.t1, h0 + hd, has, dt);
        tab(0);
        raw_steps(a, u.t0 + UQ, u.t1, h0 + hd, has, dt);
    }
    asm volatile("bar.sync 5, 512;\n" ::: "memory");           // element warps: the first steps are there
    float st[PC];
#pragma unroll
    for (int i = 0; i < PC; ++i) st[i] = 0.f;
    auto take_in = [&](int c) {                   // states <- decay * states + dS of chunk c
        float ds[PC];
        tm_ld<PC>(ds, tm + ((uint32_t)(32 * q) << 16) + 128 * (c & 1) + 64 * hd + own.p0);
        const float dec = s.tot[c & 3][hd];
#pragma unroll
        for (int i = 0; i < PC; ++i) st[i] = fmaf(dec, st[i], ds[i]);
    };
    for (int c = 0; c < chunks; ++c) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if (c > 0) nb_sync(A_F0 + hf);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int i = threadIdx.x + CT * k, col = i & 7, r = (i >> 3) & 63;
                const float w = s.w[c & 1][k][64 * hf + r];
                const uint32_t src[4] = {xr[hf][k].x, xr[hf][k].y, xr[hf][k].z, xr[hf][k].w};
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = unpack_bf16x2(src[e]);
                    v[2 * e] = f.x * w; v[2 * e + 1] = f.y * w;
                }
                for (int p = 0; p < pieces; ++p) {
                    uint32_t o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
                        const float2 f = unpack_bf16x2(o[e]);
                        v[2 * e] -= f.x; v[2 * e + 1] -= f.y;
                    }
                    *reinterpret_cast<uint4*>(s.wx[hf][p][k] + swz(r, col)) = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
            load_x(c + 1, hf);
            if (hf == 0) cp_wait();               // B of this chunk
            fence_async_smem();
            tc_fence_before();
            nb_arrive(A_W0 + hf);
            if (hf == 0 && step_warp && c + 1 < chunks) {      // (nobody reads the weights of chunk c - 1 any more)
                tab(c + 1);
                raw_steps(a, u.t0 + (int64_t)(c + 2) * UQ, u.t1, h0 + hd, has, dt);
            }
        }
        if (c > 0) { tc_fence_after(); take_in(c - 1); }
        if (c + 1 < chunks) load_B(c + 1);        // the products of chunk c - 1, which read this buffer, are complete
    }
    nb_sync(A_F0);
    tc_fence_after();
    take_in(chunks - 1);
    float* const out = a.blk + ((int64_t)blockIdx.x * a.H + h0 + hd) * a.P * a.N;
    if (has && own.n < a.N)
#pragma unroll
        for (int i = 0; i < PC; ++i)
            if (slab + own.p0 + i < a.P) out[(int64_t)(slab + own.p0 + i) * a.N + own.n] = st[i];
    if (step_warp && has && lane == 0 && slab == 0) a.blk_dec[(int64_t)blockIdx.x * a.H + h0 + hd] = log_dec;
    tc_fence_before();
    nb_sync(0);
}

// -------------------------------------------------------------------------------------------------
// The output, walking through a block from the state that enters it.
// -------------------------------------------------------------------------------------------------
enum { C_WX = 1, C_G, C_Y, C_P, C_DS, C_PX, C_NEXT };
template <int NPAN>
struct SmC {
    unsigned char C[NPAN][TILE], B[2][TILE], x[2][TILE], wx[2][TILE], z[2][TILE], S[2][NPAN * TILE / 2];
    Tab tab[2][2];                                // [chunk parity][head]
    float tot[2][2];
    int bad[2][64];                               // first row of the column that is not finite, or UQ
    uint64_t g, y, ds, px, drain;
    uint32_t tslot;
};

template <int NPAN>
__global__ void __launch_bounds__(THREADS, 1) ssm_out_umma_kernel(SsmArgs a) {
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
    if (warp == CWARPS) {
        if (lane == 0) {
            mbar_init(&s.g, 1); mbar_init(&s.y, 1); mbar_init(&s.ds, 1); mbar_init(&s.px, 1); mbar_init(&s.drain, 1);
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&s.tslot, 512);
    }
    tc_fence_before();
    nb_sync(0);
    tc_fence_after();
    const uint32_t tm = s.tslot;

    if (warp == CWARPS) {
        bool dead = false;
        const uint64_t dC = umma_desc_k128(smem_u32(s.C[0])), dBk = umma_desc_k128(smem_u32(s.B[0])), dBm = umma_desc_mn128(smem_u32(s.B[0]), TILE),
                       dS = umma_desc_mn128(smem_u32(s.S[0]), NPAN * TILE / 2), dW = umma_desc_mn128(smem_u32(s.wx[0]), TILE),
                       dX0 = umma_desc_mn128(smem_u32(s.x[0])), dX1 = umma_desc_mn128(smem_u32(s.x[1]));
        for (int c = 0; c < chunks; ++c) {
            const bool last = c + 1 == chunks;
            nb_sync(C_NEXT);                      // tiles and states are there
            if (lane == 0) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 4 * NPAN; ++k) {
                    const uint32_t at = (k >> 2) * TILE + (k & 3) * 32;
                    umma_f16_ss(tm + TM_G, adv(dC, at), adv(dBk, at), umma_idesc(128, 128, 0, 0), k > 0);
                }
                umma_commit(&s.g);
#pragma unroll
                for (int k = 0; k < 4 * NPAN; ++k)
                    umma_f16_ss(tm + TM_Y, adv(dC, (k >> 2) * TILE + (k & 3) * 32), adv(dS, 2048 * k), umma_idesc(128, 128, 0, 1), k > 0);
                umma_commit(&s.y);
            }
            __syncwarp();
            nb_sync(C_WX);
            if (lane == 0 && !last) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 8; ++k) umma_f16_ss(tm + TM_S, adv(dBm, 2048 * k), adv(dW, 2048 * k), umma_idesc(128, 128, 1, 1), k > 0);
                umma_commit(&s.ds);
            }
            __syncwarp();
            if (lane == 0) mbar_wait(&s.g, c & 1, dead, a.status, 54, a.poll_budget);
            __syncwarp();
            tc_fence_before();
            nb_arrive(C_G);
            if (lane == 0) mbar_wait(&s.y, c & 1, dead, a.status, 54, a.poll_budget);
            __syncwarp();
            tc_fence_before();
            nb_arrive(C_Y);
            nb_sync(C_P);
            if (lane == 0) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 8; ++k) umma_f16_ts(tm + TM_Y, tm + TM_P + 8 * k, adv(dX0, 2048 * k), umma_idesc(128, 64, 0, 1), 1);
#pragma unroll
                for (int k = 0; k < 8; ++k) umma_f16_ts(tm + TM_Y + 64, tm + TM_P + 64 + 8 * k, adv(dX1, 2048 * k), umma_idesc(128, 64, 0, 1), 1);
                umma_commit(&s.px);
            }
            __syncwarp();
            if (!last) {
                if (lane == 0) mbar_wait(&s.ds, c & 1, dead, a.status, 54, a.poll_budget);
                __syncwarp();
                tc_fence_before();
                nb_arrive(C_DS);
            }
            if (lane == 0) mbar_wait(&s.px, c & 1, dead, a.status, 54, a.poll_budget);
            __syncwarp();
            tc_fence_before();
            nb_arrive(C_PX);
        }
        if (lane == 0) {
            umma_commit(&s.drain);
            if (!mbar_drain(&s.drain, 0)) set_status(a.status, LAMPA_ERR_TIMEOUT, 54, 0);
        }
        __syncwarp();
        nb_sync(0);
        tmem_dealloc(tm, 512);
        return;
    }

    const int q = warp & 3, hd = warp >> 3, half = (warp >> 2) & 1, row = 32 * q + lane;
    const Own<NPAN> own(q, half, lane);
    constexpr int PC = Own<NPAN>::PC;
    const int h = h0 + hd;
    const bool has = hl + hd < hpg, step_warp = q == 0 && half == 1;
    const uint32_t tl = tm + ((uint32_t)(32 * q) << 16);
    float A2 = 0.f, bias = 0.f, dt[4];
    if (step_warp && has) { A2 = a.A[h] * LOG2E; bias = a.dt_bias ? a.dt_bias[h] : 0.f; }
    auto tab = [&](int c) {
        const float g = make_tab<true>(a, s.tab[c & 1][hd].w, &s.tab[c & 1][hd], dt, (int)min((int64_t)UQ, u.t1 - (u.t0 + (int64_t)c * UQ)), A2, bias);
        if (lane == 0) s.tot[c & 1][hd] = exp2f(g);
    };
    auto rows_of = [&](int c) { return (int)min((int64_t)UQ, u.t1 - (u.t0 + (int64_t)c * UQ)); };
    auto load_C = [&](int c) { load_panels<NPAN>(smem_u32(s.C[0]), a.C, (u.t0 + (int64_t)c * UQ) * a.c_tok + grp * a.c_grp, a.c_tok, rows_of(c), a.N, false); };
    auto load_B = [&](int c) { load_panels<NPAN>(smem_u32(s.B[0]), a.B, (u.t0 + (int64_t)c * UQ) * a.b_tok + grp * a.b_grp, a.b_tok, rows_of(c), a.N, true); };
    auto load_x = [&](int c) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            load_panels<1>(smem_u32(s.x[k]), a.x, (u.t0 + (int64_t)c * UQ) * a.x_tok + (h0 + k) * a.x_head + slab, a.x_tok, hl + k < hpg ? rows_of(c) : 0, a.P - slab, false);
    };
    // this warp's part of z: 32 rows of 64 bytes
    unsigned char* const zt = s.z[hd];
    auto load_z = [&](int c) {
        if (!a.z || !has) return;
        const int n = rows_of(c);
        const __nv_bfloat16* src = (const __nv_bfloat16*)a.z + (u.t0 + (int64_t)c * UQ) * a.z_tok + h * a.z_head + slab;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = 32 * q + 8 * k + (lane >> 2), c16 = 4 * half + (lane & 3);
            const bool ok = r < n && slab + c16 * 8 < a.P;
            if (a.z_vec) cp16(smem_u32(zt) + swz(r, c16), ok ? src + (int64_t)r * a.z_tok + c16 * 8 : src, ok);
            else {
                uint32_t w[4] = {0u, 0u, 0u, 0u};
                if (ok)
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e >> 1] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(src + (int64_t)r * a.z_tok + c16 * 8 + e)) << (16 * (e & 1));
                *reinterpret_cast<uint4*>(zt + swz(r, c16)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    };
    load_C(0);
    load_B(0);
    load_x(0);
    load_z(0);
    if (step_warp) {
        raw_steps(a, u.t0, u.t1, h, has, dt);
        tab(0);
        raw_steps(a, u.t0 + UQ, u.t1, h, has, dt);
    }
    if (threadIdx.x < 128) s.bad[threadIdx.x >> 6][threadIdx.x & 63] = UQ;
    // scores above the diagonal stay zero
    for (int b = max(q + 1, 2 * half); b < 2 * half + 2; ++b) {
        const uint32_t zero[16] = {};
        tmem_st16(tl + TM_P + 64 * hd + 16 * b, zero);
    }
    const bool single = u.single(a.bl);
    const int64_t pn = (int64_t)a.P * a.N;
    const float* enter = !has ? nullptr : single ? (a.h0 ? a.h0 + ((int64_t)u.seq * a.H + h) * pn : nullptr) : a.blk + ((int64_t)blockIdx.x * a.H + h) * pn;
    float st[PC];
#pragma unroll
    for (int i = 0; i < PC; ++i)
        st[i] = enter && own.n < a.N && slab + own.p0 + i < a.P ? enter[(int64_t)(slab + own.p0 + i) * a.N + own.n] : 0.f;
    auto put_state = [&]() {
#pragma unroll
        for (int k = 0; k < PC / 8; ++k)
            *reinterpret_cast<uint4*>(s.S[hd] + swz(own.n, own.p0 / 8 + k)) =
                make_uint4(pack_bf16x2(st[8 * k], st[8 * k + 1]), pack_bf16x2(st[8 * k + 2], st[8 * k + 3]),
                           pack_bf16x2(st[8 * k + 4], st[8 * k + 5]), pack_bf16x2(st[8 * k + 6], st[8 * k + 7]));
    };
    put_state();
    const float Dh = has && a.D ? a.D[h] : 0.f;
    cp_wait();
    fence_async_smem();
    tc_fence_before();
    nb_sync(C_NEXT);

    for (int c = 0; c < chunks; ++c) {
        const bool last = c + 1 == chunks;
        const int n = rows_of(c);
        const Tab& t = s.tab[c & 1][hd];
        // ---- wx; x stays in registers for D x
        uint32_t xr[16];
        {
            const float w = t.w[row];
            float odd = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint4 v = *reinterpret_cast<const uint4*>(s.x[hd] + swz(row, 4 * half + k));
                xr[4 * k] = v.x; xr[4 * k + 1] = v.y; xr[4 * k + 2] = v.z; xr[4 * k + 3] = v.w;
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = unpack_bf16x2(xr[4 * k + e]);
                    odd = fmaf(f.x, 0.f, odd); odd = fmaf(f.y, 0.f, odd);
                    o[e] = pack_bf16x2(f.x * w, f.y * w);
                }
                *reinterpret_cast<uint4*>(s.wx[hd] + swz(row, 4 * half + k)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
            if (odd != 0.f) {                     // NaN: some element is not finite.  It may not reach the rows above through a zero score
                for (int e = 0; e < 32; ++e) {
                    uint16_t* p = reinterpret_cast<uint16_t*>(s.x[hd] + swz(row, 4 * half + (e >> 3))) + (e & 7);
                    if ((*p & 0x7f80) == 0x7f80) { *p = 0; atomicMin(&s.bad[hd][32 * half + e], row); }
                }
            }
        }
        fence_async_smem();
        nb_arrive(C_WX);
        if (step_warp && !last) {
            tab(c + 1);
            raw_steps(a, u.t0 + (int64_t)(c + 2) * UQ, u.t1, h, has, dt);
        }
        // ---- decayed scores
        nb_sync(C_G);
        tc_fence_after();
        const float Gi = t.G[row];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int b = 2 * half + k;
            if (b > q) continue;
            float sc[32];
            tmem_ld32(sc, tl + TM_G + 32 * b);
            uint32_t o[16];
            if (b < q) {
                const float r = ex2(Gi - t.G[32 * b + 31]);
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(&t.cf[32 * b + j]);
                    o[j / 2] = pack_bf16x2(sc[j] * (f.x * r), sc[j + 1] * (f.y * r));
                    o[j / 2 + 1] = pack_bf16x2(sc[j + 2] * (f.z * r), sc[j + 3] * (f.w * r));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 g = *reinterpret_cast<const float4*>(&t.G[32 * b + j]), d = *reinterpret_cast<const float4*>(&t.d[32 * b + j]);
                    const float v0 = j <= lane ? sc[j] * (ex2(Gi - g.x) * d.x) : 0.f, v1 = j + 1 <= lane ? sc[j + 1] * (ex2(Gi - g.y) * d.y) : 0.f;
                    const float v2 = j + 2 <= lane ? sc[j + 2] * (ex2(Gi - g.z) * d.z) : 0.f, v3 = j + 3 <= lane ? sc[j + 3] * (ex2(Gi - g.w) * d.w) : 0.f;
                    o[j / 2] = pack_bf16x2(v0, v1);
                    o[j / 2 + 1] = pack_bf16x2(v2, v3);
                }
            }
            tmem_st16(tl + TM_P + 64 * hd + 16 * b, o);
        }
        // ---- e^{G_i} C S^T
        nb_sync(C_Y);
        tc_fence_after();
        if (!last) load_C(c + 1);
        {
            float y[32];
            tmem_ld32(y, tl + TM_Y + 64 * hd + 32 * half);
            const float r = ex2(Gi);
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] *= r;
            tm_st32f(tl + TM_Y + 64 * hd + 32 * half, y);
        }
        tc_fence_before();
        fence_async_smem();                       // (zeroed elements of x)
        nb_arrive(C_P);
        // ---- states
        if (!last) {
            nb_sync(C_DS);
            tc_fence_after();
            load_B(c + 1);
            float ds[PC];
            tm_ld<PC>(ds, tl + TM_S + 64 * hd + own.p0);
            const float dec = s.tot[c & 1][hd];
#pragma unroll
            for (int i = 0; i < PC; ++i) st[i] = fmaf(dec, st[i], ds[i]);
            put_state();
        }
        // ---- output
        nb_sync(C_PX);
        tc_fence_after();
        if (!last) load_x(c + 1);
        unsigned char* const stage = s.wx[hd];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float y[16];
            tmem_ld16(y, tl + TM_Y + 64 * hd + 32 * half + 16 * k);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 f = unpack_bf16x2(xr[8 * k + e]);
                y[2 * e] = fmaf(Dh, f.x, y[2 * e]);
                y[2 * e + 1] = fmaf(Dh, f.y, y[2 * e + 1]);
            }
            if (a.z) {
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const uint4 zr = *reinterpret_cast<const uint4*>(zt + swz(row, 4 * half + 2 * k + v));
                    const uint32_t zw[4] = {zr.x, zr.y, zr.z, zr.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = unpack_bf16x2(zw[e]);
                        y[8 * v + 2 * e] *= f.x * sigmoid_fast(f.x);
                        y[8 * v + 2 * e + 1] *= f.y * sigmoid_fast(f.y);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int4 bad = *reinterpret_cast<const int4*>(&s.bad[hd][32 * half + 16 * k + i]);
                if (row >= bad.x) y[i] = __int_as_float(0x7fc00000);
                if (row >= bad.y) y[i + 1] = __int_as_float(0x7fc00000);
                if (row >= bad.z) y[i + 2] = __int_as_float(0x7fc00000);
                if (row >= bad.w) y[i + 3] = __int_as_float(0x7fc00000);
            }
#pragma unroll
            for (int v = 0; v < 2; ++v)
                *reinterpret_cast<uint4*>(stage + swz(row, 4 * half + 2 * k + v)) =
                    make_uint4(pack_bf16x2(y[8 * v], y[8 * v + 1]), pack_bf16x2(y[8 * v + 2], y[8 * v + 3]),
                               pack_bf16x2(y[8 * v + 4], y[8 * v + 5]), pack_bf16x2(y[8 * v + 6], y[8 * v + 7]));
        }
        __syncwarp();
        if (has) {
            __nv_bfloat16* dst = (__nv_bfloat16*)a.y + ((u.t0 + (int64_t)c * UQ) * a.H + h) * a.P + slab;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int r = 32 * q + 8 * k + (lane >> 2), c16 = 4 * half + (lane & 3);
                if (r < n && slab + c16 * 8 < a.P)
                    *reinterpret_cast<uint4*>(dst + (int64_t)r * a.H * a.P + c16 * 8) = *reinterpret_cast<const uint4*>(stage + swz(r, c16));
            }
        }
        if (last) break;
        __syncwarp();
        load_z(c + 1);
        cp_wait();
        fence_async_smem();
        tc_fence_before();
        nb_sync(C_NEXT);
    }
    tc_fence_before();
    nb_sync(0);
}

template <int NPAN>
int launch_pan(const SsmArgs& a, int units, bool states, bool pass, cudaStream_t st) {
    static std::atomic<uint64_t> ready_s{0}, ready_o{0};
    static_assert(sizeof(SmA<NPAN>) <= MAX_SMEM && sizeof(SmC<NPAN>) <= MAX_SMEM, "tiles fit");
    const dim3 grid(units, (unsigned)(a.G * ((a.H / a.G + 1) / 2)), (a.P + 63) / 64);
    if (states) {
        if (!allow_smem(ready_s, ssm_state_umma_kernel<NPAN>, (int)sizeof(SmA<NPAN>))) return LAMPA_ERR_CUDA;
        ProfScope prof("ssm_state", st);
        if (launch_chained(ssm_state_umma_kernel<NPAN>, grid, dim3(THREADS), sizeof(SmA<NPAN>), st, a) != cudaSuccess) return LAMPA_ERR_CUDA;
    }
    if (pass) {
        const int rc = launch_ssm_pass(a, st);
        if (rc != LAMPA_OK) return rc;
    }
    if (!allow_smem(ready_o, ssm_out_umma_kernel<NPAN>, (int)sizeof(SmC<NPAN>))) return LAMPA_ERR_CUDA;
    ProfScope prof("ssm_out", st);
    return launch_chained(ssm_out_umma_kernel<NPAN>, grid, dim3(THREADS), sizeof(SmC<NPAN>), st, a) == cudaSuccess ? LAMPA_OK : LAMPA_ERR_CUDA;
}

}  // namespace

int launch_ssm_scan_umma(const SsmArgs& a, int units, bool blocks, cudaStream_t st) {
    const bool states = blocks || a.ht;
    return a.N <= 64 ? launch_pan<1>(a, units, states, states, st) : launch_pan<2>(a, units, states, states, st);
}

}  // namespace lampa
