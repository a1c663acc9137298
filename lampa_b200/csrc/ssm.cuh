// Selective state space scan: arguments and positions shared by its kernels.
//   h_t = exp(A d_t) h_{t-1} + d_t x_t B_t^T  (P x N per head),   y_t = (h_t C_t + D x_t) silu(z_t),
//   d_t = softplus(dt_t + dt_bias) or the sum itself.
#pragma once
#include "act.cuh"
#include "common.cuh"

namespace lampa {

constexpr int SSM_Q = 64;             // tokens per chunk of the mma.sync kernels

struct SsmArgs {
    const void* x; const void* dt; const void* B; const void* C; const void* z;
    const float* A; const float* D; const float* dt_bias; const float* h0;
    const int64_t* cu;
    void* y; float* ht;
    float* blk;                       // [slots][H][P][N]: end states of blocks that begin empty, then the states that enter them
    float* blk_dec;                   // [slots][H]: logarithm of a block's decay
    int32_t* status;
    int64_t x_tok, x_head, z_tok, z_head, b_tok, b_grp, c_tok, c_grp, dt_tok;   // distances in elements
    int64_t n_tok, T;                 // rows in all; tokens per sequence without cu
    int nseq;                         // sequences
    int nb;                           // blocks per sequence without cu
    int bl;                           // tokens per block
    int H, P, N, G, dt_dt, softplus;
    int vec, z_vec;                   // rows of x, B and C, or of z, are 16-byte aligned
    int z_pair, y_pair;               // two neighbours of z, or y, are one aligned word
    int poll_budget;
    int poll_budget_products;         // of the warp that issues the output pass's products (tcgen05 form)
};

// A block of tokens that one CTA walks through.  Packed sequences need no table: block b of sequence s has the number
// floor(cu[s] / bl) + s + b, which rises strictly through all blocks of all sequences in order (some numbers stay unused), so
// that a warp finds its sequence by looking at 32 offsets at a time (one round trip for up to 32 sequences).  What lies behind the last
// offset counts as one more sequence.  States are kept for the blocks of sequences that have more than one: in slots floor(2 cu[s] / bl) + b, where a
// sequence of len > bl tokens takes ceil(len / bl) <= floor(2 len / bl), so that two never meet and all lie below floor(2 n_tok / bl), however many
// sequences there are.
struct SsmUnit {
    int seq;
    int64_t bos, eos, t0, t1;         // the sequence, and this block of it
    int64_t slot;                     // of its state (sequences of several blocks)
    bool outside;                     // behind the last sequence
    __device__ __forceinline__ bool single(int bl) const { return eos - bos <= bl; }
};
__device__ __forceinline__ int64_t ssm_block_of(const SsmArgs& a, int64_t t, int bl) {            // t / bl, without a 64-bit division where there are fewer rows
    return a.n_tok <= INT32_MAX ? (int64_t)((uint32_t)min(max(t, (int64_t)0), a.n_tok) / (uint32_t)bl) : t / bl;
}
__device__ __forceinline__ bool ssm_unit(const SsmArgs& a, int u, SsmUnit& r) {           // whole warps
    int64_t b;
    if (a.cu == nullptr) {
        r.seq = u / a.nb;
        b = u - r.seq * a.nb;
        r.bos = (int64_t)r.seq * a.T;
        r.eos = r.bos + a.T;
        r.outside = false;
        r.slot = u;
    } else {
        int lo = 0, hi = a.nseq + 1;  // largest s with floor(cu[s] / bl) + s <= u
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) / 32, at = lo + (int)(threadIdx.x & 31) * step;
            const uint32_t below = __ballot_sync(0xffffffffu, at < hi && ssm_block_of(a, a.cu[min(at, hi - 1)], a.bl) + at <= u);
            if (below) lo += (31 - __clz(below)) * step;           // (the first lane's holds where the offsets are in order)
            hi = min(hi, lo + step);
        }
        r.seq = lo;
        r.outside = lo == a.nseq;
        r.bos = a.cu[lo];
        r.eos = r.outside ? a.n_tok : a.cu[lo + 1];
        if (r.bos < 0 || r.eos < r.bos || r.eos > a.n_tok) return false;      // reported by check_offsets
        b = u - (ssm_block_of(a, r.bos, a.bl) + lo);
        if (b < 0) return false;
        r.slot = ssm_block_of(a, r.bos, a.bl / 2) + b;
    }
    r.t0 = r.bos + b * a.bl;
    r.t1 = min(r.eos, r.t0 + a.bl);
    return r.t0 < r.eos;
}
inline int64_t ssm_units(int64_t n_tok, int nseq, int nb, int bl, bool packed) {
    return packed ? n_tok / bl + nseq + 1 : (int64_t)nseq * nb;
}
inline int64_t ssm_slots(int64_t n_tok, int nseq, int nb, int bl, bool packed) { return packed ? n_tok / (bl / 2) : (int64_t)nseq * nb; }

// log(1 + e^x) to fp32 rounding: the states are kept to a few parts in 10^7, and softplusf_ is good to 2e-7 of 1
__device__ __forceinline__ float ssm_step_size(float v, int softplus) {
    return softplus ? fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))) : v;
}

// Sums of exponents g = A d, of which the kernels need differences inside a chunk.  Counted from the chunk's start as one float, a token with a large
// step leaves the sum large for the rest of its chunk and rounds the small steps behind it to 2^-24 of that.  So a chunk is cut into blocks of a few
// tokens: between blocks only sums of one sign are added up (from a token to its block's end, of whole blocks, from a block's start to a
// token), each with an error of its own size; inside a block differences of sums from its start are taken, in two parts: whole numbers, which add up exactly
// (a g below SSM_CUT is cut: its exponential is zero all the same), and the rest, half at most in size.  (NaN stays NaN.)
constexpr float SSM_CUT = -128.f;
struct SsmExp { float whole, rest; };
__device__ __forceinline__ SsmExp ssm_split(float g) {
    const float c = g < SSM_CUT ? SSM_CUT : g, w = rintf(c);
    return {w, c - w};
}

int launch_ssm_pass(const SsmArgs& a, cudaStream_t st);
int launch_ssm_scan_umma(SsmArgs a, int units, bool blocks, cudaStream_t st);
int launch_ssm_scan_mma(const SsmArgs& a, int dtype, int units, bool blocks, cudaStream_t st);

}  // namespace lampa
