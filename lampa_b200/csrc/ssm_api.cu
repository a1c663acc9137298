// C entry point of the selective state space scan: checks, block length, workspace and the choice of kernels.
#include "profile.cuh"
#include "ssm.cuh"

#include <algorithm>

namespace lampa {
namespace {

bool desc_ok(const lampa_ssm_desc* d) {
    return d && d->B >= 0 && d->T >= 0 && d->H > 0 && d->P > 0 && d->N > 0 && d->G > 0 && d->H % d->G == 0 && d->nseq >= 0 &&
           !(d->nseq && d->B != 1) && d->dt_dtype >= LAMPA_BF16 && d->dt_dtype <= LAMPA_F32;
}
bool built(const lampa_ssm_desc* d) {
    return (d->dtype == LAMPA_BF16 || d->dtype == LAMPA_F16) && d->N <= 256 && d->H <= 65535 && d->P <= 65535;
}

// The tcgen05 kernels take bf16 rows in pieces of 16 bytes, and their state is one operand tile.  A single chunk is one launch of the mma.sync
// form that ends with the state (64 tokens, 8 heads of 64 x 64: 10.6 us, tcgen05 in two launches 16; 256 such prompts: 80 and 108; 128 tokens:
// 19.6 and 14.9).
bool umma_shape(const lampa_ssm_desc* d) { return d->dtype == LAMPA_BF16 && d->P % 8 == 0 && d->N % 8 == 0 && d->N <= 128 && d->T > SSM_Q; }

// Tokens per block: enough blocks for eight CTAs to an SM in the mma.sync form (24 001 packed tokens in fp16, 6 heads of 32 x 16: with eight 68 us,
// six 80, four 71, two 98, when these were compared), for one CTA (of two heads) to an SM in the tcgen05 form, where a second round of CTAs costs as much as the first.
// Sequences of one length are cut into equally many blocks (four of 2 049 tokens, 8 pairs of heads: 49 us, when these were compared; by all tokens, 160 CTAs, 60); of a packed batch's, each may end in one that is not whole.
int block_tokens(const lampa_ssm_desc* d, bool umma) {
    const int q = umma ? 128 : SSM_Q;
    const int64_t slabs = (d->P + 63) / 64, per = umma ? (int64_t)d->G * ((d->H / d->G + 1) / 2) * slabs : d->H * slabs;
    const int64_t all = (umma ? 1 : 8) * (int64_t)sm_count() / per;
    const int64_t chunks = ((int64_t)d->T + q - 1) / q;            // of a sequence, or of all of them
    const int64_t want = std::max<int64_t>(1, d->nseq ? std::max(all / 4, all - d->nseq) : all / d->B);
    return (int)std::min<int64_t>(1 << 20, std::max<int64_t>(1, (chunks + want - 1) / want)) * q;
}

struct Plan { int bl, nb; int64_t units; bool blocks; size_t state_bytes, bytes; };
Plan plan_of(const lampa_ssm_desc* d, bool umma) {
    Plan p;
    const int64_t n_tok = (int64_t)d->B * d->T;
    const int nseq = d->nseq ? d->nseq : d->B;
    p.bl = block_tokens(d, umma);
    p.nb = (int)(((int64_t)d->T + p.bl - 1) / p.bl);
    p.units = ssm_units(n_tok, nseq, p.nb, p.bl, d->nseq > 0);
    p.blocks = d->T > p.bl;                                        // some sequence may have more than one
    const int64_t slots = p.blocks ? ssm_slots(n_tok, nseq, p.nb, p.bl, d->nseq > 0) : 0;
    p.state_bytes = (size_t)slots * d->H * d->P * d->N * 4;
    p.bytes = p.state_bytes + (size_t)slots * d->H * 4;
    return p;
}

}  // namespace
}  // namespace lampa

using namespace lampa;

extern "C" int lampa_ssm_workspace_bytes(const lampa_ssm_desc* d, size_t* bytes) {
    if (!desc_ok(d) || !bytes) return LAMPA_ERR_ARG;
    if (!built(d)) return LAMPA_ERR_UNSUPPORTED;
    *bytes = 0;
    if (d->B && d->T) *bytes = std::max(plan_of(d, false).bytes, umma_shape(d) ? plan_of(d, true).bytes : 0);
    return LAMPA_OK;
}

extern "C" int lampa_ssm_scan(const lampa_ssm_desc* d, const void* x, int64_t x_tok, int64_t x_head, const void* dt, int64_t dt_tok,
                              const float* A, const void* B, int64_t b_tok, int64_t b_grp, const void* C, int64_t c_tok, int64_t c_grp,
                              const float* D, const void* z, int64_t z_tok, int64_t z_head, const float* dt_bias,
                              const float* initial_state, const int64_t* cu_seqlens, void* y, float* final_state, void* ws,
                              size_t ws_bytes, int32_t* status, void* stream) {
    if (!desc_ok(d) || (cu_seqlens != nullptr) != (d->nseq > 0)) return LAMPA_ERR_ARG;
    if (!built(d)) return LAMPA_ERR_UNSUPPORTED;
    if (d->B == 0) return LAMPA_OK;
    if (d->T == 0) {                                               // no tokens: what enters the sequences is what leaves them
        if (!final_state) return LAMPA_OK;
        SsmArgs a = {};
        a.h0 = initial_state; a.ht = final_state; a.cu = cu_seqlens; a.status = status;
        a.nseq = d->nseq ? d->nseq : d->B;
        a.bl = SSM_Q; a.H = d->H; a.P = d->P; a.N = d->N;
        return launch_ssm_pass(a, (cudaStream_t)stream);
    }
    if (!x || !dt || !A || !B || !C || !y) return LAMPA_ERR_ARG;
    auto rows16 = [](const void* q, int64_t s0, int64_t s1) { return (((uintptr_t)q | (uintptr_t)(s0 * 2) | (uintptr_t)(s1 * 2)) & 15) == 0; };
    const bool vec = d->P % 8 == 0 && d->N % 8 == 0 && rows16(x, x_tok, x_head) && rows16(B, b_tok, b_grp) && rows16(C, c_tok, c_grp);
    const int64_t n_tok = (int64_t)d->B * d->T;
    auto steps_on = [&](int64_t tok, int64_t head, int n) { return (n_tok == 1 || tok > 0) && (n == 1 || head > 0); };     // (a tensor map has no zero distances)
    const bool umma = umma_shape(d) && n_tok <= INT32_MAX - 128 && vec && ((uintptr_t)y & 15) == 0 && umma_enabled() &&
                      steps_on(x_tok, x_head, d->H) && steps_on(b_tok, b_grp, d->G) && steps_on(c_tok, c_grp, d->G);
    const Plan p = plan_of(d, umma);
    if (p.units > INT32_MAX) return LAMPA_ERR_UNSUPPORTED;
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 15))) return LAMPA_ERR_WORKSPACE;
    SsmArgs a = {};
    a.x = x; a.dt = dt; a.B = B; a.C = C; a.z = z;
    a.A = A; a.D = D; a.dt_bias = dt_bias; a.h0 = initial_state; a.cu = cu_seqlens;
    a.y = y; a.ht = final_state;
    a.blk = (float*)ws; a.blk_dec = (float*)((char*)ws + p.state_bytes);
    a.status = status;
    a.x_tok = x_tok; a.x_head = x_head; a.z_tok = z_tok; a.z_head = z_head; a.b_tok = b_tok; a.b_grp = b_grp; a.c_tok = c_tok; a.c_grp = c_grp;
    a.dt_tok = dt_tok;
    a.n_tok = n_tok; a.T = d->T; a.nseq = d->nseq ? d->nseq : d->B; a.nb = p.nb; a.bl = p.bl;
    a.H = d->H; a.P = d->P; a.N = d->N; a.G = d->G; a.dt_dt = d->dt_dtype; a.softplus = d->dt_softplus;
    a.vec = vec;
    a.z_vec = z && rows16(z, z_tok, z_head) && steps_on(z_tok, z_head, d->H);
    a.z_pair = z && d->P % 2 == 0 && (((uintptr_t)z | (uintptr_t)(z_tok * 2) | (uintptr_t)(z_head * 2)) & 3) == 0;
    a.y_pair = d->P % 2 == 0 && ((uintptr_t)y & 3) == 0;
    a.poll_budget = poll_budget();
    a.poll_budget_products = poll_budget_products();
    return umma ? launch_ssm_scan_umma(a, (int)p.units, p.blocks, (cudaStream_t)stream) : launch_ssm_scan_mma(a, d->dtype, (int)p.units, p.blocks, (cudaStream_t)stream);
}
