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

// Tokens per block: enough blocks for six CTAs to an SM.
int block_tokens(const lampa_ssm_desc* d) {
    const int64_t n_tok = (int64_t)d->B * d->T, chunks = (n_tok + SSM_Q - 1) / SSM_Q;
    const int64_t per = (int64_t)d->H * ((d->P + 63) / 64), want = std::max<int64_t>(1, 6 * sm_count() / per);
    return (int)std::min<int64_t>(1 << 20, std::max<int64_t>(2, (chunks + want - 1) / want)) * SSM_Q;
}

struct Plan { int bl, nb; int64_t units; bool blocks; size_t state_bytes, bytes; };
Plan plan_of(const lampa_ssm_desc* d) {
    Plan p;
    const int64_t n_tok = (int64_t)d->B * d->T;
    p.bl = block_tokens(d);
    p.nb = (int)(((int64_t)d->T + p.bl - 1) / p.bl);
    p.units = ssm_units(n_tok, d->nseq ? d->nseq : d->B, p.nb, p.bl, d->nseq > 0);
    p.blocks = d->T > p.bl;                                        // some sequence may have more than one
    p.state_bytes = (size_t)p.units * d->H * d->P * d->N * 4;
    p.bytes = p.blocks ? p.state_bytes + (size_t)p.units * d->H * 4 : 0;
    return p;
}

}  // namespace
}  // namespace lampa

using namespace lampa;

extern "C" int lampa_ssm_workspace_bytes(const lampa_ssm_desc* d, size_t* bytes) {
    if (!desc_ok(d) || !bytes) return LAMPA_ERR_ARG;
    if (!built(d)) return LAMPA_ERR_UNSUPPORTED;
    *bytes = d->B && d->T ? plan_of(d).bytes : 0;
    return LAMPA_OK;
}

extern "C" int lampa_ssm_scan(const lampa_ssm_desc* d, const void* x, int64_t x_tok, int64_t x_head, const void* dt, int64_t dt_tok,
                              const float* A, const void* B, int64_t b_tok, int64_t b_grp, const void* C, int64_t c_tok, int64_t c_grp,
                              const float* D, const void* z, int64_t z_tok, int64_t z_head, const float* dt_bias,
                              const float* initial_state, const int64_t* cu_seqlens, void* y, float* final_state, void* ws,
                              size_t ws_bytes, int32_t* status, void* stream) {
    if (!desc_ok(d) || (cu_seqlens != nullptr) != (d->nseq > 0)) return LAMPA_ERR_ARG;
    if (!built(d)) return LAMPA_ERR_UNSUPPORTED;
    if (d->B == 0 || d->T == 0) return LAMPA_OK;
    if (!x || !dt || !A || !B || !C || !y) return LAMPA_ERR_ARG;
    const Plan p = plan_of(d);
    if (p.units > INT32_MAX) return LAMPA_ERR_UNSUPPORTED;
    if (p.blocks && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 15))) return LAMPA_ERR_WORKSPACE;
    SsmArgs a = {};
    a.x = x; a.dt = dt; a.B = B; a.C = C; a.z = z;
    a.A = A; a.D = D; a.dt_bias = dt_bias; a.h0 = initial_state; a.cu = cu_seqlens;
    a.y = y; a.ht = final_state;
    a.blk = (float*)ws; a.blk_dec = (float*)((char*)ws + p.state_bytes);
    a.status = status;
    a.x_tok = x_tok; a.x_head = x_head; a.z_tok = z_tok; a.z_head = z_head; a.b_tok = b_tok; a.b_grp = b_grp; a.c_tok = c_tok; a.c_grp = c_grp;
    a.dt_tok = dt_tok;
    a.n_tok = (int64_t)d->B * d->T; a.T = d->T; a.nseq = d->nseq ? d->nseq : d->B; a.nb = p.nb; a.bl = p.bl;
    a.H = d->H; a.P = d->P; a.N = d->N; a.G = d->G; a.dt_dt = d->dt_dtype; a.softplus = d->dt_softplus;
    auto rows16 = [](const void* q, int64_t s0, int64_t s1) { return (((uintptr_t)q | (uintptr_t)(s0 * 2) | (uintptr_t)(s1 * 2)) & 15) == 0; };
    a.vec = d->P % 8 == 0 && d->N % 8 == 0 && rows16(x, x_tok, x_head) && rows16(B, b_tok, b_grp) && rows16(C, c_tok, c_grp);
    a.poll_budget = poll_budget();
    return launch_ssm_scan_mma(a, d->dtype, (int)p.units, p.blocks, (cudaStream_t)stream);
}
