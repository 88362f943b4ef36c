// C entry points of the gated delta rule: argument checks and launches.  No allocation, no synchronisation.
#include <math.h>

#include "gdr.cuh"

namespace kda {
namespace gdr {
cudaError_t intra(const KdaGdrParams& p, const Layout& l, cudaStream_t s);
cudaError_t fwd_state(const KdaGdrParams& p, const Layout& l, cudaStream_t s);
cudaError_t fwd_tc(const KdaGdrParams& p, const Layout& l, cudaStream_t s);
cudaError_t bwd_tc(const KdaGdrParams& p, const Layout& l, cudaStream_t s);
cudaError_t bwd_state(const KdaGdrParams& p, const Layout& l, cudaStream_t s);
cudaError_t grad(const KdaGdrParams& p, const Layout& l, cudaStream_t s);

static int sizes_ok(const KdaGdrParams& p) {
    if (p.B <= 0 || p.T <= 0 || p.H <= 0 || p.HV <= 0 || p.HV % p.H || p.N <= 0 || p.NT <= 0) return KDA_ERR_SHAPE;
    if ((p.dk != 64 && p.dk != 128) || (p.dv != 64 && p.dv != 128)) return KDA_ERR_SHAPE;
    // grids are one-dimensional, and a state panel has at least 16 of the 64 or 128 columns
    if ((long long)p.NT * p.HV > 0x7fffffffLL / 2 || (long long)p.N * p.HV > 0x7fffffffLL / 8) return KDA_ERR_SHAPE;
    return KDA_OK;
}

static int validate(const KdaGdrParams* p, bool bwd) {
    if (!p) return KDA_ERR_NULL;
    for (int t : {p->dtype, p->g_dtype})
        if (t != KDA_DTYPE_F32 && t != KDA_DTYPE_BF16) return KDA_ERR_DTYPE;
    if (const int rc = sizes_ok(*p)) return rc;
    if (p->cu_seqlens) {
        if (p->B != 1) return KDA_ERR_SHAPE;
        if (!p->chunk_seq || !p->seq_chunk_off || !p->chunk_tab) return KDA_ERR_NULL;
    } else if (p->N != p->B || (long long)p->NT != (long long)p->B * ((p->T + C - 1) / C)) {
        return KDA_ERR_SHAPE;
    }
    const bool gate = p->flags & KDA_FLAG_GATE, nosave = p->flags & KDA_FLAG_NO_SAVE;
    if (!p->q || !p->k || !p->v || !p->g || !p->beta || !p->workspace || (gate && !p->A_log) || (!bwd && !p->o)) return KDA_ERR_NULL;
    for (const void* x : {p->q, p->k, p->v, p->g, p->beta, (const void*)p->o, (const void*)p->h0, (const void*)p->ht, (const void*)p->chunk_tab})
        if ((uintptr_t)x & 15) return KDA_ERR_ALIGN;
    const Layout l = layout(*p);
    if (p->workspace_bytes < (nosave ? l.total_nosave : l.total) || ((uintptr_t)p->workspace & 255)) return KDA_ERR_WORKSPACE;
    if (!bwd) return KDA_OK;
    if (nosave) return KDA_ERR_WORKSPACE;  // the records of a forward-only call do not exist
    if (!p->grad_o || !p->grad_q || !p->grad_k || !p->grad_v || !p->grad_g || !p->grad_beta || !p->bwd_scratch) return KDA_ERR_NULL;
    if (gate && (!p->grad_A_log || (p->dt_bias && !p->grad_dt_bias))) return KDA_ERR_NULL;
    if (p->bwd_scratch_bytes < l.bwd_total || ((uintptr_t)p->bwd_scratch & 255)) return KDA_ERR_WORKSPACE;
    for (const void* x : {p->grad_o, (const void*)p->grad_q, (const void*)p->grad_k, (const void*)p->grad_v, (const void*)p->grad_g,
                          (const void*)p->grad_beta, (const void*)p->grad_ht, (const void*)p->grad_h0})
        if ((uintptr_t)x & 15) return KDA_ERR_ALIGN;
    return KDA_OK;
}
}  // namespace gdr
}  // namespace kda

using namespace kda;

extern "C" int kda_gdr_workspace_bytes(const KdaGdrParams* p, size_t* fwd_bytes, size_t* bwd_bytes) {
    if (!p) return KDA_ERR_NULL;
    if (const int rc = gdr::sizes_ok(*p)) return rc;
    const gdr::Layout l = gdr::layout(*p);
    if (fwd_bytes) *fwd_bytes = p->flags & KDA_FLAG_NO_SAVE ? l.total_nosave : l.total;
    if (bwd_bytes) *bwd_bytes = l.bwd_total;
    return KDA_OK;
}

extern "C" int kda_gdr_fwd(const KdaGdrParams* p, void* stream) {
    if (const int rc = gdr::validate(p, false)) return rc;
    const gdr::Layout l = gdr::layout(*p);
    cudaError_t e = gdr::intra(*p, l, (cudaStream_t)stream);
    if (e == cudaSuccess) e = gdr::on_tc(*p) ? gdr::fwd_tc(*p, l, (cudaStream_t)stream) : gdr::fwd_state(*p, l, (cudaStream_t)stream);
    return e == cudaSuccess ? KDA_OK : fail_cuda(e);
}

extern "C" int kda_gdr_bwd(const KdaGdrParams* p, void* stream) {
    if (const int rc = gdr::validate(p, true)) return rc;
    const gdr::Layout l = gdr::layout(*p);
    cudaError_t e = gdr::on_tc(*p) ? gdr::bwd_tc(*p, l, (cudaStream_t)stream) : gdr::bwd_state(*p, l, (cudaStream_t)stream);
    if (e == cudaSuccess) e = gdr::grad(*p, l, (cudaStream_t)stream);
    return e == cudaSuccess ? KDA_OK : fail_cuda(e);
}
