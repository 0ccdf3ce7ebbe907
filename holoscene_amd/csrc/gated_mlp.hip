// holoscene_amd/csrc/gated_mlp.hip -- entry points of the gated feed-forward block (gated_mlp.h).
#include "gated_mlp.h"

namespace {

// an activation, and for the 16-bit types one of the flags at most
bool activation_ok(const hsGatedMlp &a) {
    const int32_t planes = a.activation & ~0xff;
    return (a.activation & 0xff) <= HS_ACT_RELU && (planes == 0 || (a.dtype != HS_F32 && (planes == HS_GATED_ONE_PLANE || planes == HS_GATED_TWO_PLANES)));
}

bool sizes_ok(const hsGatedMlp &a) {
    return a.rows > 0 && a.dim > 0 && a.hidden > 0 && a.rows <= HS_GATED_MLP_MAX_ROWS && a.dim <= HS_GATED_MLP_MAX && a.hidden <= HS_GATED_MLP_MAX && a.ldx >= a.dim && a.ld_gate >= a.dim &&
           a.ld_up >= a.dim && a.ld_down >= a.hidden && hs_row::known_dtype(a.dtype) && activation_ok(a);
}

int64_t call(const hsGatedMlp &a, int what, hipStream_t s) {
    if (a.dtype == HS_BF16) return hs_gemm::gated_mlp_bf16(a, what, s);
    if (a.dtype == HS_F16) return hs_gemm::gated_mlp_f16(a, what, s);
    return hs_gemm::gated_mlp_f32(a, what, s);
}

}  // namespace

extern "C" {

int64_t hs_gated_mlp_saved_bytes(const hsGatedMlp *a) { return !a ? HS_ERR_NULL : sizes_ok(*a) ? call(*a, 4, nullptr) : HS_ERR_ARG; }
int64_t hs_gated_mlp_fwd_ws_bytes(const hsGatedMlp *a) { return !a ? HS_ERR_NULL : sizes_ok(*a) ? call(*a, 2, nullptr) : HS_ERR_ARG; }
int64_t hs_gated_mlp_bwd_ws_bytes(const hsGatedMlp *a) { return !a ? HS_ERR_NULL : sizes_ok(*a) ? call(*a, 3, nullptr) : HS_ERR_ARG; }

int hs_gated_mlp_fwd(const hsGatedMlp *a, void *stream) {
    if (!a) return HS_ERR_NULL;
    if (!sizes_ok(*a)) return HS_ERR_ARG;
    if (!a->x || !a->w_gate || !a->w_up || !a->w_down || !a->y) return HS_ERR_NULL;
    const int64_t need = call(*a, 2, nullptr);
    if (need > 0 && !a->ws) return HS_ERR_NULL;
    if (a->ws_bytes < need) return HS_ERR_ARG;
    return (int)call(*a, 0, (hipStream_t)stream);
}

int hs_gated_mlp_bwd(const hsGatedMlp *a, void *stream) {
    if (!a) return HS_ERR_NULL;
    if (!sizes_ok(*a) || a->ld_grad < a->dim) return HS_ERR_ARG;
    if (!a->x || !a->w_gate || !a->w_up || !a->w_down || !a->grad || !a->saved) return HS_ERR_NULL;
    const int64_t need = call(*a, 3, nullptr);
    if (need > 0 && !a->ws) return HS_ERR_NULL;
    if (a->ws_bytes < need) return HS_ERR_ARG;
    return (int)call(*a, 1, (hipStream_t)stream);
}

}  // extern "C"
