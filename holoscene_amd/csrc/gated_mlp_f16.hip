// holoscene_amd/csrc/gated_mlp_f16.hip -- the gated feed-forward block (gated_mlp.h) for fp16.
#include "gated_mlp.h"

int64_t hs_gemm::gated_mlp_f16(const hsGatedMlp &a, int what, hipStream_t s) { return block_call<hs_row::f16_t, hs_row::f16_t>(a, what, s); }
