// holoscene_amd/csrc/gated_mlp_bf16.hip -- the gated feed-forward block (gated_mlp.h) for bf16.
#include "gated_mlp.h"

int64_t hs_gemm::gated_mlp_bf16(const hsGatedMlp &a, int what, hipStream_t s) { return block_call<hs_row::bf16_t, hs_row::bf16_t>(a, what, s); }
