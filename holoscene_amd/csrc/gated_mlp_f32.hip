// holoscene_amd/csrc/gated_mlp_f32.hip -- the gated feed-forward block (gated_mlp.h) for fp32 (three bf16 planes per operand).
#include "gated_mlp.h"

int64_t hs_gemm::gated_mlp_f32(const hsGatedMlp &a, int what, hipStream_t s) { return block_call<hs_row::bf16_t, float>(a, what, s); }
