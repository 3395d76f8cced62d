// The grouped GLU feed-forward of a few rows per expert (skinny_gemm_kernel of
// moe_grouped_mlp.hip) for other sources: bf16 context rows by index, fp32 outputs. The hidden
// rows between the two products are bf16, as that kernel's operands are (2.3e-3 from float64
// where rounding the outputs to bf16 alone is 1.7e-3).
#pragma once

#include "common.hpp"

namespace koemi {

bool few_rows_mlp_fits(int64_t pairs, int64_t width, int64_t hidden, int64_t experts, int dtype);
// y [pairs, width]: the rows of the valid pairs alone are written; hidden_rows [pairs, hidden] bf16 is scratch.
int few_rows_mlp(const void* x, const int64_t* rows, int64_t tokens, const int64_t* offsets, const void* Wg, const void* bg,
                 const void* Wv, const void* bv, const void* Wo, const void* bo, void* hidden_rows, float* y, int64_t pairs,
                 int64_t width, int64_t hidden, int64_t experts, hipStream_t stream);

}  // namespace koemi
