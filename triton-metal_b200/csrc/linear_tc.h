// How a 16-bit operand of a matrix product can be fetched by the TMA, and the kernels that do so.
#pragma once

#include "ffn_core.h"

namespace tmc {

// An operand of `outer` rows (m of x, n of w) and K columns: contiguous along k (mn = 0) or along
// its rows' index (mn = 1), the other dimension `stride` elements apart.
struct OperandLayout {
  int mn;
  int64_t stride;
};

// x, w (and x2, w2) both as the layouts say; fp32 is not taken.
std::string launch_linear_tc(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw,
                             const LaunchCtx& ctx);

}  // namespace tmc
