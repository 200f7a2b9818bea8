// How a 16-bit operand of a matrix product can be fetched by the TMA, and the kernels that do so.
#pragma once

#include <cuda.h>

#include "ffn_core.h"

namespace tmc {

// An operand of `outer` rows (m of x, n of w) and K columns: contiguous along k (mn = 0) or along
// its rows' index (mn = 1), the other dimension `stride` elements apart.
struct OperandLayout {
  int mn;
  int64_t stride;
};

// The tensor map of an operand: boxes of 64 k by `box_outer` rows (mn = 0) or 64 rows by 64 k (mn = 1),
// 128-byte swizzled.
std::string make_operand_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t outer, int64_t K,
                             const OperandLayout& l, int box_outer);

// The kernel for few rows: `rows` of x per tile, K split over `split` CTAs of a cluster; `clocks`
// estimates its time.  False where it does not apply.
struct NarrowPlan {
  int rows, split;
  double clocks;
};
bool plan_linear_narrow(const LinearProblem& p, const OperandLayout& lx, int sm_count, NarrowPlan* plan);
std::string launch_linear_narrow(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw,
                                 const NarrowPlan& plan, const LaunchCtx& ctx);

// The kernel for many rows, and an estimate of its time in clocks.
double estimate_linear_tc(const LinearProblem& p, int sm_count);
// Accumulator columns of its tiles (128, 256 or 512) and how many tiles there are.
int linear_tc_width(const LinearProblem& p, int sm_count, int64_t* tiles);
// x, w (and x2, w2) both as the layouts say; fp32 is not taken.
std::string launch_linear_tc(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw,
                             const LaunchCtx& ctx);

}  // namespace tmc
