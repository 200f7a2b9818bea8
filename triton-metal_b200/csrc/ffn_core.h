// The feed-forward operators - linear_kernel, gated_linear_kernel, linear_sum_kernel,
// linear_pair_kernel, activation_bwd_kernel, gated_activation_bwd_kernel, residual_norm_kernel,
// residual_norm_bwd_kernel: problem descriptions and launchers.  No counterpart in the reference;
// they stand beside its matmul_kernel and attention kernels.
#pragma once

#include "tm_core.h"

namespace tmc {

enum class Act : int { None = 0, Relu = 1, Gelu = 2, GeluTanh = 3, Silu = 4, Sigmoid = 5 };
constexpr int kActCount = 6;

// The matrix products.  x [M,K] and w [K,N] have two strides each (elements); out, residual and
// the pre-activations are [M,N] with unit column stride.
enum class LinearMode : int {
  Single = 0,   // z = x w + bias; out = act(z) + residual; pre = z
  Gated = 1,    // out = act(x w) * (x w2); pre = x w, pre2 = x w2
  Sum = 2,      // out = x w + x2 w2
  Pair = 3      // out = x w, out2 = x2 w2
};
struct LinearProblem {
  Elt elt;
  Act act;
  LinearMode mode;
  const void *x, *x2, *w, *w2;
  const void *bias, *residual;   // may be null
  void *out, *out2, *pre, *pre2;   // pre, pre2 may be null
  int64_t M, N, K;
  int64_t sxm, sxk, swk, swn;
  int64_t srm, som, spm;         // row strides of residual, out / out2, pre / pre2
};

// dz = dout * act'(pre) and dbias[n] = sum_m dz (each output may be null), or, gated,
// dgate = dout * up * act'(gate) and dup = dout * act(gate).
struct ActBwdProblem {
  Elt elt;
  Act act;
  bool gated;
  const void *dout, *pre, *up;   // pre: the gate's pre-activation when gated; null means act == None
  void *dz, *dup;
  void* dbias;
  int64_t M, N;
  int64_t s_dout, s_pre, s_dz;   // row strides (dz and dup share one, pre and up share one)
};

// t = post_weight ? N(block) * post_weight : block;  s = scale * residual + gate * t;
// normed = N(s) * weight + bias.  N: root-mean-square norm, or layer norm (mean removed).
// stats[row] = {mean of s, 1/deviation of s, mean of block, 1/deviation of block}, fp32.
constexpr int64_t kNormMaxColumns = 16384;   // a row stays in the registers of one block
struct NormProblem {
  Elt elt;
  bool layer;
  const void *residual, *block, *weight, *bias, *gate, *post_weight;   // block, bias, gate, post_weight may be null
  void *sum, *normed;
  float* stats;                  // may be null in the forward pass
  float scale, eps;
  int64_t M, D, stride;          // one row stride for every [M, D] operand
  // backward
  const void *dnormed, *dsum;    // dsum may be null
  void *dresidual, *dblock, *dweight, *dbias, *dgate, *dpost;
};

// While it lives, the calling thread may set the library up (allocate, create streams, wait for its own probe)
// although a stream of the thread is being captured: none of that touches the captured stream.
struct SetUpDuringCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  SetUpDuringCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~SetUpDuringCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// Memory that lives from one point of the launch's stream to another (stream-ordered pool of the
// library's own): two calls on two streams, or two captured graphs, never share it.
std::string scratch_alloc(const LaunchCtx& ctx, size_t bytes, void** out);
void scratch_free(const LaunchCtx& ctx, void* p);

// out[i][n] = sum of partial[i][0 ... parts-1][n], in that order, for `sets` arrays.
constexpr int kMaxColumnSums = 4;
void launch_column_sums(Elt elt, const float* partial, int64_t parts, int64_t N, int sets, void* const* out,
                        const LaunchCtx& ctx);

// Any strides, any alignment, fp32 accumulation on the CUDA cores.
std::string launch_linear_simt(const LinearProblem& p, const LaunchCtx& ctx);
// fp32 operands that are contiguous along one dimension.
bool linear_f32_takes(const LinearProblem& p);
std::string launch_linear_f32(const LinearProblem& p, const LaunchCtx& ctx);
// Picks the kernel (path_option: 0 automatic, 1 the CUDA cores, 2 the tensor cores or `refused` says why
// not) and reports which it was (1 or 2).
std::string launch_linear(const LinearProblem& p, const LaunchCtx& ctx, int path_option, int* path_used,
                          std::string* refused);
// What a 16-bit product on the tensor cores runs on: the few-row kernel (tile: rows of x, split: of K) or the CTA
// pairs (tile: accumulator columns, tiles: how many).
struct TensorChoice {
  int narrow, tile, split;
  int64_t tiles;
};
TensorChoice tensor_choice(const LinearProblem& p, bool x_by_k, int sm_count);
std::string launch_activation_bwd(const ActBwdProblem& p, const LaunchCtx& ctx);
std::string launch_residual_norm(const NormProblem& p, const LaunchCtx& ctx);
std::string launch_residual_norm_bwd(const NormProblem& p, const LaunchCtx& ctx);

}  // namespace tmc
