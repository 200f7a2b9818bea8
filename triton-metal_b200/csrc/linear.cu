// Which kernel a feed-forward matrix product runs on, and the copies that make an operand fetchable.
//
// The tensor-core kernels fetch their operands by TMA, which needs one contiguous dimension, a 16-byte
// aligned base and a pitch that is a multiple of 16 bytes.  An operand that misses that (an odd width, a
// slice at an odd column, no contiguous dimension) is first copied into aligned scratch memory: one read
// and one write of it, against a product on the CUDA cores that reads element by element and waits for each
// step of 16 k (1 x 129 x 129: 36 us there, 5 with the copy; 300 x 511 x 513: 196 and 10).  Up to two such
// steps the second launch and the scratch cost the caller more than they save the GPU.

#include "ffn_core.h"
#include "linear_tc.h"

#include <algorithm>

namespace tmc {
namespace {

constexpr int64_t kCopyFromK = 33;
constexpr int64_t kMostRows = 0x7fffffff - 512;       // tiles past the edge are counted in 32 bits

// The TMA's view of an operand of `outer` rows, K columns; false if it has none.
bool layout_of(const void* base, const void* base2, int64_t outer, int64_t K, int64_t s_outer, int64_t s_k,
               OperandLayout* l) {
  if (((uintptr_t)base | (uintptr_t)base2) % 16) return false;
  auto pitch = [](int64_t stride, int64_t extent, int64_t inner) -> int64_t {
    if (extent <= 1) return (inner + 7) / 8 * 8;          // never stepped
    return stride > 0 && stride % 8 == 0 && stride < (1ll << 38) ? stride : 0;
  };
  if (s_k == 1 || K <= 1) {
    if (const int64_t p = pitch(s_outer, outer, K)) { *l = {0, p}; return true; }
  }
  if (s_outer == 1 || outer <= 1) {
    if (const int64_t p = pitch(s_k, K, outer)) { *l = {1, p}; return true; }
  }
  return false;
}

// One operand to be copied: `rows` rows of `cols` elements into dense rows `pitch` apart.
struct CopyJob {
  const uint16_t* from;
  uint16_t* to;
  int64_t rows, cols, row_stride, col_stride, pitch;
};
struct CopyJobs {
  CopyJob job[4];
};
// Eight elements from any 2-byte aligned address, contiguous: five aligned words, shifted into place.
__device__ __forceinline__ uint4 load_unaligned(const uint16_t* from) {
  const uintptr_t at = (uintptr_t)from;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
  const uint32_t w0 = __ldg(words), w1 = __ldg(words + 1), w2 = __ldg(words + 2), w3 = __ldg(words + 3);
  if (!(at & 2)) return make_uint4(w0, w1, w2, w3);
  const uint32_t w4 = __ldg(reinterpret_cast<const uint16_t*>(words + 4));    // only its lower half is ours
  return make_uint4(__funnelshift_r(w0, w1, 16), __funnelshift_r(w1, w2, 16), __funnelshift_r(w2, w3, 16),
                    __funnelshift_r(w3, w4, 16));
}
__global__ void __launch_bounds__(256) align_operands_kernel(const CopyJobs jobs) {
  const CopyJob& j = jobs.job[blockIdx.y];
  const int64_t packets = j.pitch / 8, total = j.rows * packets;
  const uint32_t narrow = total < 0x7fffffff ? (uint32_t)packets : 0;      // a 64-bit division costs a hundred instructions
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = narrow ? (int64_t)((uint32_t)i / narrow) : i / packets, c = (i - r * packets) * 8;
    const uint16_t* from = j.from + r * j.row_stride + c * j.col_stride;
    uint4 v;
    // (a packet's first word may begin two bytes early: at the operand's own first element that is not ours)
    if (j.col_stride == 1 && c + 8 <= j.cols && i > 0) {
      v = load_unaligned(from);
    } else {
      uint16_t e[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = c + k < j.cols ? from[k * j.col_stride] : (uint16_t)0;
      v.x = e[0] | (uint32_t)e[1] << 16;
      v.y = e[2] | (uint32_t)e[3] << 16;
      v.z = e[4] | (uint32_t)e[5] << 16;
      v.w = e[6] | (uint32_t)e[7] << 16;
    }
    *reinterpret_cast<uint4*>(j.to + r * j.pitch + c) = v;
  }
}

// Copies of an operand pair's members with the contiguous dimension kept (k where there is none).
struct Aligned {
  CopyJob job[2];
  int jobs = 0;
  OperandLayout layout;
  size_t bytes = 0;
  void plan(const void* a, const void* b, int64_t outer, int64_t K, int64_t s_outer, int64_t s_k) {
    const int mn = s_outer == 1 && s_k != 1;
    const int64_t rows = mn ? K : outer, cols = mn ? outer : K;
    const int64_t pitch = (cols + 7) / 8 * 8;
    layout = {mn, pitch};
    for (const void* q : {a, b}) {
      if (!q || (jobs && q == a)) continue;
      job[jobs++] = CopyJob{(const uint16_t*)q, nullptr, rows, cols, mn ? s_k : s_outer, mn ? s_outer : s_k, pitch};
      bytes += ((size_t)rows * (size_t)pitch * 2 + 255) / 256 * 256;
    }
  }
};

// The kernel for few rows or the one for many, whichever its estimate says is done first.
bool takes_narrow(const LinearProblem& p, const OperandLayout& lx, int sm_count, NarrowPlan* plan) {
  return plan_linear_narrow(p, lx, sm_count, plan) && plan->clocks < estimate_linear_tc(p, sm_count);
}
std::string launch_tensor(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw, const LaunchCtx& ctx) {
  NarrowPlan narrow{};
  if (takes_narrow(p, lx, ctx.sm_count, &narrow)) return launch_linear_narrow(p, lx, lw, narrow, ctx);
  return launch_linear_tc(p, lx, lw, ctx);
}

}  // namespace

TensorChoice tensor_choice(const LinearProblem& p, bool x_by_k, int sm_count) {
  NarrowPlan narrow{};
  TensorChoice c{};
  if (takes_narrow(p, OperandLayout{x_by_k ? 0 : 1, 0}, sm_count, &narrow)) {
    c.narrow = 1;
    c.tile = narrow.rows;
    c.split = narrow.split;
  } else {
    c.split = 1;
    c.tile = linear_tc_width(p, sm_count, &c.tiles);
  }
  return c;
}

std::string launch_linear(const LinearProblem& p, const LaunchCtx& ctx, int path_option, int* path_used,
                          std::string* refused) {
  *path_used = 1;
  OperandLayout lx{}, lw{};
  const bool x_fits = layout_of(p.x, p.x2, p.M, p.K, p.sxm, p.sxk, &lx);
  const bool w_fits = layout_of(p.w, p.w2, p.N, p.K, p.swn, p.swk, &lw);
  const char* why = p.elt == Elt::F32 ? "fp32 operands take the CUDA cores"
                    : p.K == 0 ? "K is 0"
                    : p.M > kMostRows || p.N > kMostRows || p.K > kMostRows ? "an extent within 512 of 2^31"
                    : path_option == 1 ? "the CUDA cores were asked for"
                    : path_option == 0 && p.K < kCopyFromK && !(x_fits && w_fits) ? "short, and not aligned to 16 bytes"
                                                                                 : nullptr;
  if (why) {
    if (path_option == 2) {
      *refused = why;
      return std::string();
    }
    return linear_f32_takes(p) ? launch_linear_f32(p, ctx) : launch_linear_simt(p, ctx);
  }
  *path_used = 2;
  if (x_fits && w_fits) return launch_tensor(p, lx, lw, ctx);

  Aligned cx, cw;
  if (!x_fits) cx.plan(p.x, p.x2, p.M, p.K, p.sxm, p.sxk);
  if (!w_fits) cw.plan(p.w, p.w2, p.N, p.K, p.swn, p.swk);
  void* scratch = nullptr;
  std::string e = scratch_alloc(ctx, cx.bytes + cw.bytes, &scratch);
  if (!e.empty()) {
    if (path_option == 2) return e;
    *path_used = 1;                      // no room for the copies: slower, but it needs none
    return launch_linear_simt(p, ctx);
  }
  char* at = (char*)scratch;
  CopyJobs jobs{};
  int n = 0;
  int64_t packets = 0;
  for (Aligned* c : {&cx, &cw}) {
    for (int i = 0; i < c->jobs; ++i) {
      CopyJob& j = c->job[i];
      j.to = (uint16_t*)at;
      at += ((size_t)j.rows * (size_t)j.pitch * 2 + 255) / 256 * 256;
      packets = std::max(packets, j.rows * (j.pitch / 8));
      jobs.job[n++] = j;
    }
  }
  LinearProblem q = p;
  if (cx.jobs) {
    q.x = cx.job[0].to;
    if (p.x2) q.x2 = cx.job[cx.jobs - 1].to;
    lx = cx.layout;
  }
  if (cw.jobs) {
    q.w = cw.job[0].to;
    if (p.w2) q.w2 = cw.job[cw.jobs - 1].to;
    lw = cw.layout;
  }
  const int64_t blocks = std::min<int64_t>((packets + 255) / 256, (int64_t)ctx.sm_count * 8);
  align_operands_kernel<<<dim3((unsigned)std::max<int64_t>(blocks, 1), (unsigned)n), 256, 0, ctx.stream>>>(jobs);
  ++*ctx.launches;
  cudaError_t err = cudaGetLastError();
  e = err != cudaSuccess ? std::string("copy launch failed: ") + cudaGetErrorString(err) : launch_tensor(q, lx, lw, ctx);
  scratch_free(ctx, scratch);
  return e;
}

}  // namespace tmc
