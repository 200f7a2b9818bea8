// The feed-forward matrix products on the CUDA cores: every element type, any strides and
// alignment, extents from zero up.  What comes here is what the other kernels do not take: K = 0,
// 16-bit products of K < 33 with an operand that the TMA cannot fetch (or with no memory for its
// aligned copy, or when the CUDA cores are asked for), and fp32 operands without a contiguous
// dimension (the others have linear_f32.cu).  The bound is the FMA pipe - 2 x 128 lanes x 148 SMs x
// 1.9 GHz, 72 TFLOP/s.
//
// Tile 128 x 128 x 16, 256 threads, 8 x 8 outputs each as two 4-wide halves 64 rows / columns
// apart (so that the 16-byte shared-memory reads of a quarter-warp touch distinct banks), the next
// k-step's elements held in registers while the current one is multiplied, two-wide FMAs.  The
// gated form takes its two weight matrices as the two column halves of one tile, so a thread holds
// x w and x w2 of the same four columns and multiplies them in registers.

#include "ffn_math.cuh"
#include "sm100_ptx.cuh"

namespace tmc {
namespace {

using namespace ffn;

constexpr int TM = 128, TN = 128, TK = 16;

template <typename T, bool GATED>
__global__ void __launch_bounds__(256, 2) linear_simt_kernel(const LinearProblem p) {
  __shared__ float As[2][TK][TM + 4];
  __shared__ float Bs[2][TK][TN + 4];
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  constexpr int COLS = GATED ? TN / 2 : TN;          // output columns of a tile
  const int64_t m0 = (int64_t)blockIdx.x * TM, n0 = (int64_t)blockIdx.y * COLS;
  const bool second = p.mode == LinearMode::Pair && blockIdx.z == 1;
  const T* x = (const T*)(second ? p.x2 : p.x);
  const T* w = (const T*)(second ? p.w2 : p.w);
  const int64_t steps_one = (p.K + TK - 1) / TK;
  const int64_t steps = p.mode == LinearMode::Sum ? 2 * steps_one : steps_one;
  // which index runs along a warp: the one whose stride is 1
  const bool x_by_k = p.sxk == 1, w_by_n = p.swn == 1;

  uint64_t acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0;

  float ra[8], rb[8];
  auto fetch = [&](int64_t step) {
    const bool other = step >= steps_one;              // Sum: the second pair of operands
    const int64_t k0 = (other ? step - steps_one : step) * TK;
    const T* xs = other ? (const T*)p.x2 : x;
    const T* ws = other ? (const T*)p.w2 : w;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = x_by_k ? tid / 16 + 16 * i : tid % 128, k = x_by_k ? tid % 16 : tid / 128 + 2 * i;
      const bool in = m0 + m < p.M && k0 + k < p.K;
      ra[i] = in ? to_f32(xs[(m0 + m) * p.sxm + (k0 + k) * p.sxk]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = w_by_n ? tid % 128 : tid / 16 + 16 * i, k = w_by_n ? tid / 128 + 2 * i : tid % 16;
      const int64_t col = n0 + (GATED ? n % COLS : n);
      const T* base = GATED && n >= COLS ? (const T*)p.w2 : ws;
      const bool in = col < p.N && k0 + k < p.K;
      rb[i] = in ? to_f32(base[(k0 + k) * p.swk + col * p.swn]) : 0.f;
    }
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = x_by_k ? tid / 16 + 16 * i : tid % 128, k = x_by_k ? tid % 16 : tid / 128 + 2 * i;
      As[buf][k][m] = ra[i];
      const int n = w_by_n ? tid % 128 : tid / 16 + 16 * i, kb = w_by_n ? tid / 128 + 2 * i : tid % 16;
      Bs[buf][kb][n] = rb[i];
    }
  };

  if (steps > 0) {
    fetch(0);
    stage(0);
  }
  __syncthreads();
  for (int64_t s = 0; s < steps; ++s) {
    const int buf = (int)(s & 1);
    if (s + 1 < steps) fetch(s + 1);
#pragma unroll
    for (int k = 0; k < TK; ++k) {
      const float4 a0 = *reinterpret_cast<const float4*>(&As[buf][k][ty * 4]);
      const float4 a1 = *reinterpret_cast<const float4*>(&As[buf][k][64 + ty * 4]);
      const ulonglong2 b0 = *reinterpret_cast<const ulonglong2*>(&Bs[buf][k][tx * 4]);
      const ulonglong2 b1 = *reinterpret_cast<const ulonglong2*>(&Bs[buf][k][64 + tx * 4]);
      const float a[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint64_t aa = ptx::pack_f32x2(a[i], a[i]);
        acc[i][0] = ptx::fma_f32x2(aa, b0.x, acc[i][0]);
        acc[i][1] = ptx::fma_f32x2(aa, b0.y, acc[i][1]);
        acc[i][2] = ptx::fma_f32x2(aa, b1.x, acc[i][2]);
        acc[i][3] = ptx::fma_f32x2(aa, b1.y, acc[i][3]);
      }
    }
    if (s + 1 < steps) stage(buf ^ 1);
    __syncthreads();
  }

  T* out = (T*)(second ? p.out2 : p.out);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t m = m0 + (i / 4) * 64 + ty * 4 + i % 4;
    if (m >= p.M) continue;
    float z[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) ptx::unpack_f32x2(acc[i][j], z[2 * j], z[2 * j + 1]);
    if constexpr (GATED) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + tx * 4 + j;
        if (n >= p.N) continue;
        if (p.pre) ((T*)p.pre)[m * p.spm + n] = from_f32<T>(z[j]);
        if (p.pre2) ((T*)p.pre2)[m * p.spm + n] = from_f32<T>(z[4 + j]);
        out[m * p.som + n] = from_f32<T>(act_forward<true>(p.act, z[j]) * z[4 + j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t n = n0 + (j / 4) * 64 + tx * 4 + j % 4;
        if (n >= p.N) continue;
        float v = z[j];
        if (p.bias) v += to_f32(((const T*)p.bias)[n]);
        if (p.pre) ((T*)p.pre)[m * p.spm + n] = from_f32<T>(v);
        v = act_forward<true>(p.act, v);
        if (p.residual) v += to_f32(((const T*)p.residual)[m * p.srm + n]);
        out[m * p.som + n] = from_f32<T>(v);
      }
    }
  }
}

template <typename T>
std::string launch_typed(const LinearProblem& p, const LaunchCtx& ctx) {
  const bool gated = p.mode == LinearMode::Gated;
  const int cols = gated ? TN / 2 : TN;
  const int64_t gx = (p.M + TM - 1) / TM, gy = (p.N + cols - 1) / cols;
  if (gy > 65535) return "more than " + std::to_string(65535 * cols) + " columns";
  const dim3 grid((unsigned)gx, (unsigned)gy, p.mode == LinearMode::Pair ? 2 : 1);
  if (gated) linear_simt_kernel<T, true><<<grid, 256, 0, ctx.stream>>>(p);
  else linear_simt_kernel<T, false><<<grid, 256, 0, ctx.stream>>>(p);
  ++*ctx.launches;
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return std::string("linear launch failed: ") + cudaGetErrorString(e);
  return std::string();
}

}  // namespace

std::string launch_linear_simt(const LinearProblem& p, const LaunchCtx& ctx) {
  if (p.elt == Elt::F32) return launch_typed<float>(p, ctx);
  if (p.elt == Elt::BF16) return launch_typed<__nv_bfloat16>(p, ctx);
  return launch_typed<__half>(p, ctx);
}

}  // namespace tmc
