// The feed-forward matrix products for few rows - a decoding step, a short prompt - on the tensor cores.
//
//   single  z = x w + bias; out = act(z) + residual       gated  out = act(x w) * (x w2)
//   sum     out = x w + x2 w2
//
// With M rows of x, M small, the weights are read once and are the bound: 2 bytes for 2 M operations.
// So w takes the MMA's 128-row side and the rows of x, padded to 16, 32, 64 or 128, the other
// (tcgen05.mma 128 x TOK x 16, D = (x w)^T in TMEM): a CTA owns 128 output columns, streams its part of
// w through a shared-memory ring by TMA and pads nothing that crosses the memory bus (rows of x past M
// are filled with zeros by the TMA).  128 columns a CTA leave most SMs idle, so a cluster of up to 8
// CTAs splits K: each accumulates its share, leaves it in its shared memory, and finishes 1/8 (1/S) of
// the columns from all the shares through distributed shared memory, in rank order - no workspace, no
// atomics, the same bits every time.
//
//   warps 0 ... 3 (7, 15 with more rows) read TMEM (thread = output column), then a TMA producer warp and an
//   MMA issuer warp; all of them finish the cluster's sums.  About 100 KB of ring a CTA (two CTAs an SM) keep the memory bus busy:
//   148 x 100 KB in flight against 6.5 TB/s x 1 us.

#include "ffn_math.cuh"
#include "linear_tc.h"
#include "sm100_ptx.cuh"

#include <algorithm>

namespace tmc {
namespace {

using namespace ptx;
using namespace ffn;

constexpr int BN = 128;                // output columns of a CTA
constexpr int BK = 64;
constexpr int W_BYTES = BN * BK * 2;

template <int TOK, bool GATED> struct Config {
  // the sums are finished by as many warps as there are rows to keep busy: what each does is short and waits
  // for distributed shared memory, and unrolling it instead misses the instruction cache
  static constexpr int EPI_WARPS = TOK <= 16 ? 4 : TOK <= 64 ? 8 : 16;
  static constexpr int NUM_THREADS = (EPI_WARPS + 2) * 32;
  static constexpr int X_BYTES = TOK * BK * 2;
  static constexpr int STAGE_BYTES = W_BYTES * (GATED ? 2 : 1) + X_BYTES;
  // two CTAs an SM up to 64 rows, one beyond (the shares of a cluster must fit where the ring was)
  static constexpr int RING = TOK <= 64 ? 104 * 1024 : 196 * 1024;
  static constexpr int STAGES = RING / STAGE_BYTES;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 2048;
  static constexpr int TMEM_COLS = TOK * (GATED ? 2 : 1) < 32 ? 32 : TOK * (GATED ? 2 : 1);
  static_assert(STAGES >= 2 && STAGES <= 12, "ring");
  static_assert(TOK * BN * 4 * (GATED ? 2 : 1) <= STAGES * STAGE_BYTES, "the shares fit into the ring");
};

enum Site : uint32_t { kProdEmpty = 51, kMmaFull = 52, kEpiAccFull = 53, kDrain = 54 };

struct Barriers {
  alignas(8) uint64_t full[12];
  alignas(8) uint64_t empty[12];
  alignas(8) uint64_t acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

struct alignas(64) Maps {
  CUtensorMap x, x2, w, w2;
};

struct Args {
  int M, N, K;
  int act, sum, w_mn, split;
  const void *bias, *residual;
  void *out, *pre, *pre2;
  int64_t srm, som, spm;
  int quads;                           // kQuad...: every fourth element of the operand's rows is 8-byte aligned
};
enum : int { kQuadOut = 1, kQuadPre = 2, kQuadBias = 4, kQuadResidual = 8 };

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// (not the .aligned forms: a warp whose lanes have taken different roles may still be diverged here)
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float4 load_share(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

__device__ __forceinline__ void add(float4& a, const float4& b) {
  a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
}

// The sum over the cluster of what lies at `addr` in each CTA's shared memory, in rank order.
__device__ __forceinline__ float4 gather(uint32_t addr, int split) {
  float4 part[8];
#pragma unroll
  for (int r = 0; r < 8; ++r)
    if (r < split) part[r] = load_share(addr, r);
#pragma unroll
  for (int r = 1; r < 8; ++r)
    if (r < split) add(part[0], part[r]);
  return part[0];
}

// Four neighbouring elements of an output or a bias / residual: one 8-byte access where the address allows.
template <typename T>
__device__ __forceinline__ void add4(float (&v)[4], const T* from, int left, bool quads) {
  if (quads && left >= 4) {
    const uint2 raw = *reinterpret_cast<const uint2*>(from);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) v[i] += to_f32(from[i]);
  }
}
template <typename T>
__device__ __forceinline__ void put4(T* to, const float (&v)[4], int left, bool quads) {
  if (quads && left >= 4) {
    uint2 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint2*>(to) = raw;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) to[i] = from_f32<T>(v[i]);
  }
}

// Outputs n ... n + 3 of row m (`left` of them exist) from x w, and from x w2 of a gated product.
template <typename T, bool GATED>
__device__ __forceinline__ void finish(const Args& a, int64_t m, int n, int left, float4 sum, float4 sum2) {
  float z[4] = {sum.x, sum.y, sum.z, sum.w};
  if constexpr (GATED) {
    const float up[4] = {sum2.x, sum2.y, sum2.z, sum2.w};
    if (a.pre) put4((T*)a.pre + m * a.spm + n, z, left, a.quads & kQuadPre);
    if (a.pre2) put4((T*)a.pre2 + m * a.spm + n, up, left, a.quads & kQuadPre);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = act_forward<false>((Act)a.act, z[i]) * up[i];
  } else {
    if (a.bias) add4(z, (const T*)a.bias + n, left, a.quads & kQuadBias);
    if (a.pre) put4((T*)a.pre + m * a.spm + n, z, left, a.quads & kQuadPre);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = act_forward<false>((Act)a.act, z[i]);
    if (a.residual) add4(z, (const T*)a.residual + m * a.srm + n, left, a.quads & kQuadResidual);
  }
  put4((T*)a.out + m * a.som + n, z, left, a.quads & kQuadOut);
}

template <typename T, int TOK, bool GATED>
__global__ void __launch_bounds__(Config<TOK, GATED>::NUM_THREADS, TOK <= 64 ? 2 : 1)
linear_narrow_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a, DeviceStatus* status) {
  using C = Config<TOK, GATED>;
  constexpr int STAGES = C::STAGES, STAGE_BYTES = C::STAGE_BYTES, NUM_THREADS = C::NUM_THREADS;
  constexpr int PRODUCER = C::EPI_WARPS, ISSUER = C::EPI_WARPS + 1;
  constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  Barriers& bars = *reinterpret_cast<Barriers*>(smem + STAGES * STAGE_BYTES);
  const uint32_t smem_base = smem_u32(smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cta_rank();          // 0 without a cluster
  WaitCtx wc{&bars.abort_flag, status};

  const int n0 = (int)(blockIdx.x / a.split) * BN, m0 = (int)blockIdx.y * TOK;
  const int rows = min(TOK, a.M - m0);
  const int blocks_one = (a.K + BK - 1) / BK;
  const int blocks = a.sum ? 2 * blocks_one : blocks_one;
  const int kb0 = (int)((int64_t)blocks * rank / a.split), kb1 = (int)((int64_t)blocks * (rank + 1) / a.split);

  // One k-block of both operands into a slot of the ring.
  auto fetch = [&](int kb, int stage) {
    const bool other = kb >= blocks_one;                             // sum: the second pair of operands
    const int k = (other ? kb - blocks_one : kb) * BK;
    const uint32_t bar = smem_u32(&bars.full[stage]);
    uint32_t dst = smem_base + stage * STAGE_BYTES;
    mbar_expect_tx(bar, STAGE_BYTES);
#pragma unroll
    for (int g = 0; g < (GATED ? 2 : 1); ++g) {
      const CUtensorMap* mw = g || other ? &maps.w2 : &maps.w;
      if (a.w_mn) {
        tma_load_2d(dst, mw, bar, n0, k);
        tma_load_2d(dst + 8192, mw, bar, n0 + 64, k);
      } else {
        tma_load_2d(dst, mw, bar, k, n0);
      }
      dst += W_BYTES;
    }
    tma_load_2d(dst, other ? &maps.x2 : &maps.x, bar, k, m0);
  };

  // The thread that makes the barriers fills the ring at once: the first weights are under way while the
  // TMEM is allocated and the other warps arrive.
  const int ahead = min(STAGES, kb1 - kb0);
  if (warp == PRODUCER && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&bars.full[s]), 1);
      mbar_init(smem_u32(&bars.empty[s]), 1);
    }
    mbar_init(smem_u32(&bars.acc_full), 1);
    bars.abort_flag = 0;
    fence_barrier_init();
    for (int s = 0; s < ahead; ++s) fetch(kb0 + s, s);
  }
  if (warp == ISSUER) {
    tmem_alloc(smem_u32(&bars.tmem_base), C::TMEM_COLS);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars.tmem_base;

  bool ok = true;
  if (warp == PRODUCER) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = ahead == STAGES ? 0 : ahead;
      uint32_t phase = ahead == STAGES ? 1 : 0, issued = ahead;
      for (int kb = kb0 + ahead; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1, wc, kProdEmpty)) { ok = false; break; }
        fetch(kb, stage);
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      // every copy started must have landed before the CTA leaves or the ring is reused
      const uint32_t pending = issued < (uint32_t)STAGES ? issued : (uint32_t)STAGES;
      for (uint32_t i = 0; i < pending; ++i) {
        if (--stage < 0) { stage = STAGES - 1; phase ^= 1; }
        const long long t0 = clock64();
        while (!mbar_try_wait(smem_u32(&bars.full[stage]), phase)) {
          if (clock64() - t0 > kWaitCycles) { report_timeout(wc, kDrain, stage); break; }
        }
      }
    }
  } else if (warp == ISSUER) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t n_field = TOK;
    const uint32_t idesc = make_idesc(FMT, BN, n_field, a.w_mn, 0);
    const SmemDesc w_base = make_desc_sw128(smem_base, a.w_mn ? 8192 : 0, 1024);
    const SmemDesc x_base = make_desc_sw128(smem_base + W_BYTES * (GATED ? 2 : 1), 0, 1024);
    const uint32_t w_step = a.w_mn ? 2048 : 32;
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(smem_u32(&bars.full[stage]), phase, wc, kMmaFull)) { ok = false; break; }
      tc_fence_after();
      const SmemDesc w_desc = w_base.advanced(stage * STAGE_BYTES);
      const SmemDesc x_desc = x_base.advanced(stage * STAGE_BYTES);
#pragma unroll
      for (int k = 0; k < BK / 16; ++k) {
        mma_f16_ss_elect(tmem_base, w_desc.at(k * w_step), x_desc.at(k * 32), idesc, kb > kb0 || k != 0);
        if constexpr (GATED)
          mma_f16_ss_elect(tmem_base + TOK, w_desc.at(W_BYTES + k * w_step), x_desc.at(k * 32), idesc, kb > kb0 || k != 0);
      }
      mma_commit_elect(smem_u32(&bars.empty[stage]));
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
    }
    if (ok) mma_commit_elect(smem_u32(&bars.acc_full));
  } else {
    // ------------------------------------------------------------ accumulator, thread = output column
    // (after a wait that gave up the sums are whatever is there, and the launch is reported as failed; by vote, so
    // that the lanes come to the warp-wide loads together whichever of them saw the barrier or gave up first)
    // The wait lasts as long as all of the CTA's products do, a few hundred clocks a k-block (4096 allowed).
    const WaitCtx all_blocks{&bars.abort_flag, status, kWaitCycles + 4096ll * (kb1 - kb0)};
    mbar_wait_warp(smem_u32(&bars.acc_full), 0, all_blocks, kEpiAccFull);
    tc_fence_after();
    const int quarter = warp % 4;
    const uint32_t lanes = tmem_base + ((uint32_t)(quarter * 32) << 16);
    float* share = reinterpret_cast<float*>(smem) + quarter * 32 + lane;     // [GATED][row][128 columns]: the ring is idle now
#pragma unroll 1
    for (int t = warp / 4 * 8; t < rows; t += C::EPI_WARPS / 4 * 8) {
      uint32_t z[8], up[8];
      tmem_ld_32x8(lanes + t, z);
      if constexpr (GATED) tmem_ld_32x8(lanes + TOK + t, up);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 8; ++i) {           // (rows past the last are zeros in a place of their own)
        share[(t + i) * BN] = __uint_as_float(z[i]);
        if constexpr (GATED) share[(TOK + t + i) * BN] = __uint_as_float(up[i]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  // The columns go back before the first wait for the cluster: a CTA that held them while it waited for a peer,
  // and a peer that waits for columns of another launch in the same state, would wait for each other.
  if (warp == ISSUER) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
  // Four columns of a row at a time, the shares of the whole cluster loaded before the first is added.
  if (a.split > 1) cluster_sync();     // every share is written
  const int width = BN / a.split, shift = 31 - __clz(width / 4), items = rows << shift;
#pragma unroll 1
  for (int i = threadIdx.x; i < items; i += NUM_THREADS) {
    const int t = i >> shift, c = (int)rank * width + (i - (t << shift)) * 4;
    const int left = a.N - n0 - c;
    if (left <= 0) continue;
    const uint32_t at = (uint32_t)(t * BN + c) * 4;
    float4 z, up = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.split == 1) {
      z = *reinterpret_cast<const float4*>(smem + at);
      if constexpr (GATED) up = *reinterpret_cast<const float4*>(smem + at + TOK * BN * 4);
    } else {
      z = gather(smem_base + at, a.split);
      if constexpr (GATED) up = gather(smem_base + at + TOK * BN * 4, a.split);
    }
    finish<T, GATED>(a, m0 + t, n0 + c, left, z, up);
  }
  if (a.split > 1) {
    __syncwarp();
    cluster_sync();                    // nobody still reads this CTA's share
  }
}

template <typename T, int TOK, bool GATED>
std::string launch_tok(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw, int split,
                       const LaunchCtx& ctx) {
  using C = Config<TOK, GATED>;
  const CUtensorMapDataType type =
      p.elt == Elt::BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  Maps maps{};
  std::string e = make_operand_map(&maps.x, type, p.x, p.M, p.K, lx, TOK);
  if (e.empty()) e = make_operand_map(&maps.w, type, p.w, p.N, p.K, lw, BN);
  if (e.empty() && p.x2) e = make_operand_map(&maps.x2, type, p.x2, p.M, p.K, lx, TOK);
  if (e.empty() && p.w2) e = make_operand_map(&maps.w2, type, p.w2, p.N, p.K, lw, BN);
  if (!e.empty()) return e;
  Args a{};
  a.M = (int)p.M; a.N = (int)p.N; a.K = (int)p.K;
  a.act = (int)p.act;
  a.sum = p.mode == LinearMode::Sum;
  a.w_mn = lw.mn;
  a.split = split;
  a.bias = p.bias; a.residual = p.residual;
  a.out = p.out; a.pre = p.pre; a.pre2 = p.pre2;
  a.srm = p.srm; a.som = p.som; a.spm = p.spm;
  auto quad = [&](const void* q, const void* q2, int64_t stride, int bit) {
    return (((uintptr_t)q | (uintptr_t)q2) % 8 == 0 && (p.M <= 1 || stride % 4 == 0)) ? bit : 0;
  };
  a.quads = quad(p.out, nullptr, p.som, kQuadOut) | quad(p.pre, p.pre2, p.spm, kQuadPre) | quad(p.bias, nullptr, 0, kQuadBias) |
            quad(p.residual, nullptr, p.srm, kQuadResidual);
  auto kernel = linear_narrow_kernel<T, TOK, GATED>;
  static const cudaError_t sized = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  cudaError_t err = sized;
  if (err != cudaSuccess) return cudaGetErrorString(err);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)((p.N + BN - 1) / BN * split), (unsigned)((p.M + TOK - 1) / TOK));
  config.blockDim = dim3(C::NUM_THREADS);
  config.dynamicSmemBytes = C::SMEM;
  config.stream = ctx.stream;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)split;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  err = cudaLaunchKernelEx(&config, kernel, maps, a, ctx.status);
  ++*ctx.launches;
  if (err != cudaSuccess) {
    cudaGetLastError();
    return std::string("launch failed: ") + cudaGetErrorString(err);
  }
  return std::string();
}

template <typename T, bool GATED>
std::string launch_rows(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw, const NarrowPlan& plan,
                        const LaunchCtx& ctx) {
  switch (plan.rows) {
    case 16: return launch_tok<T, 16, GATED>(p, lx, lw, plan.split, ctx);
    case 32: return launch_tok<T, 32, GATED>(p, lx, lw, plan.split, ctx);
    case 64: return launch_tok<T, 64, GATED>(p, lx, lw, plan.split, ctx);
    default: return launch_tok<T, 128, GATED>(p, lx, lw, plan.split, ctx);
  }
}

}  // namespace

bool plan_linear_narrow(const LinearProblem& p, const OperandLayout& lx, int sm_count, NarrowPlan* plan) {
  if (lx.mn || p.mode == LinearMode::Pair) return false;
  plan->rows = p.M <= 16 ? 16 : p.M <= 32 ? 32 : p.M <= 64 ? 64 : 128;
  const int64_t tiles = (p.N + BN - 1) / BN * ((p.M + plan->rows - 1) / plan->rows);
  if ((p.M + plan->rows - 1) / plan->rows > 65535 || tiles > 0x0fffffff) return false;
  const int64_t blocks = (p.K + BK - 1) / BK * (p.mode == LinearMode::Sum ? 2 : 1);
  const int64_t slots = (int64_t)sm_count * (plan->rows <= 64 ? 2 : 1);
  // The split that is done first.  An SM takes in about 38 bytes a clock (86 CTAs streamed 180 MB in 30 us), and
  // what comes from memory comes at 3400 (6.5 TB/s at 1.9 GHz); the cluster's exchange costs about 2000 clocks, the
  // rows of the sums 600 for every 512 groups of four columns.  Clusters of eight with an SM to each CTA do not
  // all fit their GPCs at once, and take twice as long.
  double best = 0;
  plan->split = 0;
  const int weights = p.mode == LinearMode::Gated ? 2 : 1;
  const double per_block = (double)(weights * 16384 + plan->rows * 128);
  const double memory = 2.0 * ((double)p.K * (double)p.N * (p.w2 ? 2 : 1) + (double)p.M * (double)p.K) / 3400.0;
  for (int split = 1; split <= (plan->rows <= 64 ? 8 : 4) && split <= blocks; split *= 2) {
    const int64_t ctas = tiles * split;
    const double each = (double)((blocks + split - 1) / split);
    const double waves = (double)((ctas + slots - 1) / slots);
    const double share = ctas > slots ? waves * (double)slots / sm_count : std::max(1.0, (double)ctas / sm_count);
    const double rows = (double)std::min<int64_t>(plan->rows, p.M);
    const double finish = (split > 1 ? 2000.0 : 0.0) + rows * (32.0 / split) / 512.0 * 600.0;
    const double time = std::max(memory, share * each * per_block / 38.0) + waves * finish;
    if (!plan->split || time < best) {
      best = time;
      plan->split = split;
    }
  }
  plan->clocks = best + 6000.0;
  return true;
}

std::string launch_linear_narrow(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw,
                                 const NarrowPlan& plan, const LaunchCtx& ctx) {
  const bool gated = p.mode == LinearMode::Gated;
  if (p.elt == Elt::BF16)
    return gated ? launch_rows<__nv_bfloat16, true>(p, lx, lw, plan, ctx)
                 : launch_rows<__nv_bfloat16, false>(p, lx, lw, plan, ctx);
  return gated ? launch_rows<__half, true>(p, lx, lw, plan, ctx) : launch_rows<__half, false>(p, lx, lw, plan, ctx);
}

}  // namespace tmc
