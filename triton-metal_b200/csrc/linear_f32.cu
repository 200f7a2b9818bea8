// The feed-forward matrix products on fp32 operands, on the CUDA cores.
//
// Products and sums are true fp32: the tensor cores' tf32 accumulator truncates, which costs an order of
// magnitude of error on sums of this length.  The bound is the FMA pipe: 128 lanes x 148 SMs x 1.9 GHz,
// 72 TFLOP/s.  A block of 256 threads owns TM x 128 outputs, TM / 16 x 8 a thread, and walks K in steps of
// 16 through a ring filled by cp.async.  Both operands lie in shared memory with k outermost, so
// a step's values are read as 16-byte vectors along the tile's edges and feed two-wide FMAs as they come;
// an operand that is contiguous along k is turned over on the way in, four bytes a copy (eight copies a
// thread and step against 512 two-wide FMAs), one that is not goes in 16 at a time.
//
// Few rows take a lower tile (TM 64, 32, 16), and few tiles a cluster of up to 8 blocks that split K: each
// leaves its sums in shared memory and finishes its share of the rows from all of them, in rank order.
// The gated form takes its two weight matrices as the two column halves of one tile.

#include "ffn_math.cuh"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <cmath>

namespace tmc {
namespace {

using namespace ffn;

constexpr int TN = 128, TK = 16;

template <int TM> struct Config {
  static constexpr int ROWS = TM / 16;                       // outputs of a thread: ROWS x 8
  // low tiles are bound by the weights' way from memory: more of them in flight
  static constexpr int STAGES = TM == 128 ? 3 : TM == 64 ? 4 : 8;
  static constexpr int A_PITCH = TM + 4, B_PITCH = TN + 4;   // floats from one k to the next
  static constexpr int A_FLOATS = TK * A_PITCH, STAGE_FLOATS = A_FLOATS + TK * B_PITCH;
  static constexpr int RING = STAGES * STAGE_FLOATS * 4, SHARE = (TM == 16 ? 8 * 16 : TM) * TN * 4;
  static constexpr int SMEM = RING > SHARE ? RING : SHARE;
};

__device__ __forceinline__ void copy16(uint32_t dst, const float* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const float* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// A thread's part in filling EDGE x 16 elements of an operand a step into shared memory, k outermost,
// `pitch` floats apart; what lies outside of `edges` x K is zero.  K_INNER: the operand is contiguous along
// k (a thread copies one k of every sixteenth edge element); else, with packets, every fourth element of a
// row is 16-byte aligned.
template <int EDGE>
struct Feed {
  const float* from;        // of the next step: the thread's first element
  int64_t hop;              // elements from one of the thread's copies to the next
  int64_t advance;          // and from step to step
  uint32_t to;              // byte offset of the first copy in the operand's piece
  int k, e, edges;          // the first copy's place; edge elements there are (from the tile's first)
  bool k_inner, packets;

  __device__ __forceinline__ void start(const float* base, int64_t stride, int64_t e0, int64_t k0, int64_t all, bool inner,
                                        bool quads, int pitch) {
    const int tid = threadIdx.x;
    k_inner = inner;
    packets = !inner && quads;
    edges = (int)min(all - e0, (int64_t)EDGE);
    if (inner) {
      k = tid % TK; e = tid / TK;
      from = base + (e0 + e) * stride + k0 + k;
      hop = 16 * stride;
      advance = TK;
    } else if (quads) {
      k = tid / (EDGE / 4); e = tid % (EDGE / 4) * 4;
      from = base + (k0 + k) * stride + e0 + e;
      hop = (1024 / EDGE) * stride;
      advance = TK * stride;
    } else {
      k = tid / EDGE; e = tid % EDGE;
      from = base + (k0 + k) * stride + e0 + e;
      hop = (256 / EDGE) * stride;
      advance = TK * stride;
    }
    to = (uint32_t)(k * pitch + e) * 4;
  }
  // `left`: elements of K from this step's first on
  __device__ __forceinline__ void step(uint32_t piece, int pitch, int64_t left) {
    const float* src = from;
    if (k_inner) {
      const bool in_k = k < left;
#pragma unroll
      for (int q = 0; q < EDGE / 16; ++q, src += hop) {
        const bool in = in_k && e + 16 * q < edges;
        copy4(piece + to + (uint32_t)(16 * q) * 4, in ? src : from, in ? 4 : 0);
      }
    } else if (packets) {
      constexpr int COPIES = EDGE * TK / 4 / 256 > 0 ? EDGE * TK / 4 / 256 : 1, ROWS = 1024 / EDGE;
      const int bytes = max(0, min(4, edges - e)) * 4;
      if (EDGE * TK / 4 >= 256 || k < TK) {
#pragma unroll
        for (int q = 0; q < COPIES; ++q, src += hop) {
          const bool in = k + ROWS * q < left && bytes > 0;
          copy16(piece + to + (uint32_t)(ROWS * q * pitch) * 4, in ? src : from, in ? bytes : 0);
        }
      }
    } else {
      constexpr int ROWS = 256 / EDGE;
#pragma unroll
      for (int q = 0; q < EDGE * TK / 256; ++q, src += hop) {
        const bool in = k + ROWS * q < left && e < edges;
        copy4(piece + to + (uint32_t)(ROWS * q * pitch) * 4, in ? src : from, in ? 4 : 0);
      }
    }
    from += advance;
  }
};

struct Form {
  int x_k, w_k;                      // the operand is contiguous along k
  int x_packets, w_packets, out_packets;
  int split;
};

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

__device__ __forceinline__ float finish(const LinearProblem& p, int64_t m, int64_t n, float z) {
  if (p.bias) z += ((const float*)p.bias)[n];
  if (p.pre) ((float*)p.pre)[m * p.spm + n] = z;
  z = act_forward<true>(p.act, z);
  if (p.residual) z += ((const float*)p.residual)[m * p.srm + n];
  return z;
}
__device__ __forceinline__ float finish_gated(const LinearProblem& p, int64_t m, int64_t n, float z, float up) {
  if (p.pre) ((float*)p.pre)[m * p.spm + n] = z;
  if (p.pre2) ((float*)p.pre2)[m * p.spm + n] = up;
  return act_forward<true>(p.act, z) * up;
}

// The k-steps of one block: its share of K (of both operand pairs in turn, for a sum) into the ring.
template <int TM, bool GATED>
struct Steps {
  using C = Config<TM>;
  static constexpr int COLS = GATED ? TN / 2 : TN;
  const LinearProblem& p;
  const Form& f;
  int64_t m0, n0, one, first, count;
  uint32_t base;
  const float *x, *w;
  Feed<TM> feed_x;
  Feed<COLS> feed_w, feed_up;

  __device__ __forceinline__ Steps(const LinearProblem& p, const Form& f, bool second, int64_t m0, int64_t n0, uint32_t rank,
                                   uint32_t base)
      : p(p), f(f), m0(m0), n0(n0), base(base) {
    x = (const float*)(second ? p.x2 : p.x);
    w = (const float*)(second ? p.w2 : p.w);
    one = (p.K + TK - 1) / TK;
    const int64_t all = p.mode == LinearMode::Sum ? 2 * one : one;
    first = all * rank / f.split;
    count = all * (rank + 1) / f.split - first;
    start(first >= one, (first >= one ? first - one : first) * TK);
  }
  __device__ __forceinline__ void start(bool other, int64_t k0) {
    const int64_t sx = f.x_k ? p.sxm : p.sxk, sw = f.w_k ? p.swn : p.swk;
    feed_x.start(other ? (const float*)p.x2 : x, sx, m0, k0, p.M, f.x_k, f.x_packets, C::A_PITCH);
    feed_w.start(other ? (const float*)p.w2 : w, sw, n0, k0, p.N, f.w_k, f.w_packets, C::B_PITCH);
    if constexpr (GATED) feed_up.start((const float*)p.w2, sw, n0, k0, p.N, f.w_k, f.w_packets, C::B_PITCH);
  }
  __device__ __forceinline__ void load(int64_t s) {
    int64_t at = first + s;
    if (p.mode == LinearMode::Sum && at >= one) {             // the second pair of operands
      if (at == one && s > 0) start(true, 0);
      at -= one;
    }
    const uint32_t a = base + (uint32_t)(s % C::STAGES) * (C::STAGE_FLOATS * 4), b = a + C::A_FLOATS * 4;
    const int64_t left = p.K - at * TK;
    feed_x.step(a, C::A_PITCH, left);
    feed_w.step(b, C::B_PITCH, left);
    if constexpr (GATED) feed_up.step(b + COLS * 4, C::B_PITCH, left);
  }
};

// Outputs of a tile whose sums lie in the shared memory of the cluster's blocks, row by row of TN.
template <bool GATED>
__device__ __forceinline__ void finish_tile(const LinearProblem& p, const Form& f, bool second, const float* smem, uint32_t base,
                                            uint32_t rank, int64_t m0, int64_t n0, int rows) {
  constexpr int COLS = GATED ? TN / 2 : TN;
  float* out = (float*)(second ? p.out2 : p.out);
  if (f.split > 1) cluster_sync();
  else __syncthreads();
  // four columns of a row at a time: a share of another block takes hundreds of clocks to come
#pragma unroll 1
  for (int i = threadIdx.x; i < rows * (COLS / 4); i += 256) {
    const int r = (int)rank * rows + i / (COLS / 4), c = i % (COLS / 4) * 4;
    const int64_t m = m0 + r, n = n0 + c;
    if (m >= p.M || n >= p.N) continue;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f), sum2 = sum;
    if (f.split > 1) {
      const uint32_t at = base + (uint32_t)(r * TN + c) * 4;
      for (int q = 0; q < f.split; ++q) {
        add(sum, load_share(at, q));
        if constexpr (GATED) add(sum2, load_share(at + COLS * 4, q));
      }
    } else {
      sum = *reinterpret_cast<const float4*>(&smem[r * TN + c]);
      if constexpr (GATED) sum2 = *reinterpret_cast<const float4*>(&smem[r * TN + COLS + c]);
    }
    float z[4] = {sum.x, sum.y, sum.z, sum.w};
    const float up[4] = {sum2.x, sum2.y, sum2.z, sum2.w};
    const int left = (int)min((int64_t)4, p.N - n);
    float* to = out + m * p.som + n;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= left) break;
      z[j] = GATED ? finish_gated(p, m, n + j, z[j], up[j]) : finish(p, m, n + j, z[j]);
      if (!f.out_packets) to[j] = z[j];
    }
    if (f.out_packets) *reinterpret_cast<float4*>(to) = make_float4(z[0], z[1], z[2], z[3]);
  }
  if (f.split > 1) {
    __syncwarp();
    cluster_sync();                        // nobody still reads this block's sums
  }
}

template <int TM, bool GATED>
__global__ void __launch_bounds__(256, 2) linear_f32_kernel(const LinearProblem p, const Form f) {
  using C = Config<TM>;
  constexpr int ROWS = C::ROWS, STAGES = C::STAGES, COLS = GATED ? TN / 2 : TN;
  extern __shared__ __align__(16) float smem[];
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  uint32_t rank = 0;
  if (f.split > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int64_t m0 = (int64_t)(blockIdx.x / f.split) * TM, n0 = (int64_t)blockIdx.y * COLS;
  const bool second = p.mode == LinearMode::Pair && blockIdx.z == 1;
  const uint32_t base = ptx::smem_u32(smem);
  Steps<TM, GATED> steps(p, f, second, m0, n0, rank, base);
  uint64_t acc[ROWS][4];
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0;

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (s < steps.count) steps.load(s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for (int64_t s = 0; s < steps.count; ++s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();                       // step s has landed for everyone, and step s - 1 is done with
    if (s + STAGES - 1 < steps.count) steps.load(s + STAGES - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const float* a = smem + (s % STAGES) * C::STAGE_FLOATS;
    const float* b = a + C::A_FLOATS;
#pragma unroll
    for (int k = 0; k < TK; ++k) {
      float av[ROWS];
      if constexpr (ROWS == 8) {
        const float4 lo = *reinterpret_cast<const float4*>(&a[k * C::A_PITCH + ty * 4]);
        const float4 hi = *reinterpret_cast<const float4*>(&a[k * C::A_PITCH + 64 + ty * 4]);
        av[0] = lo.x; av[1] = lo.y; av[2] = lo.z; av[3] = lo.w;
        av[4] = hi.x; av[5] = hi.y; av[6] = hi.z; av[7] = hi.w;
      } else {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) av[i] = a[k * C::A_PITCH + ty * ROWS + i];
      }
      const ulonglong2 b0 = *reinterpret_cast<const ulonglong2*>(&b[k * C::B_PITCH + tx * 4]);
      const ulonglong2 b1 = *reinterpret_cast<const ulonglong2*>(&b[k * C::B_PITCH + 64 + tx * 4]);
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const uint64_t aa = ptx::pack_f32x2(av[i], av[i]);
        acc[i][0] = ptx::fma_f32x2(aa, b0.x, acc[i][0]);
        acc[i][1] = ptx::fma_f32x2(aa, b0.y, acc[i][1]);
        acc[i][2] = ptx::fma_f32x2(aa, b1.x, acc[i][2]);
        acc[i][3] = ptx::fma_f32x2(aa, b1.y, acc[i][3]);
      }
    }
  }

  // The block's sums to its shared memory; each block of a cluster then finishes TM / split rows from all of
  // them.  (A rolled loop over shared memory: the activation's code appears once, not per output.)
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = ROWS == 8 ? (i / 4) * 64 + ty * 4 + i % 4 : ty * ROWS + i;
      ulonglong2 v;
      v.x = acc[i][2 * h];
      v.y = acc[i][2 * h + 1];
      *reinterpret_cast<ulonglong2*>(&smem[r * TN + h * 64 + tx * 4]) = v;
    }
  finish_tile<GATED>(p, f, second, smem, base, rank, m0, n0, TM / f.split);
}

// Up to 16 rows: the tile's warps take different k of a step instead of different rows, each holding all 16
// rows of four columns a lane - a weight is then read from shared memory once, not once per warp - and their
// sums are joined at the end, in warp order.
template <bool GATED>
__global__ void __launch_bounds__(256, 2) linear_f32_low_kernel(const LinearProblem p, const Form f) {
  using C = Config<16>;
  constexpr int STAGES = C::STAGES, COLS = GATED ? TN / 2 : TN, WARPS = 8;
  extern __shared__ __align__(16) float smem[];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  uint32_t rank = 0;
  if (f.split > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int64_t m0 = (int64_t)(blockIdx.x / f.split) * 16, n0 = (int64_t)blockIdx.y * COLS;
  const bool second = p.mode == LinearMode::Pair && blockIdx.z == 1;
  const uint32_t base = ptx::smem_u32(smem);
  Steps<16, GATED> steps(p, f, second, m0, n0, rank, base);
  uint64_t acc[16][2];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i][0] = acc[i][1] = 0;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (s < steps.count) steps.load(s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for (int64_t s = 0; s < steps.count; ++s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();
    if (s + STAGES - 1 < steps.count) steps.load(s + STAGES - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const float* a = smem + (s % STAGES) * C::STAGE_FLOATS;
    const float* b = a + C::A_FLOATS;
#pragma unroll
    for (int kk = 0; kk < TK / WARPS; ++kk) {
      const int k = warp * (TK / WARPS) + kk;
      const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(&b[k * C::B_PITCH + lane * 4]);
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&a[k * C::A_PITCH + i]);
        const float av[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t aa = ptx::pack_f32x2(av[j], av[j]);
          acc[i + j][0] = ptx::fma_f32x2(aa, w.x, acc[i + j][0]);
          acc[i + j][1] = ptx::fma_f32x2(aa, w.y, acc[i + j][1]);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    ulonglong2 v;
    v.x = acc[i][0];
    v.y = acc[i][1];
    *reinterpret_cast<ulonglong2*>(&smem[(warp * 16 + i) * TN + lane * 4]) = v;
  }
  __syncthreads();
  for (int i = tid; i < 16 * TN; i += 256) {
    float total = smem[i];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) total += smem[w * 16 * TN + i];
    smem[i] = total;                       // (only this thread reads or writes column i of any warp's part)
  }
  finish_tile<GATED>(p, f, second, smem, base, rank, m0, n0, 16 / f.split);
}

// Two blocks an SM.  K is split while that leaves room for every block at once and eight steps for each; and in
// two where the last round of blocks would leave SMs idle (2048 x 1024 x 4096, 1.73 rounds: 408 -> 372 us): a round
// counts 1, a last one that gives an SM one block at most 0.6, the exchange 0.03.
int split_of(int64_t tiles, int64_t steps, int sm_count) {
  int split = 1;
  while (split < 8 && tiles * split <= sm_count && steps / (split * 2) >= 8) split *= 2;
  auto rounds = [&](int64_t blocks) {
    const double r = (double)blocks / (2.0 * sm_count);
    const double whole = std::floor(r), rest = r - whole;
    return whole + (rest == 0 ? 0.0 : rest <= 0.5 ? 0.6 : 1.0);
  };
  if (split == 1 && steps >= 32 && rounds(2 * tiles) / 2 + 0.06 < rounds(tiles) + 0.03) split = 2;
  return split;
}

template <int TM, bool GATED>
std::string launch_tile(const LinearProblem& p, const LaunchCtx& ctx) {
  using C = Config<TM>;
  Form f{};
  auto packets = [](const void* a, const void* b, int64_t stride) {
    return (((uintptr_t)a | (uintptr_t)b) % 16 == 0 && stride % 4 == 0) ? 1 : 0;
  };
  f.x_k = p.sxk == 1;
  f.w_k = p.swn != 1;
  f.x_packets = packets(p.x, p.x2, p.sxk);
  f.w_packets = packets(p.w, p.w2, p.swk);
  f.out_packets = packets(p.out, p.out2, p.som) && p.N % 4 == 0;
  const int cols = GATED ? TN / 2 : TN;
  const int64_t gx = (p.M + TM - 1) / TM, gy = (p.N + cols - 1) / cols;
  const int64_t gz = p.mode == LinearMode::Pair ? 2 : 1;
  if (gy > 65535) return "more than " + std::to_string(65535 * cols) + " columns";
  if (gx > 0x0fffffff) return "too many rows";
  const int64_t steps = (p.K + TK - 1) / TK * (p.mode == LinearMode::Sum ? 2 : 1);
  f.split = split_of(gx * gy * gz, steps, ctx.sm_count);
  auto kernel = TM == 16 ? linear_f32_low_kernel<GATED> : linear_f32_kernel<TM == 16 ? 32 : TM, GATED>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(gx * f.split), (unsigned)gy, (unsigned)gz);
  config.blockDim = dim3(256);
  config.dynamicSmemBytes = C::SMEM;
  config.stream = ctx.stream;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)f.split;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = f.split > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&config, kernel, p, f);
  ++*ctx.launches;
  if (e != cudaSuccess) {
    cudaGetLastError();
    return std::string("launch failed: ") + cudaGetErrorString(e);
  }
  return std::string();
}

template <int TM>
std::string launch_rows(const LinearProblem& p, const LaunchCtx& ctx) {
  return p.mode == LinearMode::Gated ? launch_tile<TM, true>(p, ctx) : launch_tile<TM, false>(p, ctx);
}

}  // namespace

bool linear_f32_takes(const LinearProblem& p) {
  return p.elt == Elt::F32 && p.K > 0 && (p.sxk == 1 || p.sxm == 1) && (p.swn == 1 || p.swk == 1);
}

std::string launch_linear_f32(const LinearProblem& p, const LaunchCtx& ctx) {
  if (p.M <= 16) return launch_rows<16>(p, ctx);
  if (p.M <= 32) return launch_rows<32>(p, ctx);
  if (p.M <= 64) return launch_rows<64>(p, ctx);
  // the full tile where it - its K split, if need be - fills the SMs, the half tile otherwise
  const int64_t cols = p.mode == LinearMode::Gated ? 64 : 128;
  const int64_t tiles = (p.M + 127) / 128 * ((p.N + cols - 1) / cols) * (p.mode == LinearMode::Pair ? 2 : 1);
  const int64_t steps = (p.K + TK - 1) / TK * (p.mode == LinearMode::Sum ? 2 : 1);
  return tiles * split_of(tiles, steps, ctx.sm_count) >= ctx.sm_count ? launch_rows<128>(p, ctx) : launch_rows<64>(p, ctx);
}

}  // namespace tmc
