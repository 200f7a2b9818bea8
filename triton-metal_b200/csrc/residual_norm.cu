// residual_norm_kernel and residual_norm_bwd_kernel: the join of a block's output with the residual
// stream, with the norm behind the block (optional) and the norm in front of the next one.
//
//   t = post_weight ? N(block) * post_weight : block
//   s = scale * residual + gate * t            (stored, rounded once)
//   normed = N(s) * weight + bias              (from the unrounded s)
//   N(v) = (v - mean(v)) / sqrt(var(v) + eps), or v / sqrt(mean(v^2) + eps)
//
// Backward, with s^ = (s - mean) * r, y^ likewise from block, h = dnormed * weight:
//   ds = dsum + r (h - [mean(h)] - s^ mean(h s^))
//   dresidual = scale ds;  dt = gate ds;  dblock = dt, or r_y (h_y - [mean(h_y)] - y^ mean(h_y y^))
//   with h_y = dt post_weight;  dweight = sum dnormed s^;  dbias = sum dnormed;
//   dgate = sum ds t;  dpost = sum dt y^       ([mean(...)]: layer norm only; sums over the rows)
//
// HBM-bound: each [M, D] operand crosses the memory bus once.  A row belongs to one warp or one
// block, which keeps it in registers between the passes (statistics, second statistics, result), so
// the variance is a true second pass over the centred values and costs no memory traffic.  The
// backward kernel walks its rows with the column sums in registers and leaves one partial row per
// warp or block in scratch memory for a second, ordered summation.

#include "ffn_math.cuh"

#include <algorithm>

namespace tmc {
namespace {

using namespace ffn;

// Sum over the THREADS threads of a row (one warp, or a whole block).  `slot` alternates between
// calls, so that a call never overwrites what a slow warp still reads from the one before.
template <int THREADS>
struct RowSum {
  float (*shared)[2][THREADS / 32];   // [slot][value][warp]
  int slot = 0;
  __device__ __forceinline__ void operator()(float& a, float& b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (THREADS > 32) {
      const int warp = threadIdx.x / 32;
      if (threadIdx.x % 32 == 0) {
        shared[slot][0][warp] = a;
        shared[slot][1][warp] = b;
      }
      __syncthreads();
      a = 0.f;
      b = 0.f;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) {
        a += shared[slot][0][w];
        b += shared[slot][1][w];
      }
      slot ^= 1;
    }
  }
};

// A row (or a vector of D weights) in registers: PACKS packets of VEC elements, packet i of thread t
// being number i * THREADS + t.
template <typename T, int VEC, int THREADS, int PACKS>
struct Row {
  static __device__ __forceinline__ int column(int i, int t) { return (i * THREADS + t) * VEC; }
  static __device__ __forceinline__ void load(const T* p, int64_t D, int t, float (&v)[PACKS][VEC]) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int c = column(i, t);
      if (c < D) load_vec<T, VEC>(p + c, v[i]);
      else
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = 0.f;
    }
  }
  static __device__ __forceinline__ void store(T* p, int64_t D, int t, const float (&v)[PACKS][VEC]) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int c = column(i, t);
      if (c < D) store_vec<T, VEC>(p + c, v[i]);
    }
  }
};

// mean (0 unless LAYER) and reciprocal deviation of the row
template <int VEC, int THREADS, int PACKS, typename Sum>
__device__ __forceinline__ void statistics(const float (&v)[PACKS][VEC], bool layer, int64_t D, int t, float eps,
                                           Sum& sum, float& mean, float& rstd) {
  const float inv = 1.f / (float)D;
  float unused = 0.f;
  mean = 0.f;
  if (layer) {
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) total += v[i][e];
    sum(total, unused);
    mean = total * inv;
  }
  float square = 0.f;
#pragma unroll
  for (int i = 0; i < PACKS; ++i) {
    if ((i * THREADS + t) * VEC >= D) continue;      // elements past the row are not (0 - mean)
#pragma unroll
    for (int e = 0; e < VEC; ++e) square = fmaf(v[i][e] - mean, v[i][e] - mean, square);
  }
  sum(square, unused);
  rstd = 1.f / sqrtf(square * inv + eps);
}

template <typename T, int VEC, int THREADS, int PACKS>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS) residual_norm_kernel(const NormProblem p) {
  using R = Row<T, VEC, THREADS, PACKS>;
  constexpr int ROWS = THREADS < 128 ? 128 / THREADS : 1;      // rows of a block
  __shared__ float shared[2][2][THREADS / 32];
  RowSum<THREADS> sum{shared};
  const int t = ROWS > 1 ? threadIdx.x % THREADS : threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / THREADS : 0);
  if (row >= p.M) return;                                       // whole warps (ROWS > 1), or nothing
  const int64_t at = row * p.stride;
  float s[PACKS][VEC];
  R::load((const T*)p.residual + at, p.D, t, s);
  float mean_y = 0.f, rstd_y = 0.f, mean, rstd;
  if (p.block) {
    float y[PACKS][VEC], f[PACKS][VEC];
    R::load((const T*)p.block + at, p.D, t, y);
    if (p.post_weight) {
      statistics<VEC, THREADS, PACKS>(y, p.layer, p.D, t, p.eps, sum, mean_y, rstd_y);
      R::load((const T*)p.post_weight, p.D, t, f);
#pragma unroll
      for (int i = 0; i < PACKS; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[i][e] = (y[i][e] - mean_y) * rstd_y * f[i][e];
    }
    if (p.gate) {
      R::load((const T*)p.gate, p.D, t, f);
#pragma unroll
      for (int i = 0; i < PACKS; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[i][e] *= f[i][e];
    }
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[i][e] = fmaf(p.scale, s[i][e], y[i][e]);
  } else {
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[i][e] *= p.scale;
  }
  if (p.sum) R::store((T*)p.sum + at, p.D, t, s);
  statistics<VEC, THREADS, PACKS>(s, p.layer, p.D, t, p.eps, sum, mean, rstd);
  if (p.stats && t == 0)
    *reinterpret_cast<float4*>(p.stats + row * 4) = make_float4(mean, rstd, mean_y, rstd_y);
  float w[PACKS][VEC];
  R::load((const T*)p.weight, p.D, t, w);
#pragma unroll
  for (int i = 0; i < PACKS; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[i][e] = (s[i][e] - mean) * rstd * w[i][e];
  if (p.bias) {
    R::load((const T*)p.bias, p.D, t, w);
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[i][e] += w[i][e];
  }
  R::store((T*)p.normed + at, p.D, t, s);
}

// BRANCH: the gate or the post norm is there, so dgate / dpost are summed too.  Partial sums:
// [dweight, dbias, dgate, dpost][row group][D].
template <typename T, int VEC, int THREADS, int PACKS, bool BRANCH>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS)
residual_norm_bwd_kernel(const NormProblem p, float* __restrict__ partial, int64_t groups) {
  using R = Row<T, VEC, THREADS, PACKS>;
  constexpr int ROWS = THREADS < 128 ? 128 / THREADS : 1;
  __shared__ float shared[2][2][THREADS / 32];
  RowSum<THREADS> sum{shared};
  const int t = ROWS > 1 ? threadIdx.x % THREADS : threadIdx.x;
  const int64_t group = (int64_t)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / THREADS : 0);
  const float inv = 1.f / (float)p.D;
  float sum_w[PACKS][VEC], sum_b[PACKS][VEC], sum_g[BRANCH ? PACKS : 1][VEC], sum_p[BRANCH ? PACKS : 1][VEC];
#pragma unroll
  for (int i = 0; i < PACKS; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sum_w[i][e] = sum_b[i][e] = 0.f;
      if (BRANCH) sum_g[i][e] = sum_p[i][e] = 0.f;
    }
  float w[PACKS][VEC];
  R::load((const T*)p.weight, p.D, t, w);

  for (int64_t row = group; row < p.M; row += groups) {
    const int64_t at = row * p.stride;
    const float4 st = *reinterpret_cast<const float4*>(p.stats + row * 4);
    float s[PACKS][VEC], dn[PACKS][VEC], ds[PACKS][VEC];
    R::load((const T*)p.sum + at, p.D, t, s);
    R::load((const T*)p.dnormed + at, p.D, t, dn);
    if (p.dsum) R::load((const T*)p.dsum + at, p.D, t, ds);
    else
#pragma unroll
      for (int i = 0; i < PACKS; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) ds[i][e] = 0.f;
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float hat = (s[i][e] - st.x) * st.y;
        sum_w[i][e] = fmaf(dn[i][e], hat, sum_w[i][e]);
        sum_b[i][e] += dn[i][e];
        dn[i][e] *= w[i][e];                         // h
        s[i][e] = hat;
        c1 = fmaf(dn[i][e], hat, c1);
        c2 += dn[i][e];
      }
    sum(c1, c2);
    c1 *= inv;
    c2 = p.layer ? c2 * inv : 0.f;
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) ds[i][e] = fmaf(st.y, dn[i][e] - c2 - s[i][e] * c1, ds[i][e]);
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[i][e] = ds[i][e] * p.scale;
    if (p.dresidual) R::store((T*)p.dresidual + at, p.D, t, s);
    if constexpr (BRANCH) {
      float y[PACKS][VEC], f[PACKS][VEC];
      R::load((const T*)p.block + at, p.D, t, y);
      if (p.post_weight) {
        float g[PACKS][VEC];
        R::load((const T*)p.post_weight, p.D, t, f);
        if (p.gate) R::load((const T*)p.gate, p.D, t, g);
        float d1 = 0.f, d2 = 0.f;
#pragma unroll
        for (int i = 0; i < PACKS; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float hat = (y[i][e] - st.z) * st.w;
            if (p.gate) {
              sum_g[i][e] = fmaf(ds[i][e], hat * f[i][e], sum_g[i][e]);
              ds[i][e] *= g[i][e];                   // dt
            }
            sum_p[i][e] = fmaf(ds[i][e], hat, sum_p[i][e]);
            ds[i][e] *= f[i][e];                     // h_y
            y[i][e] = hat;
            d1 = fmaf(ds[i][e], hat, d1);
            d2 += ds[i][e];
          }
        sum(d1, d2);
        d1 *= inv;
        d2 = p.layer ? d2 * inv : 0.f;
#pragma unroll
        for (int i = 0; i < PACKS; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) ds[i][e] = st.w * (ds[i][e] - d2 - y[i][e] * d1);
      } else {
        R::load((const T*)p.gate, p.D, t, f);
#pragma unroll
        for (int i = 0; i < PACKS; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            sum_g[i][e] = fmaf(ds[i][e], y[i][e], sum_g[i][e]);
            ds[i][e] *= f[i][e];
          }
      }
    }
    if (p.dblock) R::store((T*)p.dblock + at, p.D, t, ds);
  }
  if (group < groups) {
    const int64_t set = groups * p.D;
    auto keep = [&](int which, const float (&v)[PACKS][VEC]) {
      float* to = partial + which * set + group * p.D;
#pragma unroll
      for (int i = 0; i < PACKS; ++i) {
        const int c = R::column(i, t);
        if (c >= p.D) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) to[c + e] = v[i][e];
      }
    };
    int next = 0;
    if (p.dweight) keep(next++, sum_w);
    if (p.dbias) keep(next++, sum_b);
    if constexpr (BRANCH) {
      if (p.dgate) keep(next++, sum_g);
      if (p.dpost) keep(next++, sum_p);
    }
  }
}

template <typename T, int VEC, int THREADS, int PACKS>
std::string launch_sized(const NormProblem& p, const LaunchCtx& ctx, bool backward) {
  constexpr int BLOCK = THREADS < 128 ? 128 : THREADS, ROWS = BLOCK / THREADS;
  const int64_t blocks = (p.M + ROWS - 1) / ROWS;
  if (!backward) {
    if (blocks > 0x7fffffff) return "too many rows";
    residual_norm_kernel<T, VEC, THREADS, PACKS><<<(unsigned)blocks, BLOCK, 0, ctx.stream>>>(p);
    ++*ctx.launches;
  } else {
    const bool branch = p.gate || p.post_weight;
    auto kernel = branch ? residual_norm_bwd_kernel<T, VEC, THREADS, PACKS, true>
                         : residual_norm_bwd_kernel<T, VEC, THREADS, PACKS, false>;
    static int resident[2] = {0, 0};       // blocks of this kernel an SM holds
    if (!resident[branch]) {
      int n = 0;
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, BLOCK, 0) != cudaSuccess || n < 1) n = 1;
      resident[branch] = n;
    }
    // (no rows: one block, whose sums are zero)
    const int64_t grid = std::min<int64_t>(std::max<int64_t>(blocks, 1), (int64_t)ctx.sm_count * resident[branch]);
    const int64_t groups = grid * ROWS;
    void* outs[kMaxColumnSums] = {};
    int sets = 0;
    if (p.dweight) outs[sets++] = p.dweight;
    if (p.dbias) outs[sets++] = p.dbias;
    if (p.dgate) outs[sets++] = p.dgate;
    if (p.dpost) outs[sets++] = p.dpost;
    void* partial = nullptr;
    if (sets) {
      std::string err = scratch_alloc(ctx, (size_t)sets * (size_t)groups * (size_t)p.D * 4, &partial);
      if (!err.empty()) return err;
    }
    kernel<<<(unsigned)grid, BLOCK, 0, ctx.stream>>>(p, (float*)partial, groups);
    ++*ctx.launches;
    if (sets) {
      launch_column_sums(p.elt, (const float*)partial, groups, p.D, sets, outs, ctx);
      scratch_free(ctx, partial);
    }
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return std::string("residual norm launch failed: ") + cudaGetErrorString(e);
  return std::string();
}

template <typename T>
std::string launch_typed(const NormProblem& p, const LaunchCtx& ctx, bool backward) {
  constexpr int VEC = 16 / sizeof(T);
  uintptr_t bases = 0;
  for (const void* q : {p.residual, p.block, p.weight, p.bias, p.gate, p.post_weight, (const void*)p.sum,
                        (const void*)p.normed, p.dnormed, p.dsum, (const void*)p.dresidual, (const void*)p.dblock})
    bases |= (uintptr_t)q;
  if (bases % 16 == 0 && p.stride % VEC == 0 && p.D % VEC == 0) {
    const int64_t packets = p.D / VEC;
    if (packets <= 32) return launch_sized<T, VEC, 32, 1>(p, ctx, backward);
    if (packets <= 64) return launch_sized<T, VEC, 32, 2>(p, ctx, backward);
    if (packets <= 128) return launch_sized<T, VEC, 128, 1>(p, ctx, backward);
    if (packets <= 256) return launch_sized<T, VEC, 256, 1>(p, ctx, backward);
    if (packets <= 512) return launch_sized<T, VEC, 512, 1>(p, ctx, backward);
    if (packets <= 1024) return launch_sized<T, VEC, 512, 2>(p, ctx, backward);
    if (packets <= 2048) return launch_sized<T, VEC, 512, 4>(p, ctx, backward);
    if constexpr (VEC == 4) return launch_sized<T, VEC, 512, 8>(p, ctx, backward);
  }
  if (p.D <= 128) return launch_sized<T, 1, 32, 4>(p, ctx, backward);
  if (p.D <= 512) return launch_sized<T, 1, 128, 4>(p, ctx, backward);
  if (p.D <= 1024) return launch_sized<T, 1, 256, 4>(p, ctx, backward);
  if (p.D <= 2048) return launch_sized<T, 1, 512, 4>(p, ctx, backward);
  if (p.D <= 4096) return launch_sized<T, 1, 512, 8>(p, ctx, backward);
  if (p.D <= 8192) return launch_sized<T, 1, 512, 16>(p, ctx, backward);
  return launch_sized<T, 1, 512, 32>(p, ctx, backward);
}

std::string launch(const NormProblem& p, const LaunchCtx& ctx, bool backward) {
  if (p.D > kNormMaxColumns) return "more than " + std::to_string(kNormMaxColumns) + " columns";
  if (p.elt == Elt::F32) return launch_typed<float>(p, ctx, backward);
  if (p.elt == Elt::BF16) return launch_typed<__nv_bfloat16>(p, ctx, backward);
  return launch_typed<__half>(p, ctx, backward);
}

}  // namespace

std::string launch_residual_norm(const NormProblem& p, const LaunchCtx& ctx) { return launch(p, ctx, false); }
std::string launch_residual_norm_bwd(const NormProblem& p, const LaunchCtx& ctx) { return launch(p, ctx, true); }

}  // namespace tmc
