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
// Aligned rows of more than 512 bytes are streamed: persistent blocks fetch their next rows by bulk
// copies into a shared-memory ring while they work on the current one, and keep the weights in
// registers.  HBM-bound: each [M, D] operand crosses the memory bus once.  A row belongs to one warp or one
// block, which keeps it in registers between the passes (statistics, second statistics, result), so
// the variance is a true second pass over the centred values and costs no memory traffic.  The
// backward kernel walks its rows with the column sums in registers and leaves one partial row per
// warp or block in scratch memory for a second, ordered summation.  The widest rows do not fit:
// the backward pass of more than 8192 columns (of more than 4096 where a gate or post norm adds its sums
// and the row is not streamed) keeps part of a row in local memory, 0.3 to 2.1 KB a thread by the
// compiler's report; that is traffic between the passes, through L1, which the narrower rows do not have.

#include "ffn_math.cuh"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <atomic>

namespace tmc {
namespace {

using namespace ffn;

// Sum over the THREADS threads of a row (one warp, or a whole block).  `slot` alternates between
// calls, so that a call never overwrites what a slow warp still reads from the one before.
template <int THREADS>
struct RowSum {
  float (*shared)[2][THREADS / 32];   // [slot][value][warp]
  int slot = 0;
  __device__ __forceinline__ void operator()(float& a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if constexpr (THREADS == 32) {
      __syncwarp();                       // what the lanes read before it, they have read
    } else {
      if (threadIdx.x % 32 == 0) shared[slot][0][threadIdx.x / 32] = a;
      __syncthreads();
      a = 0.f;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) a += shared[slot][0][w];
      slot ^= 1;
    }
  }
  __device__ __forceinline__ void operator()(float& a, float& b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (THREADS == 32) {
      __syncwarp();
    } else {
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
  mean = 0.f;
  if (layer) {
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) total += v[i][e];
    sum(total);
    mean = total * inv;
  }
  float square = 0.f;
#pragma unroll
  for (int i = 0; i < PACKS; ++i) {
    if ((i * THREADS + t) * VEC >= D) continue;      // elements past the row are not (0 - mean)
#pragma unroll
    for (int e = 0; e < VEC; ++e) square = fmaf(v[i][e] - mean, v[i][e] - mean, square);
  }
  sum(square);
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

// ---- streamed rows -----------------------------------------------------------------------------

enum Site : uint32_t { kRowFull = 61 };

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

constexpr int MAX_STAGES = 8, MAX_STREAMS = 4;
constexpr size_t kRingBytes = 220 * 1024;      // of an SM's shared memory

// The rows a block will work on, `streams` operands each, fetched ahead into a ring of `stages` slots.
// Slot s holds the rows number s, s + stages, ... of the block; a slot is refilled by the first thread
// once a block-wide barrier has shown that every thread has read it.
struct RowRing {
  const char* base[MAX_STREAMS];
  int64_t pitch;          // bytes from row to row
  uint32_t bytes;         // of a row
  uint32_t smem, bars;
  int streams, stages;
  __device__ __forceinline__ uint32_t slot(int stage, int stream) const {
    return smem + (uint32_t)(stage * streams + stream) * bytes;
  }
  __device__ __forceinline__ void fetch(int stage, int64_t row) const {
    const uint32_t bar = bars + stage * 8;
    ptx::mbar_expect_tx(bar, bytes * streams);
    for (int i = 0; i < streams; ++i) bulk_load(slot(stage, i), base[i] + row * pitch, bytes, bar);
  }
};

// Two neighbouring elements as fp32 in one 64-bit register: the arithmetic below is two-wide throughout
// (at 16 bits an element the passes over a row are bound by instructions as much as by memory).
template <typename T> __device__ __forceinline__ uint64_t widen(uint32_t word);
template <> __device__ __forceinline__ uint64_t widen<__nv_bfloat16>(uint32_t word) {
  return ptx::pack_f32x2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
}
template <> __device__ __forceinline__ uint64_t widen<__half>(uint32_t word) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&word));
  return ptx::pack_f32x2(f.x, f.y);
}
template <typename T> __device__ __forceinline__ uint32_t narrow(uint64_t pair);
template <> __device__ __forceinline__ uint32_t narrow<__nv_bfloat16>(uint64_t pair) {
  float lo, hi;
  ptx::unpack_f32x2(pair, lo, hi);
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t narrow<__half>(uint64_t pair) {
  float lo, hi;
  ptx::unpack_f32x2(pair, lo, hi);
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint64_t both(float v) { return ptx::pack_f32x2(v, v); }
__device__ __forceinline__ float joined(uint64_t pair) {
  float lo, hi;
  ptx::unpack_f32x2(pair, lo, hi);
  return lo + hi;
}

// 16-byte packets of a row or of a weight vector, packet i of thread t being number i * THREADS + t, and
// their elements as pairs.
template <typename T, int THREADS, int PACKS>
struct Packets {
  static constexpr int VEC = 16 / sizeof(T), PAIRS = VEC / 2;
  static __device__ __forceinline__ bool inside(int i, int D, int t) { return (i * THREADS + t) * VEC < D; }
  static __device__ __forceinline__ void unpack(const uint4& raw, uint64_t (&v)[PAIRS]) {
    if constexpr (sizeof(T) == 4) {
      v[0] = ptx::pack_f32x2(__uint_as_float(raw.x), __uint_as_float(raw.y));
      v[1] = ptx::pack_f32x2(__uint_as_float(raw.z), __uint_as_float(raw.w));
    } else {
      v[0] = widen<T>(raw.x);
      v[1] = widen<T>(raw.y);
      v[2] = widen<T>(raw.z);
      v[3] = widen<T>(raw.w);
    }
  }
  static __device__ __forceinline__ uint4 shared_packet(int i, uint32_t row, int D, int t) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (inside(i, D, t))
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w)
                   : "r"(row + (uint32_t)(i * THREADS + t) * 16)
                   : "memory");
    return raw;
  }
  static __device__ __forceinline__ uint4 global_packet(int i, const void* p, int D, int t) {
    return p && inside(i, D, t) ? __ldg(reinterpret_cast<const uint4*>(p) + i * THREADS + t) : make_uint4(0, 0, 0, 0);
  }
  static __device__ __forceinline__ void store(int i, T* p, int D, int t, const uint64_t (&v)[PAIRS]) {
    if (!inside(i, D, t)) return;
    uint4 raw;
    if constexpr (sizeof(T) == 4) {
      raw.x = (uint32_t)v[0]; raw.y = (uint32_t)(v[0] >> 32);
      raw.z = (uint32_t)v[1]; raw.w = (uint32_t)(v[1] >> 32);
    } else {
      raw.x = narrow<T>(v[0]); raw.y = narrow<T>(v[1]); raw.z = narrow<T>(v[2]); raw.w = narrow<T>(v[3]);
    }
    reinterpret_cast<uint4*>(p)[i * THREADS + t] = raw;
  }
  // mean (0 unless `layer`) and reciprocal deviation of the row
  template <typename Sum>
  static __device__ __forceinline__ void statistics(const uint64_t (&v)[PACKS][PAIRS], bool layer, int D, int t, float eps,
                                                    Sum& sum, float& mean, float& rstd) {
    const float inv = 1.f / (float)D;
    mean = 0.f;
    if (layer) {
      uint64_t total = 0;
#pragma unroll
      for (int i = 0; i < PACKS; ++i)
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) total = ptx::add_f32x2(total, v[i][e]);
      mean = joined(total);
      sum(mean);
      mean *= inv;
    }
    const uint64_t shift = both(-mean);
    uint64_t square = 0;
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      if (!inside(i, D, t)) continue;                   // elements past the row are not (0 - mean)
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        const uint64_t c = layer ? ptx::add_f32x2(v[i][e], shift) : v[i][e];
        square = ptx::fma_f32x2(c, c, square);
      }
    }
    float q = joined(square);
    sum(q);
    rstd = 1.f / sqrtf(q * inv + eps);
  }
};

template <typename T, int THREADS, int PACKS>
__global__ void __launch_bounds__(THREADS, THREADS > 256 && THREADS < 512 ? 2 : 512 / THREADS)
residual_norm_stream_kernel(const NormProblem p, int stages, DeviceStatus* status) {
  using P = Packets<T, THREADS, PACKS>;
  constexpr int PAIRS = P::PAIRS;
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ __align__(8) uint64_t bars[MAX_STAGES];
  __shared__ int abort_flag;
  __shared__ float shared[2][2][THREADS / 32];
  RowSum<THREADS> sum{shared};
  const int t = threadIdx.x, D = (int)p.D;
  ptx::WaitCtx wc{&abort_flag, status};
  RowRing ring;
  ring.pitch = p.stride * (int64_t)sizeof(T);
  ring.bytes = (uint32_t)(D * sizeof(T));
  ring.smem = ptx::smem_u32(ring_smem);
  ring.bars = ptx::smem_u32(bars);
  ring.stages = stages;
  ring.streams = p.block ? 2 : 1;
  ring.base[0] = (const char*)p.residual;
  ring.base[1] = (const char*)p.block;
  if (t == 0) {
    abort_flag = 0;
    for (int s = 0; s < stages; ++s) ptx::mbar_init(ring.bars + s * 8, 1);
    ptx::fence_barrier_init();
    for (int s = 0; s < stages; ++s) {
      const int64_t row = blockIdx.x + (int64_t)s * gridDim.x;
      if (row < p.M) ring.fetch(s, row);
    }
  }
  // the weights stay in registers, as packets; gate and post weight as one factor
  uint4 weight[PACKS], bias[PACKS];
  uint64_t factor[PACKS][PAIRS];
#pragma unroll
  for (int i = 0; i < PACKS; ++i) {
    weight[i] = P::global_packet(i, p.weight, D, t);
    bias[i] = P::global_packet(i, p.bias, D, t);
    uint64_t g[PAIRS];
    P::unpack(P::global_packet(i, p.gate ? p.gate : p.post_weight, D, t), factor[i]);
    if (p.gate && p.post_weight) {
      P::unpack(P::global_packet(i, p.post_weight, D, t), g);
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) factor[i][e] = ptx::mul_f32x2(factor[i][e], g[e]);
    }
  }
  const bool scaled = p.gate || p.post_weight;
  const uint64_t scale = both(p.scale);
  __syncthreads();

  int stage = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    // A wait that gives up leaves the block in step: it goes on with whatever is there and the launch is
    // reported as failed.
    ptx::mbar_wait(ring.bars + stage * 8, phase, wc, kRowFull);
    uint64_t s[PACKS][PAIRS];
    float mean_y = 0.f, rstd_y = 0.f, mean, rstd;
    if (p.block) {
#pragma unroll
      for (int i = 0; i < PACKS; ++i) P::unpack(P::shared_packet(i, ring.slot(stage, 1), D, t), s[i]);
      if (p.post_weight) {
        P::statistics(s, p.layer, D, t, p.eps, sum, mean_y, rstd_y);
        const uint64_t shift = both(-mean_y), r = both(rstd_y);
#pragma unroll
        for (int i = 0; i < PACKS; ++i)
#pragma unroll
          for (int e = 0; e < PAIRS; ++e) {
            if (p.layer) s[i][e] = ptx::add_f32x2(s[i][e], shift);
            s[i][e] = ptx::mul_f32x2(s[i][e], r);
          }
      }
    }
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      uint64_t r[PAIRS];
      P::unpack(P::shared_packet(i, ring.slot(stage, 0), D, t), r);
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        if (scaled) s[i][e] = ptx::mul_f32x2(s[i][e], factor[i][e]);
        s[i][e] = p.block ? ptx::fma_f32x2(scale, r[e], s[i][e]) : ptx::mul_f32x2(scale, r[e]);
      }
      if (p.sum) P::store(i, (T*)p.sum + row * p.stride, D, t, s[i]);
    }
    P::statistics(s, p.layer, D, t, p.eps, sum, mean, rstd);
    // (its block-wide barrier came after every thread's reads of the slot)
    const int64_t next = row + (int64_t)stages * gridDim.x;
    if (t == 0) {
      if (next < p.M) ring.fetch(stage, next);
      if (p.stats) *reinterpret_cast<float4*>(p.stats + row * 4) = make_float4(mean, rstd, mean_y, rstd_y);
    }
    const uint64_t shift = both(-mean), r = both(rstd);
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      uint64_t w[PAIRS], b[PAIRS];
      P::unpack(weight[i], w);
      if (p.bias) P::unpack(bias[i], b);
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        if (p.layer) s[i][e] = ptx::add_f32x2(s[i][e], shift);
        s[i][e] = ptx::mul_f32x2(s[i][e], r);
        s[i][e] = p.bias ? ptx::fma_f32x2(s[i][e], w[e], b[e]) : ptx::mul_f32x2(s[i][e], w[e]);
      }
      P::store(i, (T*)p.normed + row * p.stride, D, t, s[i]);
    }
    if (++stage == stages) { stage = 0; phase ^= 1; }
  }
}

// BRANCH: gate or post norm.  FULL: layer norm, or dbias is wanted.  With a post norm, dgate and
// dpost are both the sum of ds y^ over the rows, times post_weight and times gate: one sum for the two.
template <typename T, int THREADS, int PACKS, bool BRANCH, bool FULL>
__global__ void __launch_bounds__(THREADS, 512 / THREADS)
residual_norm_bwd_stream_kernel(const NormProblem p, int stages, float* __restrict__ partial, DeviceStatus* status) {
  using P = Packets<T, THREADS, PACKS>;
  constexpr int PAIRS = P::PAIRS;
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ __align__(8) uint64_t bars[MAX_STAGES];
  __shared__ int abort_flag;
  __shared__ float shared[2][2][THREADS / 32];
  RowSum<THREADS> sum{shared};
  const int t = threadIdx.x, D = (int)p.D;
  const float inv = 1.f / (float)D;
  ptx::WaitCtx wc{&abort_flag, status};
  RowRing ring;
  ring.pitch = p.stride * (int64_t)sizeof(T);
  ring.bytes = (uint32_t)(D * sizeof(T));
  ring.smem = ptx::smem_u32(ring_smem);
  ring.bars = ptx::smem_u32(bars);
  ring.stages = stages;
  ring.streams = 2;
  ring.base[0] = (const char*)p.sum;
  ring.base[1] = (const char*)p.dnormed;
  const int at_dsum = p.dsum ? ring.streams : 0;
  if (p.dsum) ring.base[ring.streams++] = (const char*)p.dsum;
  const int at_block = BRANCH ? ring.streams : 0;
  if (BRANCH) ring.base[ring.streams++] = (const char*)p.block;
  if (t == 0) {
    abort_flag = 0;
    for (int s = 0; s < stages; ++s) ptx::mbar_init(ring.bars + s * 8, 1);
    ptx::fence_barrier_init();
    for (int s = 0; s < stages; ++s) {
      const int64_t row = blockIdx.x + (int64_t)s * gridDim.x;
      if (row < p.M) ring.fetch(s, row);
    }
  }
  uint4 weight[PACKS];
  uint64_t factor[BRANCH ? PACKS : 1][PAIRS];           // gate times post weight
  uint64_t sum_w[PACKS][PAIRS], sum_b[FULL ? PACKS : 1][PAIRS], sum_y[BRANCH ? PACKS : 1][PAIRS];
#pragma unroll
  for (int i = 0; i < PACKS; ++i) {
    weight[i] = P::global_packet(i, p.weight, D, t);
    if constexpr (BRANCH) {
      uint64_t g[PAIRS];
      P::unpack(P::global_packet(i, p.gate ? p.gate : p.post_weight, D, t), factor[i]);
      if (p.gate && p.post_weight) {
        P::unpack(P::global_packet(i, p.post_weight, D, t), g);
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) factor[i][e] = ptx::mul_f32x2(factor[i][e], g[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < PAIRS; ++e) {
      sum_w[i][e] = 0;
      if (FULL) sum_b[i][e] = 0;
      if (BRANCH) sum_y[i][e] = 0;
    }
  }
  const uint64_t scale = both(p.scale);
  __syncthreads();

  int stage = 0;
  uint32_t phase = 0;
  // the statistics come a row ahead
  const float4* stats = reinterpret_cast<const float4*>(p.stats);
  float4 st_next = blockIdx.x < p.M ? __ldg(stats + blockIdx.x) : make_float4(0.f, 0.f, 0.f, 0.f);
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const float4 st = st_next;
    if (row + gridDim.x < p.M) st_next = __ldg(stats + row + gridDim.x);
    ptx::mbar_wait(ring.bars + stage * 8, phase, wc, kRowFull);
    uint64_t hat[PACKS][PAIRS], h[PACKS][PAIRS];
    uint64_t c1p = 0, c2p = 0;
    const uint64_t r = both(st.y);
    {
      const uint64_t shift = both(-st.x);
#pragma unroll
      for (int i = 0; i < PACKS; ++i) {
        uint64_t dn[PAIRS];
        P::unpack(P::shared_packet(i, ring.slot(stage, 0), D, t), hat[i]);
        P::unpack(P::shared_packet(i, ring.slot(stage, 1), D, t), dn);
        P::unpack(weight[i], h[i]);
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {
          if (FULL) hat[i][e] = ptx::add_f32x2(hat[i][e], shift);
          hat[i][e] = ptx::mul_f32x2(hat[i][e], r);
          sum_w[i][e] = ptx::fma_f32x2(dn[e], hat[i][e], sum_w[i][e]);
          if (FULL) sum_b[i][e] = ptx::add_f32x2(sum_b[i][e], dn[e]);
          h[i][e] = ptx::mul_f32x2(dn[e], h[i][e]);
          c1p = ptx::fma_f32x2(h[i][e], hat[i][e], c1p);
          if (FULL) c2p = ptx::add_f32x2(c2p, h[i][e]);
        }
      }
    }
    float c1 = joined(c1p), c2 = joined(c2p);
    if (FULL) sum(c1, c2);
    else sum(c1);
    // Its block-wide barrier came after every thread was done with the row before: that slot is free.
    if (t == 0 && row != blockIdx.x) {
      const int64_t next = row + (int64_t)(stages - 1) * gridDim.x;
      if (next < p.M) ring.fetch(stage == 0 ? stages - 1 : stage - 1, next);
    }
    const uint64_t c1n = both(-c1 * inv), c2n = both(FULL && p.layer ? -c2 * inv : 0.f);
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      uint64_t ds[PAIRS], out[PAIRS];
      if (p.dsum) {
        P::unpack(P::shared_packet(i, ring.slot(stage, at_dsum), D, t), ds);
      } else {
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) ds[e] = 0;
      }
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        uint64_t v = ptx::fma_f32x2(hat[i][e], c1n, h[i][e]);
        if (FULL) v = ptx::add_f32x2(v, c2n);
        h[i][e] = ptx::fma_f32x2(r, v, ds[e]);             // ds
        out[e] = ptx::mul_f32x2(h[i][e], scale);
      }
      if (p.dresidual) P::store(i, (T*)p.dresidual + row * p.stride, D, t, out);
    }
    if constexpr (BRANCH) {
      const bool post = p.post_weight != nullptr;
      const uint64_t ry = both(st.w), shift = both(-st.z);
      uint64_t d1p = 0, d2p = 0;
#pragma unroll
      for (int i = 0; i < PACKS; ++i) {
        P::unpack(P::shared_packet(i, ring.slot(stage, at_block), D, t), hat[i]);
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {
          if (post) {
            if (FULL) hat[i][e] = ptx::add_f32x2(hat[i][e], shift);
            hat[i][e] = ptx::mul_f32x2(hat[i][e], ry);
          }
          sum_y[i][e] = ptx::fma_f32x2(h[i][e], hat[i][e], sum_y[i][e]);
          h[i][e] = ptx::mul_f32x2(h[i][e], factor[i][e]);
          if (post) {
            d1p = ptx::fma_f32x2(h[i][e], hat[i][e], d1p);
            if (FULL) d2p = ptx::add_f32x2(d2p, h[i][e]);
          }
        }
      }
      if (post) {
        float d1 = joined(d1p), d2 = joined(d2p);
        if (FULL) sum(d1, d2);
        else sum(d1);
        const uint64_t d1n = both(-d1 * inv), d2n = both(FULL && p.layer ? -d2 * inv : 0.f);
#pragma unroll
        for (int i = 0; i < PACKS; ++i)
#pragma unroll
          for (int e = 0; e < PAIRS; ++e) {
            uint64_t v = ptx::fma_f32x2(hat[i][e], d1n, h[i][e]);
            if (FULL) v = ptx::add_f32x2(v, d2n);
            h[i][e] = ptx::mul_f32x2(ry, v);
          }
      }
    }
    if (p.dblock) {
#pragma unroll
      for (int i = 0; i < PACKS; ++i) P::store(i, (T*)p.dblock + row * p.stride, D, t, h[i]);
    }
    if (++stage == stages) { stage = 0; phase ^= 1; }
  }

  const int64_t set = (int64_t)gridDim.x * D;
  float* to = partial + (int64_t)blockIdx.x * D;
  // `times` (or null): a weight vector the sums are multiplied by
  auto keep = [&](const uint64_t (&v)[PACKS][PAIRS], const void* times) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      if (!P::inside(i, D, t)) continue;
      uint64_t f[PAIRS];
      P::unpack(P::global_packet(i, times, D, t), f);
#pragma unroll
      for (int e = 0; e < PAIRS; ++e)
        reinterpret_cast<uint64_t*>(to + (i * THREADS + t) * P::VEC)[e] = times ? ptx::mul_f32x2(v[i][e], f[e]) : v[i][e];
    }
    to += set;
  };
  if (p.dweight) keep(sum_w, nullptr);
  if constexpr (FULL) {
    if (p.dbias) keep(sum_b, nullptr);
  }
  if constexpr (BRANCH) {
    if (p.dgate) keep(sum_y, p.post_weight);
    if (p.dpost) keep(sum_y, p.gate);
  }
}

// The gradients wanted of the weight vectors, in the order of the partial sums.
int sum_outputs(const NormProblem& p, void* (&outs)[kMaxColumnSums]) {
  int sets = 0;
  for (void* q : {p.dweight, p.dbias, p.dgate, p.dpost})
    if (q) outs[sets++] = q;
  return sets;
}

template <typename T, int THREADS, int PACKS>
std::string launch_stream(const NormProblem& p, const LaunchCtx& ctx, bool backward) {
  const bool branch = backward && (p.gate || p.post_weight);
  const bool full = p.layer || p.dbias;
  const int streams = backward ? 2 + (p.dsum ? 1 : 0) + (branch ? 1 : 0) : (p.block ? 2 : 1);
  const size_t row = (size_t)streams * (size_t)p.D * sizeof(T);
  // Registers hold 512 threads an SM (two forward blocks of 320 or 384: 5120 columns in 98 us instead of 156);
  // the ring takes what is left of the shared memory, at most MAX_STAGES rows a block.
  const int want = !backward && THREADS > 256 && THREADS < 512 ? 2 : 512 / THREADS;
  const size_t budget = kRingBytes / want;
  // (the backward ring refills a slot one row late, so it needs two)
  const int stages = (int)std::min<size_t>(MAX_STAGES, std::max<size_t>(backward ? 2 : 1, budget / row));
  const size_t smem = stages * row;
  const void* kernel =
      !backward ? (const void*)residual_norm_stream_kernel<T, THREADS, PACKS>
      : branch  ? (full ? (const void*)residual_norm_bwd_stream_kernel<T, THREADS, PACKS, true, true>
                        : (const void*)residual_norm_bwd_stream_kernel<T, THREADS, PACKS, true, false>)
                : (full ? (const void*)residual_norm_bwd_stream_kernel<T, THREADS, PACKS, false, true>
                        : (const void*)residual_norm_bwd_stream_kernel<T, THREADS, PACKS, false, false>);
  // blocks of this kernel and ring an SM holds, asked for once: the kernel's number, the ring's size, the answer
  static std::atomic<uint64_t> known[5];
  const int which = !backward ? 0 : 1 + (branch ? 2 : 0) + (full ? 1 : 0);
  cudaError_t e = cudaSuccess;
  uint64_t entry = known[which].load(std::memory_order_relaxed);
  if (entry >> 8 != smem) {
    int blocks = 1;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingBytes);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, THREADS, smem);
    if (e != cudaSuccess) return cudaGetErrorString(e);
    entry = (uint64_t)smem << 8 | (uint64_t)std::max(blocks, 1);
    known[which].store(entry, std::memory_order_relaxed);
  }
  const int resident = (int)(entry & 255);
  const int64_t grid = std::min<int64_t>(std::max<int64_t>(p.M, 1), (int64_t)ctx.sm_count * resident);
  if (!backward) {
    residual_norm_stream_kernel<T, THREADS, PACKS><<<(unsigned)grid, THREADS, smem, ctx.stream>>>(p, stages, ctx.status);
    ++*ctx.launches;
  } else {
    void* outs[kMaxColumnSums] = {};
    const int sets = sum_outputs(p, outs);
    void* partial = nullptr;
    if (sets) {
      std::string err = scratch_alloc(ctx, (size_t)sets * (size_t)grid * (size_t)p.D * 4, &partial);
      if (!err.empty()) return err;
    }
    float* part = (float*)partial;
    int n = stages;
    DeviceStatus* status = ctx.status;
    void* args[] = {(void*)&p, &n, &part, &status};
    e = cudaLaunchKernel(kernel, dim3((unsigned)grid), dim3(THREADS), args, smem, ctx.stream);
    ++*ctx.launches;
    if (sets) {
      launch_column_sums(p.elt, part, grid, p.D, sets, outs, ctx);
      scratch_free(ctx, partial);
    }
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  else cudaGetLastError();
  if (e != cudaSuccess) return std::string("residual norm launch failed: ") + cudaGetErrorString(e);
  return std::string();
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
    static std::atomic<int> known[2];      // blocks of this kernel an SM holds
    int resident = known[branch].load(std::memory_order_relaxed);
    if (!resident) {
      int n = 0;
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, BLOCK, 0) != cudaSuccess || n < 1) n = 1;
      known[branch].store(resident = n, std::memory_order_relaxed);
    }
    // (no rows: one block, whose sums are zero)
    const int64_t grid = std::min<int64_t>(std::max<int64_t>(blocks, 1), (int64_t)ctx.sm_count * resident);
    const int64_t groups = grid * ROWS;
    void* outs[kMaxColumnSums] = {};
    const int sets = sum_outputs(p, outs);
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
    // (two rows of the backward pass's four operands, or one of the forward's, have to fit; at 64 packets a warp
    // to a row without the ring took 104 us forward and 325 back where this takes 110 and 160)
    if (packets > 32 && (size_t)p.D * sizeof(T) * (backward ? 8 : 2) <= kRingBytes) {
      // As few warps a row as hold it: the block-wide sums are what a row waits for (4096 bf16 columns
      // forward and back: 91 and 158 us with two packets a thread, 132 and 173 with one).
      if (packets <= 64) return launch_stream<T, 32, 2>(p, ctx, backward);
      if (packets <= 128) return launch_stream<T, 64, 2>(p, ctx, backward);
      if (packets <= 256) return launch_stream<T, 128, 2>(p, ctx, backward);
      if (packets <= 512) return launch_stream<T, 256, 2>(p, ctx, backward);
      if (packets <= 640) return launch_stream<T, 320, 2>(p, ctx, backward);
      if (packets <= 768) return launch_stream<T, 384, 2>(p, ctx, backward);
      if (packets <= 1024) return launch_stream<T, 512, 2>(p, ctx, backward);
      if (packets <= 2048) return launch_stream<T, 512, 4>(p, ctx, backward);
    }
    if (packets <= 32) return launch_sized<T, VEC, 32, 1>(p, ctx, backward);
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
