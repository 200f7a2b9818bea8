// The element-wise part of the feed-forward backward passes.
//
//   activation_bwd_kernel        dz = dout * act'(pre),  dbias[n] = sum_m dz[m, n]
//   gated_activation_bwd_kernel  dgate = dout * up * act'(gate),  dup = dout * act(gate)
//
// HBM-bound: every operand is read or written once, in 16-byte packets where the rows allow.  A
// block is 32 packets wide and 8 rows high and walks down its share of the rows, so a warp's
// access is 512 contiguous bytes and each thread keeps the column sums of dz (fp32, before dz is
// rounded) in registers.  The sums of a block are joined in shared memory, those of several row
// blocks through scratch memory in a second kernel: a fixed order, so that a call always gives the
// same bits.

#include "ffn_math.cuh"

#include <algorithm>
#include <mutex>

namespace tmc {

// ---- stream-ordered scratch -------------------------------------------------------------------
std::string scratch_alloc(const LaunchCtx& ctx, size_t bytes, void** out) {
  *out = nullptr;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  static std::mutex lock;
  static cudaMemPool_t pool = nullptr;      // one device per process
  if (e == cudaSuccess) {
    std::lock_guard<std::mutex> guard(lock);
    if (!pool) {
      cudaMemPoolProps props{};
      props.allocType = cudaMemAllocationTypePinned;
      props.handleTypes = cudaMemHandleTypeNone;
      props.location.type = cudaMemLocationTypeDevice;
      props.location.id = device;
      e = cudaMemPoolCreate(&pool, &props);
      if (e == cudaSuccess) {
        uint64_t keep = 64ull << 20;         // freed scratch beyond this goes back to the device
        cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep);
      }
    }
  }
  if (e == cudaSuccess) e = cudaMallocFromPoolAsync(out, bytes, pool, ctx.stream);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return "could not allocate " + std::to_string(bytes) + " bytes of scratch memory: " + cudaGetErrorString(e);
  }
  return std::string();
}
void scratch_free(const LaunchCtx& ctx, void* p) {
  if (p) cudaFreeAsync(p, ctx.stream);
}

namespace {

using namespace ffn;

constexpr int CX = 32, RY = 8;

template <typename T, int VEC, bool GATED>
__global__ void __launch_bounds__(CX * RY) activation_bwd_kernel(const ActBwdProblem p, float* __restrict__ partial,
                                                                 int64_t rows_per_block) {
  const int tx = threadIdx.x % CX, ty = threadIdx.x / CX;
  const int64_t col = ((int64_t)blockIdx.x * CX + tx) * VEC;
  const int64_t first = (int64_t)blockIdx.y * rows_per_block;
  const int64_t last = min(first + rows_per_block, p.M);
  float sum[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
  if (col < p.N) {
    with_act(p.act, [&](auto tag) {
      constexpr Act act = decltype(tag)::value;
      constexpr bool precise = sizeof(T) == 4;
#pragma unroll 1                         // more in flight costs the blocks that would hide it (4: 40 % slower)
      for (int64_t m = first + ty; m < last; m += RY) {
        float d[VEC];
        load_vec<T, VEC>((const T*)p.dout + m * p.s_dout + col, d);
        if constexpr (GATED) {
          float g[VEC], u[VEC], du[VEC];
          load_vec<T, VEC>((const T*)p.pre + m * p.s_pre + col, g);
          load_vec<T, VEC>((const T*)p.up + m * p.s_pre + col, u);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float value, slope;
            act_both<precise>(act, g[i], value, slope);
            du[i] = d[i] * value;
            d[i] = d[i] * u[i] * slope;
          }
          store_vec<T, VEC>((T*)p.dup + m * p.s_dz + col, du);
        } else if constexpr (act != Act::None) {
          float z[VEC];
          load_vec<T, VEC>((const T*)p.pre + m * p.s_pre + col, z);
#pragma unroll
          for (int i = 0; i < VEC; ++i) d[i] *= act_derivative<precise>(act, z[i]);
        }
        if (p.dz) store_vec<T, VEC>((T*)p.dz + m * p.s_dz + col, d);
        if constexpr (!GATED) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum[i] += d[i];
        }
      }
    });
  }
  if constexpr (!GATED) {
    if (!p.dbias) return;
    __shared__ float joined[RY][CX * VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) joined[ty][tx * VEC + i] = sum[i];
    __syncthreads();
    for (int c = threadIdx.x; c < CX * VEC; c += CX * RY) {
      float total = 0.f;
#pragma unroll
      for (int r = 0; r < RY; ++r) total += joined[r][c];
      const int64_t n = (int64_t)blockIdx.x * CX * VEC + c;
      if (n >= p.N) continue;
      if (partial) partial[(int64_t)blockIdx.y * p.N + n] = total;
      else ((T*)p.dbias)[n] = from_f32<T>(total);
    }
  }
}

template <typename T, int VEC>
std::string launch_vec(const ActBwdProblem& p, const LaunchCtx& ctx) {
  const int64_t gx = (p.N + CX * VEC - 1) / (CX * VEC);
  // Each block has at least 32 rows; up to 64 one block takes them all and no second launch is needed.  With
  // column sums about eight blocks per SM, so that the sums stay cheap; without, more (8192 x 4096 gated: 62 us
  // with eight, 53 with 24).
  int64_t gy = std::max<int64_t>(1, (int64_t)ctx.sm_count * (p.gated ? 24 : 8) / gx);
  gy = p.M <= 64 && !p.gated ? 1 : std::min(gy, std::max<int64_t>(1, (p.M + 31) / 32));
  gy = std::min<int64_t>(gy, 65535);
  const int64_t rows = std::max<int64_t>(1, (p.M + gy - 1) / gy);
  gy = std::max<int64_t>(1, (p.M + rows - 1) / rows);
  if (gx > 0x7fffffff) return "too many columns";
  const dim3 grid((unsigned)gx, (unsigned)gy);
  if (p.gated) {
    activation_bwd_kernel<T, VEC, true><<<grid, CX * RY, 0, ctx.stream>>>(p, nullptr, rows);
    ++*ctx.launches;
  } else {
    void* partial = nullptr;
    if (p.dbias && gy > 1) {
      std::string err = scratch_alloc(ctx, (size_t)gy * (size_t)p.N * 4, &partial);
      if (!err.empty()) return err;
    }
    activation_bwd_kernel<T, VEC, false><<<grid, CX * RY, 0, ctx.stream>>>(p, (float*)partial, rows);
    ++*ctx.launches;
    if (partial) {
      void* outs[kMaxColumnSums] = {p.dbias};
      launch_column_sums(p.elt, (const float*)partial, gy, p.N, 1, outs, ctx);
      scratch_free(ctx, partial);
    }
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return std::string("activation backward launch failed: ") + cudaGetErrorString(e);
  return std::string();
}

template <typename T>
std::string launch_typed(const ActBwdProblem& p, const LaunchCtx& ctx) {
  constexpr int VEC = 16 / sizeof(T);
  uintptr_t bases = (uintptr_t)p.dout | (uintptr_t)p.dz;
  int64_t strides = p.s_dout | (p.dz ? p.s_dz : 0);
  if (p.act != Act::None || p.gated) { bases |= (uintptr_t)p.pre; strides |= p.s_pre; }
  if (p.gated) bases |= (uintptr_t)p.up | (uintptr_t)p.dup;
  const bool packets = bases % 16 == 0 && strides % VEC == 0 && p.N % VEC == 0;
  return packets ? launch_vec<T, VEC>(p, ctx) : launch_vec<T, 1>(p, ctx);
}

// out[n] = sum over `parts` rows of partial[part][n], for up to kMaxColumnSums sets at once.
struct SumOutputs {
  void* out[kMaxColumnSums];
};
// COLS columns and ROWS shares of the partial rows a block: the rows come from L2, eight in flight a thread.
template <typename T, int COLS, int ROWS>
__global__ void __launch_bounds__(COLS * ROWS) column_sums_kernel(const float* __restrict__ partial, int64_t parts, int64_t N,
                                                                  const SumOutputs outs) {
  __shared__ float joined[ROWS][COLS + 1];
  const int tx = threadIdx.x % COLS, ty = threadIdx.x / COLS;
  const int64_t n = (int64_t)blockIdx.x * COLS + tx;
  const float* base = partial + (int64_t)blockIdx.y * parts * N;
  float total = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int64_t r = ty; r < parts; r += ROWS) total += base[r * N + n];
  }
  joined[ty][tx] = total;
  __syncthreads();
#pragma unroll
  for (int step = ROWS / 2; step > 0; step /= 2) {
    if (ty < step) joined[ty][tx] += joined[ty + step][tx];
    __syncthreads();
  }
  if (ty == 0 && n < N) ((T*)outs.out[blockIdx.y])[n] = from_f32<T>(joined[0][tx]);
}

template <typename T>
void launch_sums(const float* partial, int64_t parts, int64_t N, int sets, const SumOutputs& outs, const LaunchCtx& ctx) {
  auto grid = [&](int cols) { return dim3((unsigned)((N + cols - 1) / cols), (unsigned)sets); };
  // As many threads as the SMs hold at once, so few columns are split over more rows: 3 x 4096 columns of 296 rows
  // took 17 us with 64 shares, 7 with 8; 2 x 1023 of 740 rows 17 us with 8, 8 with 64.
  const int64_t columns = N * sets;
  if (columns >= 8192) column_sums_kernel<T, 32, 8><<<grid(32), 256, 0, ctx.stream>>>(partial, parts, N, outs);
  else if (columns >= 4096) column_sums_kernel<T, 32, 32><<<grid(32), 1024, 0, ctx.stream>>>(partial, parts, N, outs);
  else column_sums_kernel<T, 16, 64><<<grid(16), 1024, 0, ctx.stream>>>(partial, parts, N, outs);
}

}  // namespace

void launch_column_sums(Elt elt, const float* partial, int64_t parts, int64_t N, int sets, void* const* out,
                        const LaunchCtx& ctx) {
  SumOutputs outs{};
  for (int i = 0; i < sets; ++i) outs.out[i] = out[i];
  if (elt == Elt::F32) launch_sums<float>(partial, parts, N, sets, outs, ctx);
  else if (elt == Elt::BF16) launch_sums<__nv_bfloat16>(partial, parts, N, sets, outs, ctx);
  else launch_sums<__half>(partial, parts, N, sets, outs, ctx);
  ++*ctx.launches;
}

std::string launch_activation_bwd(const ActBwdProblem& p, const LaunchCtx& ctx) {
  if (p.elt == Elt::F32) return launch_typed<float>(p, ctx);
  if (p.elt == Elt::BF16) return launch_typed<__nv_bfloat16>(p, ctx);
  return launch_typed<__half>(p, ctx);
}

}  // namespace tmc
