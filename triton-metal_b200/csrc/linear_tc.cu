// The feed-forward matrix products on the 5th-generation tensor cores, 16-bit operands with fp32
// accumulation: pairs of CTAs on one tile (tcgen05.mma.cta_group::2).
//
//   single  z = x w + bias; out = act(z) + residual       gated  out = act(x w) * (x w2)
//   sum     out = x w + x2 w2                              pair   out = x w and out2 = x2 w2
//
// One CTA per SM, two CTAs (a cluster) per 256 x BN tile.  CTA r holds rows r*128 ... of the x tile and
// half of the w tile's columns; the tensor cores of both SMs read both halves, so each SM's shared
// memory is filled with - and read for - half the w bytes a tile of its own would need.  The gated form
// is the same tile with CTA 0's half taken from w and CTA 1's from w2: accumulator column c and column
// c + BN/2 are then x w and x w2 of the same output column, and the product is taken in the epilogue
// where both are registers of one thread.  The sum runs one K loop over both operand pairs; the pair
// walks the columns of both results as one wider matrix, so that a shared x panel stays in L2.
//
//   warp 16  TMA producer (one lane): 64-deep k-blocks into a ring; both CTAs' loads complete on the
//            leader's barrier
//   warp 17  of the leader: tcgen05.mma 256 x BN x 16 into one of two TMEM accumulators; its commits
//            release the ring slots and publish the accumulators in both CTAs
//   warps 0-15  epilogue, thread = row, four warps per 32 rows (with two, the activations' latencies kept a
//            K = 1024 gelu tile at 841 TFLOP/s): bias, activation, residual, rounding;
//            32-column pieces leave through shared memory and TMA stores (clipped at the edges by the
//            tensor map), or, where the output's rows are not 16-byte aligned, as coalesced elements
//
// Either operand may be contiguous along k or along its other dimension (the descriptors say which), so
// transposed weights and the products of the backward pass (dz w^T, x^T dz) need no copies.

#include "ffn_math.cuh"
#include "linear_tc.h"
#include "sm100_ptx.cuh"

#include <algorithm>

namespace tmc {
namespace {

using namespace ptx;
using namespace ffn;

constexpr int BM = 128;                // rows of one CTA; a pair owns 256
constexpr int BK = 64;
constexpr int EPI_WARPS = 16;
constexpr int NUM_THREADS = (EPI_WARPS + 2) * 32;
constexpr int TMEM_COLS = 512;
constexpr int BOX = 32 * 64;           // one warp's staged piece: 32 rows x 32 columns
constexpr int A_BYTES = BM * BK * 2;

// A tile is HALVES accumulators of BN columns side by side.
template <int BN, int HALVES> struct Config {
  static constexpr int B_BYTES = BN / 2 * BK * 2;         // this CTA's part of one accumulator's w columns
  static constexpr int STAGE_BYTES = A_BYTES + HALVES * B_BYTES;
  static constexpr int STAGES = HALVES == 2 ? 4 : BN == 256 ? 6 : 7;
  static constexpr int SMEM = STAGES * STAGE_BYTES + EPI_WARPS * BOX + 2048;
};

enum Site : uint32_t { kProdEmpty = 41, kMmaFull = 42, kMmaAccEmpty = 43, kEpiAccFull = 44, kDrain = 45, kTmemReady = 46 };

struct Barriers {
  alignas(8) uint64_t full[8];
  alignas(8) uint64_t empty[8];
  alignas(8) uint64_t acc_full[2];
  alignas(8) uint64_t acc_empty[2];
  alignas(8) uint64_t tmem_ready;
  uint32_t tmem_base;
  int abort_flag;
};

struct alignas(64) Maps {
  CUtensorMap x, x2, w, w2, out, out2, pre, pre2;
};

struct Args {
  int M, N, K;
  int act, mode;
  int x_mn, w_mn;                      // 1: the operand is contiguous along m (n), 0: along k
  int tma_out, tma_pre;                // rows of out, out2 (pre, pre2) are 16-byte aligned
  int vec_bias, vec_residual;
  const void *bias, *residual;
  void *out, *out2, *pre, *pre2;
  int64_t srm, som, spm;
  int group_m;
};

// ---- the pair ---------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// (not the .aligned forms: a warp whose lanes have taken different roles may still be diverged here)
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// A tile load of this CTA's shared memory that completes on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void mma_pair_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, e;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs once every MMA issued so far has finished.
__device__ __forceinline__ void commit_pair_elect(uint32_t bar) {
  asm volatile(
      "{\n"
      ".reg .pred e;\n"
      ".reg .b16 both;\n"
      "mov.b16 both, 3;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n"
      "}\n" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t slot, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t base, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}

// Groups of row blocks, column by column, odd groups backwards: see gemm_tc.cu.
__device__ __forceinline__ void tile_coords(int tile, int tiles_m, int tiles_n, int group_m, int& tm, int& tn) {
  const int per_group = group_m * tiles_n;
  const int group = tile / per_group;
  const int first_m = group * group_m;
  const int rows = min(tiles_m - first_m, group_m);
  const int in_group = tile - group * per_group;
  tm = first_m + in_group % rows;
  tn = in_group / rows;
  if (group & 1) tn = tiles_n - 1 - tn;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// 32 columns of one row, rounded, into a warp's staged piece (the 64-byte-swizzled layout of a tile of 32
// rows x 32 columns: 16-byte chunks XORed with the row pair).
template <typename T>
__device__ __forceinline__ void stage_row(uint32_t piece, int lane, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t chunk = (uint32_t)j ^ (uint32_t)((lane >> 1) & 3);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece + lane * 64 + chunk * 16),
                 "r"(pack2<T>(v[j * 8 + 0], v[j * 8 + 1])), "r"(pack2<T>(v[j * 8 + 2], v[j * 8 + 3])),
                 "r"(pack2<T>(v[j * 8 + 4], v[j * 8 + 5])), "r"(pack2<T>(v[j * 8 + 6], v[j * 8 + 7]))
                 : "memory");
  }
}
// The staged piece element by element, for outputs whose rows are not 16-byte aligned.
template <typename T>
__device__ __forceinline__ void store_elements(T* base, int64_t stride, uint32_t piece, int lane, int row0, int col0,
                                               int M, int N) {
  const int rows = min(32, M - row0);
  for (int r = 0; r < rows; ++r) {
    const uint32_t chunk = (uint32_t)(lane / 8) ^ (uint32_t)((r >> 1) & 3);
    uint16_t bits;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(piece + r * 64 + chunk * 16 + (lane % 8) * 2) : "memory");
    if (col0 + lane < N) reinterpret_cast<uint16_t*>(base + (int64_t)(row0 + r) * stride + col0)[lane] = bits;
  }
}

// v += the next 32 of `left` elements; `packets`: they are 16-byte aligned.
template <typename T>
__device__ __forceinline__ void add_row(float (&v)[32], const T* from, int left, bool packets) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float e[8];
    if (packets && j * 8 + 8 <= left) {
      load_vec<T, 8>(from + j * 8, e);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = j * 8 + i < left ? to_f32(from[j * 8 + i]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j * 8 + i] += e[i];
  }
}

__device__ __forceinline__ void load_tmem(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld_32x32(addr, r);
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

template <typename T, bool GATED, int BN, int HALVES>
__global__ void __launch_bounds__(NUM_THREADS, 1) __cluster_dims__(2, 1, 1)
linear_tc_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a, DeviceStatus* status) {
  using C = Config<BN, HALVES>;
  constexpr int STAGES = C::STAGES, STAGE_BYTES = C::STAGE_BYTES;
  constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  constexpr int COLS = GATED ? BN / 2 : BN;           // output columns of an accumulator
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  Barriers& bars = *reinterpret_cast<Barriers*>(smem + STAGES * STAGE_BYTES + EPI_WARPS * BOX);
  const uint32_t smem_base = smem_u32(smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cta_rank();
  WaitCtx wc{&bars.abort_flag, status};

  const int tiles_m = (a.M + 2 * BM - 1) / (2 * BM);
  const int tiles_one = (a.N + HALVES * COLS - 1) / (HALVES * COLS);
  const int tiles_n = a.mode == (int)LinearMode::Pair ? 2 * tiles_one : tiles_one;
  const int num_tiles = tiles_m * tiles_n;
  const int blocks_one = (a.K + BK - 1) / BK;
  const int k_blocks = a.mode == (int)LinearMode::Sum ? 2 * blocks_one : blocks_one;
  const int first = blockIdx.x / 2, step = gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&bars.full[s]), 1);
      mbar_init(smem_u32(&bars.empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.acc_full[i]), 1);
      mbar_init(smem_u32(&bars.acc_empty[i]), 2 * EPI_WARPS);
    }
    mbar_init(smem_u32(&bars.tmem_ready), 2);
    bars.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == EPI_WARPS && lane == 0) {
    tma_prefetch_desc(&maps.x);
    tma_prefetch_desc(&maps.w);
  }
  __syncwarp();
  cluster_sync();                       // both CTAs' barriers exist: the loads begin while the TMEM is allocated

  if (warp == EPI_WARPS) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        int tm, tn;
        tile_coords(tile, tiles_m, tiles_n, a.group_m, tm, tn);
        const bool second = tn >= tiles_one;                       // pair: the second product
        if (second) tn -= tiles_one;
        const int row = (tm * 2 + (int)rank) * BM;
        const int col = tn * HALVES * COLS + (GATED ? 0 : (int)rank * (BN / 2));
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1, wc, kProdEmpty)) { ok = false; break; }
          const bool other = second || kb >= blocks_one;           // sum: the second pair of operands
          const int k = (kb >= blocks_one ? kb - blocks_one : kb) * BK;
          const CUtensorMap* mx = other ? &maps.x2 : &maps.x;
          const CUtensorMap* mw = (GATED ? rank != 0 : other) ? &maps.w2 : &maps.w;
          const uint32_t bar = map_to_cta(smem_u32(&bars.full[stage]), 0);
          const uint32_t dst = smem_base + stage * STAGE_BYTES;
          if (rank == 0) mbar_expect_tx(smem_u32(&bars.full[stage]), 2 * STAGE_BYTES);
          if (a.x_mn) {
#pragma unroll
            for (int b = 0; b < BM / 64; ++b) tma_load_pair(dst + b * 8192, mx, bar, row + b * 64, k);
          } else {
            tma_load_pair(dst, mx, bar, k, row);
          }
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            const uint32_t to = dst + A_BYTES + h * C::B_BYTES;
            if (a.w_mn) {
#pragma unroll
              for (int b = 0; b < BN / 128; ++b) tma_load_pair(to + b * 8192, mw, bar, col + h * COLS + b * 64, k);
            } else {
              tma_load_pair(to, mw, bar, k, col + h * COLS);
            }
          }
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // Before leaving, every slot this thread filled must have been released: the commit that does so
      // arrives on both CTAs, and the copies have then landed too.
      const uint32_t pending = issued < (uint32_t)STAGES ? issued : (uint32_t)STAGES;
      int s = stage;
      uint32_t ph = phase;
      for (uint32_t i = 0; i < pending && ok; ++i) {
        if (--s < 0) { s = STAGES - 1; ph ^= 1; }
        ok = mbar_wait(smem_u32(&bars.empty[s]), ph, wc, kProdEmpty);
      }
      // After a wait that gave up, copies may still be in flight.  Those of both CTAs complete on the
      // leader's barriers: it waits for them (bounded), the peer at the cluster barrier below.
      if (!ok && rank == 0) {
        for (uint32_t i = 0; i < pending; ++i) {
          if (--stage < 0) { stage = STAGES - 1; phase ^= 1; }
          const long long t0 = clock64();
          while (!mbar_try_wait(smem_u32(&bars.full[stage]), phase)) {
            if (clock64() - t0 > kWaitCycles) { report_timeout(wc, kDrain, stage); break; }
          }
        }
      }
    }
  } else if (warp == EPI_WARPS + 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    tmem_alloc_pair(smem_u32(&bars.tmem_base), TMEM_COLS);
    tc_fence_before();
    if (lane == 0) arrive_at(map_to_cta(smem_u32(&bars.tmem_ready), 0));
    __syncwarp();
    if (rank == 0 && mbar_wait_warp(smem_u32(&bars.tmem_ready), 0, wc, kTmemReady)) {
      tc_fence_after();
      const uint32_t tmem_base = *(volatile uint32_t*)&bars.tmem_base;
      const uint32_t idesc = make_idesc(FMT, 2 * BM, BN, a.x_mn, a.w_mn);
      const SmemDesc a_base = make_desc_sw128(smem_base, a.x_mn ? 8192 : 0, 1024);
      const SmemDesc b_base = make_desc_sw128(smem_base + A_BYTES, a.w_mn ? 8192 : 0, 1024);
      // 16 k further on: 32 bytes along a k-contiguous row, 16 rows of 128 bytes otherwise
      const uint32_t a_step = a.x_mn ? 2048 : 32, b_step = a.w_mn ? 2048 : 32;
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      auto products = [&](int at, int half, int acc, bool first_block) {
        const SmemDesc a_desc = a_base.advanced(at * STAGE_BYTES);
        const SmemDesc b_desc = b_base.advanced(at * STAGE_BYTES + half * C::B_BYTES);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          mma_pair_elect(tmem_base + acc * 256, a_desc.at(k * a_step), b_desc.at(k * b_step), idesc, !first_block || k != 0);
      };
      for (int tile = first; tile < num_tiles && ok; tile += step, ++local) {
        if constexpr (HALVES == 1) {
          const int acc = local & 1;
          if (!mbar_wait_warp(smem_u32(&bars.acc_empty[acc]), ((local >> 1) & 1) ^ 1, wc, kMmaAccEmpty)) { ok = false; break; }
          tc_fence_after();
          for (int kb = 0; kb < k_blocks; ++kb) {
            if (!mbar_wait_warp(smem_u32(&bars.full[stage]), phase, wc, kMmaFull)) { ok = false; break; }
            tc_fence_after();
            products(stage, 0, acc, kb == 0);
            commit_pair_elect(smem_u32(&bars.empty[stage]));
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
          }
          if (ok) commit_pair_elect(smem_u32(&bars.acc_full[acc]));
        } else {
          // Both accumulators are still being read when the tile's operands are there: the first k-blocks go
          // into the first half as soon as that is free, and catch up with the second when it is.
          const int lead = min(STAGES, k_blocks);
          int at = stage;
          uint32_t ph = phase;
          if (!mbar_wait_warp(smem_u32(&bars.acc_empty[0]), (local & 1) ^ 1, wc, kMmaAccEmpty)) { ok = false; break; }
          tc_fence_after();
          for (int kb = 0; kb < lead; ++kb) {
            if (!mbar_wait_warp(smem_u32(&bars.full[at]), ph, wc, kMmaFull)) { ok = false; break; }
            tc_fence_after();
            products(at, 0, 0, kb == 0);
            if (++at == STAGES) { at = 0; ph ^= 1; }
          }
          if (!ok) break;
          if (lead == k_blocks) commit_pair_elect(smem_u32(&bars.acc_full[0]));
          if (!mbar_wait_warp(smem_u32(&bars.acc_empty[1]), (local & 1) ^ 1, wc, kMmaAccEmpty)) { ok = false; break; }
          tc_fence_after();
          for (int kb = 0; kb < k_blocks; ++kb) {
            if (kb >= lead) {
              if (!mbar_wait_warp(smem_u32(&bars.full[stage]), phase, wc, kMmaFull)) { ok = false; break; }
              tc_fence_after();
              products(stage, 0, 0, false);
              if (kb == k_blocks - 1) commit_pair_elect(smem_u32(&bars.acc_full[0]));
            }
            products(stage, 1, 1, kb == 0);
            commit_pair_elect(smem_u32(&bars.empty[stage]));
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
          }
          if (ok) commit_pair_elect(smem_u32(&bars.acc_full[1]));
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (warps 0-15)
    const int quarter = warp % 4, part = warp / 4;
    const uint32_t piece = smem_base + STAGES * STAGE_BYTES + warp * BOX;
    const Act act = (Act)a.act;
    // one wait of these warps lasts as long as a tile's products do: up to 1040 clocks a k-block (4096 allowed)
    const WaitCtx tile_wait{&bars.abort_flag, status, kWaitCycles + 4096ll * k_blocks};
    bool staged = false;                // a TMA store may still be reading the piece
    bool ok = true;
    int local = 0;
    for (int tile = first; tile < num_tiles && ok; tile += step, ++local) {
      int tm, tn;
      tile_coords(tile, tiles_m, tiles_n, a.group_m, tm, tn);
      const bool second = tn >= tiles_one;
      if (second) tn -= tiles_one;
      const int row0 = (tm * 2 + (int)rank) * BM + quarter * 32;
      const int row = row0 + lane;
      // out of a warp's registers into one of the outputs
      auto emit = [&](const CUtensorMap* map, bool tma, void* base, int64_t stride, int col0, const float (&v)[32]) {
        if (staged && lane == 0) tma_store_wait_read();
        __syncwarp();
        stage_row<T>(piece, lane, v);
        if (tma) fence_proxy_async();
        __syncwarp();
        if (!tma) {
          store_elements<T>((T*)base, stride, piece, lane, row0, col0, a.M, a.N);
        } else if (lane == 0) {
          tma_store_2d(map, piece, col0, row0);
          tma_store_commit();
        }
        staged = tma;
      };
#pragma unroll 1
      for (int half = 0; half < HALVES; ++half) {
        const int acc = HALVES == 2 ? half : local & 1;
        const uint32_t turn = HALVES == 2 ? local & 1 : (local >> 1) & 1;
        // (the lanes leave together: one that gave up alone would be missed by the next warp-wide load)
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.acc_full[acc]), turn, tile_wait, kEpiAccFull))) { ok = false; break; }
        tc_fence_after();
        // (the allocation is ordered before the products that filled the accumulator)
        const uint32_t lanes = *(volatile uint32_t*)&bars.tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * 256;
        const int first_col = (tn * HALVES + half) * COLS;
        // the accumulator may be overwritten: tell the leader, from both CTAs
        bool released = false;
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(map_to_cta(smem_u32(&bars.acc_empty[acc]), 0));
          released = true;
        };
#pragma unroll 1
        for (int c = part * 32; c < COLS && row0 < a.M && first_col + c < a.N; c += 128) {
          // one piece: 32 output columns
          const int col0 = first_col + c;
          const bool last = c + 128 >= COLS || col0 + 128 >= a.N;
          float v[32];
          load_tmem(lanes + c, v);
          if constexpr (GATED) {
            float up[32];
            load_tmem(lanes + BN / 2 + c, up);
            if (last) release();
            if (a.pre) emit(&maps.pre, a.tma_pre, a.pre, a.spm, col0, v);
            if (a.pre2) emit(&maps.pre2, a.tma_pre, a.pre2, a.spm, col0, up);
            with_act(act, [&](auto tag) { act_row<decltype(tag)::value>(v); });
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= up[i];
          } else {
            if (last) release();
            if (a.bias) add_row<T>(v, (const T*)a.bias + col0, a.N - col0, a.vec_bias);
            if (a.pre) emit(&maps.pre, a.tma_pre, a.pre, a.spm, col0, v);
            if (act != Act::None)
              with_act(act, [&](auto tag) { act_row<decltype(tag)::value>(v); });
            if (a.residual && row < a.M)
              add_row<T>(v, (const T*)a.residual + (int64_t)row * a.srm + col0, a.N - col0, a.vec_residual);
          }
          emit(second ? &maps.out2 : &maps.out, a.tma_out, second ? a.out2 : a.out, a.som, col0, v);
        }
        if (!released) release();
      }
    }
    if (lane == 0) tma_store_wait_read();    // the staged pieces must outlive the stores' reads
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();                       // nobody still reads, writes or signals the other's memory
  if (warp == EPI_WARPS + 1) {
    tc_fence_after();
    tmem_dealloc_pair(*(volatile uint32_t*)&bars.tmem_base, TMEM_COLS);
  }
}

// ---- host ----------------------------------------------------------------------------------------

std::string output_map(CUtensorMap* map, CUtensorMapDataType type, void* base, int64_t M, int64_t N,
                       int64_t stride) {
  uint64_t dims[2] = {(uint64_t)N, (uint64_t)M};
  uint64_t strides[1] = {(uint64_t)(M > 1 ? stride : (N + 7) / 8 * 8) * 2};
  uint32_t box[2] = {32u, 32u};
  return make_tensor_map(map, type, 2, base, dims, strides, box, 64);
}

template <typename T, bool GATED, int BN, int HALVES>
std::string launch_tile(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw, const LaunchCtx& ctx) {
  using C = Config<BN, HALVES>;
  constexpr int COLS = GATED ? BN / 2 : BN;
  const CUtensorMapDataType type =
      p.elt == Elt::BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  Maps maps{};
  Args a{};
  a.M = (int)p.M; a.N = (int)p.N; a.K = (int)p.K;
  a.act = (int)p.act;
  a.mode = (int)p.mode;
  a.x_mn = lx.mn; a.w_mn = lw.mn;
  a.bias = p.bias; a.residual = p.residual;
  a.out = p.out; a.out2 = p.out2; a.pre = p.pre; a.pre2 = p.pre2;
  a.srm = p.srm; a.som = p.som; a.spm = p.spm;
  a.group_m = 8;                     // row blocks (of 256) walked together: 4, 16 and 32 were 2 to 7 % slower
  auto aligned = [&](const void* q, int64_t stride) { return (uintptr_t)q % 16 == 0 && (p.M <= 1 || (stride % 8 == 0 && stride < (1ll << 38))); };
  a.tma_out = aligned(p.out, p.som) && aligned(p.out2, p.som);
  a.tma_pre = aligned(p.pre, p.spm) && aligned(p.pre2, p.spm);
  a.vec_bias = (uintptr_t)p.bias % 16 == 0;
  a.vec_residual = (uintptr_t)p.residual % 16 == 0 && p.srm % 8 == 0;
  std::string e = make_operand_map(&maps.x, type, p.x, p.M, p.K, lx, BM);
  if (e.empty()) e = make_operand_map(&maps.w, type, p.w, p.N, p.K, lw, BN / 2);
  if (e.empty() && p.x2) e = make_operand_map(&maps.x2, type, p.x2, p.M, p.K, lx, BM);
  if (e.empty() && p.w2) e = make_operand_map(&maps.w2, type, p.w2, p.N, p.K, lw, BN / 2);
  if (e.empty() && a.tma_out) e = output_map(&maps.out, type, p.out, p.M, p.N, p.som);
  if (e.empty() && a.tma_out && p.out2) e = output_map(&maps.out2, type, p.out2, p.M, p.N, p.som);
  if (e.empty() && a.tma_pre && p.pre) e = output_map(&maps.pre, type, p.pre, p.M, p.N, p.spm);
  if (e.empty() && a.tma_pre && p.pre2) e = output_map(&maps.pre2, type, p.pre2, p.M, p.N, p.spm);
  if (!e.empty()) return e;
  auto kernel = linear_tc_kernel<T, GATED, BN, HALVES>;
  static const cudaError_t sized = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  cudaError_t err = sized;
  if (err != cudaSuccess) return cudaGetErrorString(err);
  const int64_t tiles = ((p.M + 2 * BM - 1) / (2 * BM)) * ((p.N + HALVES * COLS - 1) / (HALVES * COLS)) * (p.mode == LinearMode::Pair ? 2 : 1);
  if (tiles > 0x3fffffff) return "too many tiles";
  const int64_t pairs = std::min<int64_t>(tiles, ctx.sm_count / 2);
  kernel<<<(unsigned)(2 * pairs), NUM_THREADS, C::SMEM, ctx.stream>>>(maps, a, ctx.status);
  ++*ctx.launches;
  err = cudaGetLastError();
  if (err != cudaSuccess) return std::string("launch failed: ") + cudaGetErrorString(err);
  return std::string();
}

// Tiles of 256 rows and `width` accumulator columns.
int64_t tile_count(const LinearProblem& p, int width) {
  const int64_t cols = p.mode == LinearMode::Gated ? width / 2 : width;
  return ((p.M + 2 * BM - 1) / (2 * BM)) * ((p.N + cols - 1) / cols) * (p.mode == LinearMode::Pair ? 2 : 1);
}

// Clocks of a launch with tiles of 256 x `width` accumulator columns.  What an SM takes in bounds the narrower
// ones: a k-block's products take 256, 512 and 1024 clocks at 128, 256 and 512 columns and ask for 96, 64 and 48
// bytes a clock; measured on 8192 x 4096 x 16384, 281, 420 and 791 ns a k-block of every pair.  The widest leaves no
// second accumulator, so part of its epilogue is not hidden under the next tile's products.
double tile_clocks(const LinearProblem& p, int width, int sm_count) {
  const int64_t tiles = tile_count(p, width);
  const int64_t blocks = (p.K + BK - 1) / BK * (p.mode == LinearMode::Sum ? 2 : 1);
  const int64_t waves = (tiles + sm_count / 2 - 1) / (sm_count / 2);
  const bool light = p.act == Act::None && p.mode != LinearMode::Gated && !p.pre && !p.residual;
  const double block = width == 512 ? 1040.0 : width == 256 ? 552.0 : 380.0;
  return (double)waves * ((double)blocks * block + (width == 512 ? (light ? 2000.0 : 6000.0) : 300.0));
}
// The width that is done first.
int tile_width(const LinearProblem& p, int sm_count) {
  int best = 256;
  for (int width : {128, 512})
    if (tile_clocks(p, width, sm_count) < tile_clocks(p, best, sm_count)) best = width;
  return best;
}

template <typename T, bool GATED>
std::string launch_width(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw, const LaunchCtx& ctx) {
  switch (tile_width(p, ctx.sm_count)) {
    case 128: return launch_tile<T, GATED, 128, 1>(p, lx, lw, ctx);
    case 256: return launch_tile<T, GATED, 256, 1>(p, lx, lw, ctx);
    default: return launch_tile<T, GATED, 256, 2>(p, lx, lw, ctx);
  }
}

template <typename T>
std::string launch_typed(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw, const LaunchCtx& ctx) {
  return p.mode == LinearMode::Gated ? launch_width<T, true>(p, lx, lw, ctx) : launch_width<T, false>(p, lx, lw, ctx);
}

}  // namespace

std::string make_operand_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t outer, int64_t K,
                             const OperandLayout& l, int box_outer) {
  uint64_t dims[2], strides[1];
  uint32_t box[2];
  if (!l.mn) {
    dims[0] = (uint64_t)K; dims[1] = (uint64_t)outer;
    box[0] = BK; box[1] = (uint32_t)box_outer;
  } else {
    dims[0] = (uint64_t)outer; dims[1] = (uint64_t)K;
    box[0] = 64; box[1] = BK;
  }
  strides[0] = (uint64_t)l.stride * 2;
  return make_tensor_map(map, type, 2, base, dims, strides, box);
}

int linear_tc_width(const LinearProblem& p, int sm_count, int64_t* tiles) {
  const int width = tile_width(p, sm_count);
  *tiles = tile_count(p, width);
  return width;
}

double estimate_linear_tc(const LinearProblem& p, int sm_count) {
  // Few tiles get less of it than many do (128 x 4096 x 4096: 516 clocks a 128-column k-block), and a launch takes
  // 5 us with nothing to do.  With few rows it is bound by its operands' way from memory, at 2600 bytes a clock.
  const double bytes = 2.0 * ((double)p.K * (double)p.N * (p.w2 ? 2 : 1) + (double)p.M * (double)p.K);
  const double products = 1.33 * tile_clocks(p, tile_width(p, sm_count), sm_count);
  return std::max(products, bytes / 2600.0) + 9500.0;
}

std::string launch_linear_tc(const LinearProblem& p, const OperandLayout& lx, const OperandLayout& lw,
                             const LaunchCtx& ctx) {
  if (p.elt == Elt::BF16) return launch_typed<__nv_bfloat16>(p, lx, lw, ctx);
  return launch_typed<__half>(p, lx, lw, ctx);
}

}  // namespace tmc
