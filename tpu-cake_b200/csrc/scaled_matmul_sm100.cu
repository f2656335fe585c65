// Block-scaled 8-bit matmul for sm_100a: out[m, n] = sum over k of
// (lhs[m, k] 2^(sl[m, k / 128] - 127)) * (rhs[n, k] 2^(sr[n, k / 128] - 127)), e4m3 codes, e8m0 scales, f32
// accumulation in tensor memory, one rounding to the output type.
//
// The scales are powers of two, so the tensor core applies them itself (kind::mxf8f6f4, one scale per
// operand row and 32 k; the four 32-deep steps of a 128-deep block name the same byte): nothing is
// multiplied in the epilogue and no partial sum leaves tensor memory before the end of the contraction.
// With scales of any mantissa every 128-deep block's 128 x N products would have to be read back, scaled
// and added in registers.
//
// One kernel template, two shapes of work. "A" is the 128-row operand of a block, "B" the one of BN rows.
//   wide    A = lhs, B = rhs: 256 x BN output tiles by pairs of blocks (cta_group::2: each block loads 128 rows of
//           A and half of B's, and one of them issues for both), persistent, with two accumulators, so that a
//           tile's epilogue runs under the next one's main loop (one at BN = 256, where scales leave no
//           room: for a single wave of tiles). A block fetches 128 + BN / 2 rows of 128 bytes for 2 BN cycles of
//           MMA: 67 bytes a cycle at BN = 224; the 128 x 224 tile of a block alone needs 98, and L2 gives
//           an SM about 64.
//   narrow  A = rhs, B = lhs: 128 columns of the output by BN tokens. Few tokens: bound by reading rhs
//           once, and the contraction of a tile is split over the blocks of a cluster, which add their
//           partial sums through distributed shared memory in rank order (no workspace, no atomics: the
//           same bits every time). Two blocks share an SM: 6.2 TB/s where one reaches 5.0.
// Warps: 0 TMA producer (128-byte swizzled rows of 128 codes, one k block per stage), 1 MMA issue and
// tensor memory, 2 scales to shared memory, 3 scales on to tensor memory, 4-7 epilogue. Warp 2 gathers a
// 32-bit word -- four k blocks' bytes -- per operand row, so that scales are taken as they lie, with any
// stride, and puts them into shared memory in the order tcgen05.cp wants: lane i's 16 bytes are rows i,
// 32 + i, 64 + i, 96 + i.
//
// Measured (codes of normal values; device time of graph replays): 4096 x 8192 x 8192 182 us, 3.03 PFLOP/s, the
// issuing warp taking 465 cycles per k block of 448 MMA cycles; 8192 x 16384 x 8192 840 us cold and 918 us
// (2.40 PFLOP/s) after a second of load, when the power cap holds the clock near 1.26 GHz (cuBLAS in bf16:
// 1.40 PFLOP/s then). Decode: 64 x 8192 x 16384 26.5 us (5.2 TB/s), 1 x 8192 x 8192 14.2 us: 4 us pass before the
// first and after the last k block (dependency to first scales 1 to 1.5, cluster reduction 1.3).
#include <cuda_bf16.h>
#include <string.h>

#include <algorithm>
#include <cmath>

#include "cake_host.h"
#include "cake_ptx.cuh"

namespace cake {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsA = 128;
constexpr int kBlockK = 128;  // codes (= bytes) of a k block: one swizzle row, one scale
constexpr int kUmmaK = 32;
constexpr int kScaleSlots = 2;          // shared-memory ring of scales, 16 k blocks (four words a row) each
constexpr int kSlotWords = 4;
constexpr int kScaleSets = 3;           // sets of scale columns in tensor memory, used in turn
constexpr int kStagingSlots = 2;        // pieces of 32 rows x 128 bytes an epilogue warp may have in flight
constexpr uint32_t kStagingBytes = 32 * 128;
constexpr int kReducePitch = kRowsA + 4;  // floats between two tokens' partial sums
constexpr long long kBudgetCycles = 4000000000ll;  // about two seconds of SM clock

constexpr int pow2_at_least(int v) {
  int p = 32;
  while (p < v) p *= 2;
  return p;
}

template <int BN, bool NARROW>
struct Cfg {
  static constexpr uint32_t kABytes = kRowsA * kBlockK;
  static constexpr int kLoadB = NARROW ? BN : BN / 2;  // rows of B that this block loads
  static constexpr uint32_t kStageBytes = kABytes + kLoadB * kBlockK;
  static_assert(kStageBytes % 1024 == 0, "swizzle atoms");
  static constexpr int kScaleBlocksB = (BN + 127) / 128;
  static constexpr uint32_t kWordBytes = 512 * (1 + kScaleBlocksB);  // one word of every operand row
  static constexpr uint32_t kScaleSlotBytes = kSlotWords * kWordBytes;
  static constexpr uint32_t kStaging = NARROW ? 0 : 4 * kStagingSlots * kStagingBytes;
  // Narrow: two blocks share an SM. Wide: one block has it all.
  static constexpr uint32_t kRoom = (NARROW ? 112 * 1024 : 226 * 1024) - 1024 /*alignment*/ - 512 /*barriers*/;
  static constexpr int kFit = static_cast<int>((kRoom - kStaging - kScaleSlots * kScaleSlotBytes) / kStageBytes);
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  // Accumulators, then kScaleSets sets of scale columns (4 for A, 4 per 128 rows of B).
  // Two accumulators of 256 columns would leave no room for scales.
  static constexpr int kAccumulators = NARROW || BN > 224 ? 1 : 2;
  static constexpr int kScaleCols = 4 * (1 + kScaleBlocksB);
  static constexpr int kScaleBase = kAccumulators * BN;
  static constexpr int kTmemCols = pow2_at_least(kScaleBase + kScaleSets * kScaleCols);
  static_assert(kTmemCols <= (NARROW ? 256 : 512), "tensor memory of an SM");
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + kStaging + kScaleSlots * kScaleSlotBytes + 512 + 1024;
  static_assert(!NARROW || BN * kReducePitch * 4 <= kStages * kStageBytes, "partial sums take the operand ring's place");
};

struct Params {
  int32_t rows_a, rows_b;    // rows of the two operands (wide: m and n; narrow: n and m)
  int32_t tiles_a, tiles_b;
  int32_t k_blocks;
  int32_t split;             // blocks of a cluster that share a tile (narrow)
  int32_t out_f32, tma_store;
  const uint8_t* scales_a;
  const uint8_t* scales_b;
  int64_t scales_a_stride, scales_b_stride;
  void* out;
  int64_t out_stride;
  int32_t* status;
};

__device__ __forceinline__ void record(int32_t* status, int code, int d0, int d1, int d2) {
  if (status && atomicCAS(status, 0, code) == 0) {
    status[1] = d0;
    status[2] = d1;
    status[3] = d2;
  }
}

// Bounded wait that also gives up when another role of this block has.
__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long start = clock64();
  while (true) {
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - start > kBudgetCycles) return false;
  }
}

// The scale bytes of COUNT operand rows for 16 k blocks, from k block kb on, as four words each; anything past
// the last k block. `align`: the rows' addresses and kb are multiples of it (16, 8, 4 or 1). Every branch is the
// whole warp's and has all rows' loads inside, so that they are under way together. Ordinary loads: this kernel
// may have started before the one that writes the scales ended, so they are not read-only for its lifetime.
template <int COUNT>
__device__ __forceinline__ void load_scales(uint32_t (&w)[COUNT][4], const uint8_t* const (&row)[COUNT], int kb, int k_blocks, int align) {
  if (align == 16 && kb + 16 <= k_blocks) {
#pragma unroll
    for (int r = 0; r < COUNT; ++r) {
      const uint4 v = *reinterpret_cast<const uint4*>(row[r] + kb);
      w[r][0] = v.x;
      w[r][1] = v.y;
      w[r][2] = v.z;
      w[r][3] = v.w;
    }
    return;
  }
  if (align >= 8 && kb + 16 <= k_blocks) {
#pragma unroll
    for (int r = 0; r < COUNT; ++r) {
      const uint2 lo = *reinterpret_cast<const uint2*>(row[r] + kb), hi = *reinterpret_cast<const uint2*>(row[r] + kb + 8);
      w[r][0] = lo.x;
      w[r][1] = lo.y;
      w[r][2] = hi.x;
      w[r][3] = hi.y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = kb + 4 * i;
    if (align >= 4 && at + 4 <= k_blocks) {
#pragma unroll
      for (int r = 0; r < COUNT; ++r) w[r][i] = *reinterpret_cast<const uint32_t*>(row[r] + at);
    } else if (at < k_blocks) {
      uint32_t byte[COUNT][4];
#pragma unroll
      for (int r = 0; r < COUNT; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) byte[r][j] = row[r][min(at + j, k_blocks - 1)];
#pragma unroll
      for (int r = 0; r < COUNT; ++r) w[r][i] = byte[r][0] | (byte[r][1] << 8) | (byte[r][2] << 16) | (byte[r][3] << 24);
    } else {
#pragma unroll
      for (int r = 0; r < COUNT; ++r) w[r][i] = 0x7F7F7F7Fu;
    }
  }
}

__device__ __forceinline__ int scale_alignment(const uint8_t* scales, int64_t stride, int kb_begin) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(scales) | static_cast<uintptr_t>(stride) | static_cast<uintptr_t>(kb_begin);
  return (bits & 15) == 0 ? 16 : (bits & 7) == 0 ? 8 : (bits & 3) == 0 ? 4 : 1;
}

// Consecutive tiles walk 8 row tiles down before moving one column tile right, so that the blocks of a
// wave share both operands' rows in L2.
__device__ __forceinline__ void raster(int t, int tiles_a, int tiles_b, int& ta, int& tb) {
  constexpr int kHigh = 8;
  const int group = kHigh * tiles_b;
  const int g = t / group;
  const int rows = min(kHigh, tiles_a - g * kHigh);
  const int r = t - g * group;
  ta = g * kHigh + r % rows;
  tb = r / rows;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The same for a barrier on which the other block of the pair arrives too.
__device__ __forceinline__ bool wait_or_abort_cluster(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const long long start = clock64();
  while (true) {
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait_cluster(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - start > kBudgetCycles) return false;
  }
}

__device__ __forceinline__ void store_as(char* at, uint32_t v, float) { *reinterpret_cast<uint32_t*>(at) = v; }
__device__ __forceinline__ void store_as(char* at, uint32_t v, __nv_bfloat16) { *reinterpret_cast<__nv_bfloat16*>(at) = __float2bfloat16_rn(__uint_as_float(v)); }

// One column of up to 16 tokens.
template <typename T>
__device__ __forceinline__ void store_tokens(char* at, int64_t stride, const uint32_t (&v)[16], int tokens) {
  if (tokens >= 16) {
#pragma unroll
    for (int j = 0; j < 16; ++j, at += stride) store_as(at, v[j], T());
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j, at += stride)
      if (j < tokens) store_as(at, v[j], T());
  }
}

// The accumulator has been read: one arrival of four (eight in a pair) on the issuing block's barrier.
__device__ __forceinline__ void release_accumulator(uint64_t* bar, int lane) {
  tcgen05_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive_remote(cluster_addr(smem_u32(bar), 0));
}

// The warp's staging slot that comes next, once the store that had it has read it.
__device__ __forceinline__ uint8_t* next_slot(const Params& p, uint8_t* staging, int& staged, int lane) {
  uint8_t* slot = staging + (staged % kStagingSlots) * kStagingBytes;
  if (p.tma_store && staged >= kStagingSlots) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kStagingSlots - 1) : "memory");
    __syncwarp();
  }
  ++staged;
  return slot;
}

// Staged boxes of 32 rows x 32 columns of T to the output.
template <typename T>
__device__ __forceinline__ void leave(const Params& p, const CUtensorMap& map, const uint8_t* slot, int row0, int col, int boxes, int lane) {
  if (p.tma_store) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      for (int b = 0; b < boxes; ++b) {
        if (col + 32 * b < p.rows_b)
          asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                       ::"l"(reinterpret_cast<uint64_t>(&map)), "r"(smem_u32(slot + b * 32 * 32 * sizeof(T))), "r"(col + 32 * b), "r"(row0)
                       : "memory");
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    return;
  }
  // Rows whose pitch, base or length is not a multiple of 16 bytes: one row of 32 columns per store.
  __syncwarp();
  const int rows = min(32, p.rows_a - row0);
  for (int b = 0; b < boxes; ++b) {
    const int c = col + 32 * b + lane;
    if (c < p.rows_b) {
      T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(row0) * p.out_stride + c;
      const uint8_t* box = slot + b * 32 * 32 * sizeof(T);
      for (int r = 0; r < rows; ++r, dst += p.out_stride) {
        const int piece = sizeof(T) == 4 ? (lane >> 2) ^ (r & 7) : (lane >> 3) ^ ((r >> 1) & 3);
        *dst = reinterpret_cast<const T*>(box + r * 32 * sizeof(T) + piece * 16)[lane % (16 / sizeof(T))];
      }
    }
  }
  __syncwarp();
}

// This block's share of a tile's pieces (one token, four columns): the sums over the cluster's blocks in rank
// order. Distributed shared memory answers slowly, so a thread has up to BLOCKS * AHEAD loads under way.
template <int BLOCKS, int AHEAD>
__device__ __forceinline__ void reduce_pieces(const Params& p, uint32_t base, int rank, int col0, int token0, int pieces) {
  const int step = p.split * kThreads;
  for (int first = rank * kThreads + static_cast<int>(threadIdx.x); first < pieces; first += AHEAD * step) {
    float4 v[AHEAD][BLOCKS];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = first + a * step;
      if (i < pieces) {
        const uint32_t at = base + ((i / (kRowsA / 4)) * kReducePitch + (i % (kRowsA / 4)) * 4) * 4;
#pragma unroll
        for (int s = 0; s < BLOCKS; ++s) v[a][s] = s < p.split ? ld_cluster_f32x4(at, s) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = first + a * step;
      if (i >= pieces) break;
      float4 sum = v[a][0];
#pragma unroll
      for (int s = 1; s < BLOCKS; ++s) {
        sum.x += v[a][s].x;
        sum.y += v[a][s].y;
        sum.z += v[a][s].z;
        sum.w += v[a][s].w;
      }
      const float e[4] = {sum.x, sum.y, sum.z, sum.w};
      const int col = col0 + (i % (kRowsA / 4)) * 4;
      const int64_t dst = static_cast<int64_t>(token0 + i / (kRowsA / 4)) * p.out_stride + col;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (col + j < p.rows_a) {
          if (p.out_f32) static_cast<float*>(p.out)[dst + j] = e[j];
          else static_cast<__nv_bfloat16*>(p.out)[dst + j] = __float2bfloat16_rn(e[j]);
        }
      }
    }
  }
}

// A whole warp waits: the result is the warp's, so that what follows stays uniform.
template <bool CLUSTER>
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
  if (__all_sync(0xffffffffu, CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, CLUSTER ? wait_or_abort_cluster(bar, parity, abort_flag) : wait_or_abort(bar, parity, abort_flag));
}

// One block (narrow) or a pair (wide): the instructions that differ.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (PAIR) tcgen05_commit_pair(bar);
  else tcgen05_commit(bar);
}

// The same for a barrier that only the issuing block waits on.
template <bool PAIR>
__device__ __forceinline__ void tcgen05_commit_as(uint32_t bar) {
  if (PAIR) tcgen05_commit_pair_local(bar);
  else tcgen05_commit(bar);
}

template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t dst, uint32_t src) {
  if (PAIR) tcgen05_cp_32x128b_warpx4_pair(dst, umma_desc_scales(src));
  else tcgen05_cp_32x128b_warpx4(dst, umma_desc_scales(src));
}

template <int BN, bool NARROW>
__global__ void __launch_bounds__(kThreads, NARROW ? 2 : 1)
    cake_scaled_matmul_sm100(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                             const __grid_constant__ CUtensorMap map_out, const __grid_constant__ Params p) {
  using C = Cfg<BN, NARROW>;
  constexpr int STAGES = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* staging = smem + STAGES * C::kStageBytes;
  uint8_t* scale_ring = staging + C::kStaging;
  uint64_t* bars = reinterpret_cast<uint64_t*>(scale_ring + kScaleSlots * C::kScaleSlotBytes);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* scale_full = empty_bar + STAGES;
  uint64_t* scale_empty = scale_full + kScaleSlots;
  uint64_t* tmem_full = scale_empty + kScaleSlots;
  uint64_t* tmem_empty = tmem_full + 2;
  uint64_t* set_full = tmem_empty + 2;
  uint64_t* set_empty = set_full + kScaleSets;
  uint64_t* drain_bar = set_empty + kScaleSets;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int num_tiles = p.tiles_a * p.tiles_b;
  // Narrow: one tile per cluster, this block's share of its k blocks. Wide: tiles by stride, all k blocks;
  // rank 0 issues for the pair.
  constexpr bool PAIR = !NARROW;
  const int rank = static_cast<int>(blockIdx.x) % (NARROW ? p.split : 2);
  const int first_tile = static_cast<int>(blockIdx.x) / (NARROW ? p.split : 2);
  const int tile_step = NARROW ? num_tiles : static_cast<int>(gridDim.x) / 2;
  const bool leader = NARROW || rank == 0;
  const int kb_begin = NARROW ? static_cast<int>(static_cast<int64_t>(p.k_blocks) * rank / p.split) : 0;
  const int kb_end = NARROW ? static_cast<int>(static_cast<int64_t>(p.k_blocks) * (rank + 1) / p.split) : p.k_blocks;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      mbar_init(smem_u32(&scale_full[s]), PAIR ? 2 : 1);
      mbar_init(smem_u32(&scale_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&tmem_full[b]), 1);
      mbar_init(smem_u32(&tmem_empty[b]), PAIR ? 8 : 4);
    }
    for (int s = 0; s < kScaleSets; ++s) {
      mbar_init(smem_u32(&set_full[s]), 1);
      mbar_init(smem_u32(&set_empty[s]), 1);
    }
    mbar_init(smem_u32(&drain_bar[0]), 1);
    mbar_init(smem_u32(&drain_bar[1]), 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_b);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), C::kTmemCols);
    } else {
      tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
      tmem_relinquish();
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // both blocks' barriers exist before either is arrived on
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // The kernel before this one may still run. Every working warp waits for it before it does anything else, the
  // producer and the scales warp after they have worked out where they will read.
  grid_dependency_trigger();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first_tile; t < num_tiles && ok; t += tile_step) {
        int ta, tb;
        raster(t, p.tiles_a, p.tiles_b, ta, tb);
        if (t == first_tile) grid_dependency_wait();
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!wait_or_abort(smem_u32(&empty_bar[stage]), phase ^ 1, abort_flag)) {
            if (!*abort_flag) record(p.status, 1, blockIdx.x, t, 100 + stage);
            *abort_flag = 1;
            ok = false;
            break;
          }
          const uint32_t full = smem_u32(&full_bar[stage]);
          const uint32_t dst = smem_u32(smem + stage * C::kStageBytes);
          if (PAIR) {
            // Both blocks' copies complete on the issuing block's barrier.
            if (leader) mbar_arrive_expect_tx(full, 2 * C::kStageBytes);
            const uint32_t bar = cluster_addr(full, 0);
            tma_load_2d_pair(dst, &map_a, bar, kb * kBlockK, (ta * 2 + rank) * kRowsA);
            tma_load_2d_pair(dst + C::kABytes, &map_b, bar, kb * kBlockK, tb * BN + rank * C::kLoadB);
          } else {
            mbar_arrive_expect_tx(full, C::kStageBytes);
            tma_load_2d(dst, &map_a, full, kb * kBlockK, ta * kRowsA);
            tma_load_2d(dst + C::kABytes, &map_b, full, kb * kBlockK, tb * BN);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) {
        // Let copies in flight land before the block's shared memory is released (a pair's both complete
        // on rank 0's barriers, and rank 1 leaves after rank 0).
        for (int s = 0; s < STAGES; ++s)
          mbar_wait_bounded(smem_u32(&full_bar[s]), s < stage ? phase : (phase ^ 1), 200000000ll);
      }
    }
  } else if (warp == 1 && leader) {
    // ------------------------------------------------------------------ MMA issue
    // The tensor pipe queues next to nothing behind the MMA it works on: what the issuing warp does between
    // two k blocks shows as soon as it takes longer than one MMA. So this loop is kept to one wait, four
    // MMAs and one commit per k block (one more of each per four), with the control flow warp-uniform and
    // the descriptors stepped, not built.
    grid_dependency_wait();  // its waits are bounded from here on
    const bool issuer = elect_one();
    const uint64_t desc0 = umma_desc_sw128(smem_u32(smem), 16, 1024);
    constexpr uint32_t kStageStep = C::kStageBytes >> 4;
    constexpr uint32_t kIdesc = umma_idesc_mxf8(PAIR ? 2 * kRowsA : kRowsA, BN, 0);
    uint32_t stage = 0, phase = 0, set = 0, set_phase = 0;
    int it = 0;
    bool ok = true, ready = false;  // ready: the next k block's operands have been seen to be there
    for (int t = first_tile; t < num_tiles && ok; t += tile_step, ++it) {
      const int buf = C::kAccumulators == 2 ? (it & 1) : 0;
      const uint32_t acc_phase = C::kAccumulators == 2 ? ((it >> 1) & 1) : (it & 1);
      if (!wait_warp<PAIR>(smem_u32(&tmem_empty[buf]), acc_phase ^ 1, abort_flag)) {
        if (!*abort_flag && issuer) record(p.status, 1, blockIdx.x, t, 200 + buf);
        *abort_flag = 1;
        break;
      }
      tcgen05_fence_after();
      const uint32_t tmem_d = tmem_base + buf * BN;
      uint32_t accumulate = 0;
      for (int kb = kb_begin; kb < kb_end && ok; kb += 4) {
        if (!wait_warp<false>(smem_u32(&set_full[set]), set_phase, abort_flag)) {
          if (!*abort_flag && issuer) record(p.status, 1, blockIdx.x, t, 500 + set);
          *abort_flag = 1;
          ok = false;
          break;
        }
        const uint32_t sfa = tmem_base + C::kScaleBase + set * C::kScaleCols;
#pragma unroll
        for (int byte = 0; byte < 4; ++byte) {
          if (kb + byte >= kb_end) break;
          if (!ready && !wait_warp<false>(smem_u32(&full_bar[stage]), phase, abort_flag)) {
            if (!*abort_flag && issuer) record(p.status, 1, blockIdx.x, t, 300 + stage);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tcgen05_fence_after();
          const uint32_t next_stage = stage + 1 == STAGES ? 0 : stage + 1, next_phase = next_stage == 0 ? phase ^ 1 : phase;
          const bool seen = mbar_test_wait(smem_u32(&full_bar[next_stage]), next_phase);  // answers while MMAs are issued
          if (issuer) {
            const uint64_t a_desc = desc0 + stage * kStageStep;
            const uint64_t b_desc = a_desc + (C::kABytes >> 4);
            const uint32_t idesc = kIdesc | (byte << 4) | (static_cast<uint32_t>(byte) << 29);
#pragma unroll
            for (int kk = 0; kk < kBlockK / kUmmaK; ++kk) {
              // K-major rows of 128 bytes, groups of eight 1024 bytes apart; a step of 32 codes is 32 bytes
              // inside the swizzle row.
              if (PAIR) tcgen05_mma_mxf8_pair(tmem_d, a_desc + kk * (kUmmaK >> 4), b_desc + kk * (kUmmaK >> 4), idesc, sfa, sfa + 4, accumulate);
              else tcgen05_mma_mxf8(tmem_d, a_desc + kk * (kUmmaK >> 4), b_desc + kk * (kUmmaK >> 4), idesc, sfa, sfa + 4, accumulate);
              accumulate = 1;
            }
            commit<PAIR>(smem_u32(&empty_bar[stage]));
          }
          accumulate = 1;
          ready = __all_sync(0xffffffffu, seen);
          stage = next_stage;
          phase = next_phase;
        }
        if (ok && issuer) tcgen05_commit_as<PAIR>(smem_u32(&set_empty[set]));
        if (++set == kScaleSets) {
          set = 0;
          set_phase ^= 1;
        }
      }
      if (ok && issuer) commit<PAIR>(smem_u32(&tmem_full[buf]));
    }
    // Everything issued above has retired before tensor memory is released.
    if (issuer) commit<PAIR>(smem_u32(drain_bar));
    __syncwarp();
    mbar_wait_bounded(smem_u32(drain_bar), 0, kBudgetCycles);
  } else if (warp == 3 && leader) {
    // ------------------------------------------------------------------ scales into tensor memory
    // Word by word from the ring to one of kScaleSets sets of columns, as soon as the MMAs of the word that
    // had the set are done; the slot of the ring is free when its last copy is.
    if (lane == 0) {
      uint32_t slot = 0, slot_phase = 0, set = 0, set_phase = 0;
      bool ok = true;
      grid_dependency_wait();
      for (int t = first_tile; t < num_tiles && ok; t += tile_step) {
        for (int kb = kb_begin; kb < kb_end; kb += 4) {
          const int word = ((kb - kb_begin) / 4) % kSlotWords;
          if (!wait_or_abort(smem_u32(&set_empty[set]), set_phase ^ 1, abort_flag) ||
              (word == 0 && !wait_or_abort_cluster(smem_u32(&scale_full[slot]), slot_phase, abort_flag))) {
            if (!*abort_flag) record(p.status, 1, blockIdx.x, t, 700 + slot);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tcgen05_fence_after();
          const uint32_t src = smem_u32(scale_ring + slot * C::kScaleSlotBytes + word * C::kWordBytes);
          const uint32_t dst = tmem_base + C::kScaleBase + set * C::kScaleCols;
#pragma unroll
          for (int b = 0; b <= C::kScaleBlocksB; ++b) copy_scales<PAIR>(dst + 4 * b, src + 512 * b);
          tcgen05_commit_as<PAIR>(smem_u32(&set_full[set]));
          if (word == kSlotWords - 1 || kb + 4 >= kb_end) {
            commit<PAIR>(smem_u32(&scale_empty[slot]));
            if (++slot == kScaleSlots) {
              slot = 0;
              slot_phase ^= 1;
            }
          }
          if (++set == kScaleSets) {
            set = 0;
            set_phase ^= 1;
          }
        }
      }
      // As above: no copy is under way when tensor memory is released.
      tcgen05_commit_as<PAIR>(smem_u32(drain_bar + 1));
      mbar_wait_bounded(smem_u32(drain_bar + 1), 0, kBudgetCycles);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ scales
    // 16 k blocks at a time: one fence and one arrival for four words, and few loads, each of which touches a
    // line per operand row. A word at a time, all of it took longer than the word's MMAs. Rows past an operand's end (and past the tile's)
    // get the last row's scales: their codes are zeros, or not there, and what comes of them is not stored.
    const int align = min(scale_alignment(p.scales_a, p.scales_a_stride, kb_begin), scale_alignment(p.scales_b, p.scales_b_stride, kb_begin));
    constexpr int kRowsOfB = (BN + 31) / 32;
    uint32_t slot = 0, slot_phase = 0;
    bool ok = true;
    for (int t = first_tile; t < num_tiles && ok; t += tile_step) {
      int ta, tb;
      raster(t, p.tiles_a, p.tiles_b, ta, tb);
      const uint8_t* row[4 + kRowsOfB];  // of A, then of B
#pragma unroll
      for (int c = 0; c < 4; ++c) row[c] = p.scales_a + min((PAIR ? ta * 2 + rank : ta) * kRowsA + c * 32 + lane, p.rows_a - 1) * p.scales_a_stride;
#pragma unroll
      for (int c = 0; c < kRowsOfB; ++c) row[4 + c] = p.scales_b + min(tb * BN + c * 32 + lane, p.rows_b - 1) * p.scales_b_stride;
      if (t == first_tile) grid_dependency_wait();
      for (int kb = kb_begin; kb < kb_end; kb += 4 * kSlotWords) {
        uint32_t w[4 + kRowsOfB][4];  // [32 rows each][word]
        load_scales<4 + kRowsOfB>(w, row, kb, p.k_blocks, align);
        if (!wait_warp<false>(smem_u32(&scale_empty[slot]), slot_phase ^ 1, abort_flag)) {
          if (!*abort_flag && lane == 0) record(p.status, 1, blockIdx.x, t, 600 + slot);
          *abort_flag = 1;
          ok = false;
          break;
        }
        uint8_t* dst = scale_ring + slot * C::kScaleSlotBytes + lane * 16;
#pragma unroll
        for (int i = 0; i < kSlotWords; ++i) {
#pragma unroll
          for (int c = 0; c < 4 + kRowsOfB; c += 4) {
            uint32_t v[4];  // columns past B's last rows: any
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = w[c + j < 4 + kRowsOfB ? c + j : 0][i];
            *reinterpret_cast<uint4*>(dst + i * C::kWordBytes + 128 * c) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_remote(cluster_addr(smem_u32(&scale_full[slot]), 0));
          else mbar_arrive(smem_u32(&scale_full[slot]));
        }
        if (++slot == kScaleSlots) {
          slot = 0;
          slot_phase ^= 1;
        }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue
    grid_dependency_wait();
    const int q = warp & 3;  // the lane quarter of tensor memory this warp may read
    uint8_t* my_staging = staging + q * kStagingSlots * kStagingBytes;
    int staged = 0, it = 0;
    for (int t = first_tile; t < num_tiles; t += tile_step, ++it) {
      int ta, tb;
      raster(t, p.tiles_a, p.tiles_b, ta, tb);
      const int buf = C::kAccumulators == 2 ? (it & 1) : 0;
      const uint32_t acc_phase = C::kAccumulators == 2 ? ((it >> 1) & 1) : (it & 1);
      // Warp-uniform: tcgen05.ld is a warp's instruction.
      if (!__all_sync(0xffffffffu, wait_or_abort(smem_u32(&tmem_full[buf]), acc_phase, abort_flag))) {
        if (!*abort_flag && lane == 0) record(p.status, 1, blockIdx.x, t, 400 + buf);
        *abort_flag = 1;
        break;
      }
      tcgen05_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BN;
      const int row0 = (PAIR ? ta * 2 + rank : ta) * kRowsA + q * 32;
      if (NARROW) {
        // Lane = output column, register = token. Alone, the block stores 32 columns of a token at a
        // time; sharing the tile, it leaves its partial sums in the operand ring, which is free: the
        // last MMA has read it.
        const int tokens = min(BN, p.rows_b - tb * BN);
        float* partial = reinterpret_cast<float*>(smem) + q * 32 + lane;
        const int col = row0 + lane;
        const int64_t stride = p.out_stride * (p.out_f32 ? 4 : 2);
        char* dst = static_cast<char*>(p.out) + tb * BN * stride + static_cast<int64_t>(col) * (p.out_f32 ? 4 : 2);
#pragma unroll 1
        for (int c = 0; c < tokens; c += 16) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(t_row + c, v);
          tmem_ld_wait();
          if (p.split > 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j) partial[(c + j) * kReducePitch] = __uint_as_float(v[j]);
          } else if (col < p.rows_a) {
            if (p.out_f32) store_tokens<float>(dst, stride, v, tokens - c);
            else store_tokens<__nv_bfloat16>(dst, stride, v, tokens - c);
            dst += 16 * stride;
          }
        }
        tcgen05_fence_before();
        continue;
      }
      // Wide: lane = output row, register = column. 32 rows x 128 bytes at a time (64 columns of bf16, as two
      // boxes of 32, or 32 of f32) leave through shared memory, in the layout of a swizzled tensor store's box.
      if (p.out_f32) {
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(t_row + c, v);
          tmem_ld_wait();
          if (c == BN - 32) release_accumulator(&tmem_empty[buf], lane);
          const int col = tb * BN + c;
          if (row0 >= p.rows_a || col >= p.rows_b) continue;  // warp-uniform
          uint8_t* slot = next_slot(p, my_staging, staged, lane);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(slot + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          leave<float>(p, map_out, slot, row0, col, 1, lane);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < BN; c += 64) {
          const int boxes = c + 32 < BN ? 2 : 1;
          uint32_t v[2][32];
          tmem_ld_32x32b_x32(t_row + c, v[0]);
          if (boxes == 2) tmem_ld_32x32b_x32(t_row + c + 32, v[1]);
          tmem_ld_wait();
          if (c + 64 >= BN) release_accumulator(&tmem_empty[buf], lane);
          const int col = tb * BN + c;
          if (row0 >= p.rows_a || col >= p.rows_b) continue;  // warp-uniform
          uint8_t* slot = next_slot(p, my_staging, staged, lane);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (b >= boxes) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = pack_bf16(__uint_as_float(v[b][8 * j + 2 * e]), __uint_as_float(v[b][8 * j + 2 * e + 1]));
              *reinterpret_cast<uint4*>(slot + b * 2048 + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          leave<__nv_bfloat16>(p, map_out, slot, row0, col, boxes, lane);
        }
      }
    }
    // Shared memory outlives every tensor store that still reads it.
    if (!NARROW && p.tma_store && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();

  if (NARROW && p.split > 1) {
    // Every block of the cluster takes its share of the tile's (token, four columns) pieces and adds the
    // partial sums of all blocks in rank order.
    grid_dependency_wait();  // at once by now: for the warps that have not waited yet
    cluster_sync();
    int ta, tb;
    raster(first_tile, p.tiles_a, p.tiles_b, ta, tb);
    const int tokens = min(BN, p.rows_b - tb * BN);
    const int pieces = tokens * (kRowsA / 4);
    if (!*abort_flag) {
      const uint32_t base = smem_u32(smem);
      if (p.split <= 2) reduce_pieces<2, 4>(p, base, rank, ta * kRowsA, tb * BN, pieces);
      else if (p.split <= 4) reduce_pieces<4, 2>(p, base, rank, ta * kRowsA, tb * BN, pieces);
      else reduce_pieces<8, 1>(p, base, rank, ta * kRowsA, tb * BN, pieces);
    }
    __syncwarp();
    cluster_sync();  // no block leaves while another reads its shared memory
  }
  tcgen05_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // neither block leaves while the other's instructions may touch it
  tcgen05_fence_after();
  if (warp == 1) {
    if (PAIR) tmem_dealloc_pair(tmem_base, C::kTmemCols);
    else tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

}  // namespace
}  // namespace cake

// ====================================================================================== host

namespace {

using cake::fail;

// What a launch has to know about the current device, looked up once per device.
struct Device {
  int index = -1;
  int sm_count = 0;
};

int32_t current_device(Device* d) {
  static int sm_counts[64] = {};
  CAKE_CUDA_TRY(cudaGetDevice(&d->index));
  const bool cached = d->index >= 0 && d->index < 64;
  if (cached && sm_counts[d->index] > 0) {
    d->sm_count = sm_counts[d->index];
    return CAKE_OK;
  }
  int major = 0;
  CAKE_CUDA_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, d->index));
  if (major != 10) return fail(CAKE_ERR_UNSUPPORTED, "libcake_b200 needs an sm_100 GPU, found compute capability %d.x", major);
  CAKE_CUDA_TRY(cudaDeviceGetAttribute(&d->sm_count, cudaDevAttrMultiProcessorCount, d->index));
  if (cached) sm_counts[d->index] = d->sm_count;
  return CAKE_OK;
}

template <int BN, bool NARROW>
int32_t launch(const Device& device, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& out,
               const cake::Params& p, cudaStream_t stream) {
  using C = cake::Cfg<BN, NARROW>;
  auto kernel = cake::cake_scaled_matmul_sm100<BN, NARROW>;
  // The opt-in to more than 48 KB of dynamic shared memory is a per-device attribute.
  static bool configured[64] = {};
  const bool cached = device.index >= 0 && device.index < 64;
  if (!cached || !configured[device.index]) {
    CAKE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    if (cached) configured[device.index] = true;
  }
  const int64_t tiles = static_cast<int64_t>(p.tiles_a) * p.tiles_b;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = NARROW ? p.split : 2;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(NARROW ? tiles * p.split : 2 * (tiles < device.sm_count / 2 ? tiles : device.sm_count / 2)));
  config.blockDim = dim3(cake::kThreads);
  config.dynamicSmemBytes = C::kSmemBytes;
  config.stream = stream;
  config.attrs = attrs;
  config.numAttrs = NARROW && p.split == 1 ? 1 : 2;
  CAKE_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, a, b, out, p));
  return CAKE_OK;
}

int32_t encode_operand(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t stride, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(stride)};
  const uint32_t box[2] = {cake::kBlockK, static_cast<uint32_t>(box_rows)};
  return cake::encode_tensor_map_as(map, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT8);
}

// What a call runs: the tile, and for narrow tiles the blocks that share one.
struct Choice {
  int tile, split;
};

bool is_narrow(int tile) { return tile <= 128; }

// Nanoseconds that a call of this shape is expected to take, from times measured at 1 to 1024 rows and
// extents of 1024 to 8192 (graph replays, one after the other): good to about a fifth, and the neighbours of the
// least are within that of each other. Some 4000 pass before the first and after the last k block.
// `lines`: operand rows start on 128-byte lines; otherwise each of a block's 128-byte rows is two requests to L2.
double narrow_ns(int64_t m, int64_t n, int64_t k_blocks, int tile, int split, int sm_count, bool lines) {
  const double blocks = static_cast<double>((n + 127) / 128) * ((m + tile - 1) / tile) * split;
  const double kb = static_cast<double>((k_blocks + split - 1) / split);
  // One k block of one block's: what the tensor core takes for 128 x 64 or less, more with the bytes that the
  // SM has to fetch for it (and for the block it shares the SM with).
  const bool alone = blocks <= sm_count;
  const double k_block = (tile <= 32 ? (alone ? 210 : 235) : tile == 64 ? (alone ? 245 : 330) : (alone ? 345 : 430)) * (lines ? 1 : 1.5);
  const double waves = std::ceil(blocks / (2.0 * sm_count));
  const double fetch = blocks * kb * (16384 + 128.0 * tile) / (lines ? 17000 : 11300);
  // HBM at 5.0 TB/s with one block's ring in flight per SM, 6.2 with two; less if several blocks want the same rows.
  const double hbm = static_cast<double>(n) * k_blocks * 128 / (alone ? 5000 : 6200) * (m > tile ? 1.25 : 1);
  const double sharing = split > 1 ? waves * split * (200 + 6.0 * tile) : 0;
  return 4000 + 10.0 * tile + (waves - 1) * 2000 + std::max({waves * kb * k_block, fetch, hbm}) + sharing;
}

// tensor_store: the output's rows are whole 16-byte pieces. Other rows leave 64 bytes at a time, most of them
// parts of 32-byte sectors: four times as slow (1001 x 5120 x 4096: 21 us, x 4099: 29 us).
double wide_ns(int64_t m, int64_t n, int64_t k_blocks, int tile, int sm_count, bool lines, bool tensor_store) {
  const double tiles = static_cast<double>((m + 255) / 256) * ((n + tile - 1) / tile), pairs = sm_count / 2;
  const double waves = std::ceil(tiles / pairs);
  const double main_loop = k_blocks * (60 + 1.07 * tile) * (tiles > 0.6 * pairs ? 1.18 : 1) * (lines ? 1 : 1.25);  // L2 is shared by as many
  const double epilogue = tile * (tensor_store ? 10 : 38);
  // 256 columns leave no second accumulator, so nothing hides a tile's epilogue.
  return 4500 + (tile == 256 ? waves * (main_loop + epilogue) : waves * std::max(main_loop, epilogue) + epilogue);
}

Choice choose(const cake_scaled_matmul_desc& d, int64_t m, int sm_count, bool lines, bool tensor_store) {
  Choice best = {d.tile, d.k_split};
  const int64_t k_blocks = (d.k + cake::kBlockK - 1) / cake::kBlockK;
  double least = 0;
  for (int tile : {16, 32, 64, 128, 192, 224, 256}) {
    if (d.tile != 0 && tile != d.tile) continue;
    for (int split : {1, 2, 4, 8}) {
      if (split > 1 && (!is_narrow(tile) || split > k_blocks || (d.k_split != 0 && d.tile != 0))) break;
      const double ns = is_narrow(tile) ? narrow_ns(m, d.n, k_blocks, tile, split, sm_count, lines)
                                     : wide_ns(m, d.n, k_blocks, tile, sm_count, lines, tensor_store);
      if (least == 0 || ns < least) {
        least = ns;
        best = {tile, split};
      }
    }
  }
  if (d.k_split > 0) best.split = static_cast<int>(std::min<int64_t>(d.k_split, k_blocks));
  return best;
}

}  // namespace

extern "C" {

int32_t cake_scaled_matmul_enqueue(const cake_scaled_matmul_desc* desc, int64_t m, const void* lhs, int64_t lhs_row_stride,
                                   const void* lhs_scales, int64_t lhs_scales_row_stride, const void* rhs,
                                   int64_t rhs_row_stride, const void* rhs_scales, int64_t rhs_scales_row_stride,
                                   void* out, int64_t out_row_stride, int32_t* status_device, void* stream) {
  if (!desc) return fail(CAKE_ERR_INVALID_ARGUMENT, "cake_scaled_matmul_enqueue: null argument");
  const cake_scaled_matmul_desc& d = *desc;
  // Rows and columns are tensor-map coordinates; a tile past the end must not wrap around either. A tile's
  // contraction has to end well within the two seconds that a wait may take: 2^20 k blocks take 0.4.
  if (d.n < 1 || d.n > INT32_MAX / 2 || d.k < 1 || d.k >= (1 << 27))
    return fail(CAKE_ERR_INVALID_ARGUMENT, "scaled matmul extents must be n = 1 to 2^30 - 1 and k = 1 to 2^27 - 1: n=%lld k=%lld", (long long)d.n, (long long)d.k);
  if (d.out_dtype != CAKE_DTYPE_F32 && d.out_dtype != CAKE_DTYPE_BF16)
    return fail(CAKE_ERR_INVALID_ARGUMENT, "out_dtype must be CAKE_DTYPE_F32 or CAKE_DTYPE_BF16");
  if (d.tile != 0 && d.tile != 16 && d.tile != 32 && d.tile != 64 && d.tile != 128 && d.tile != 192 && d.tile != 224 && d.tile != 256)
    return fail(CAKE_ERR_UNSUPPORTED, "tile must be 0, 16, 32, 64, 128, 192, 224 or 256, got %d", d.tile);
  if (d.k_split < 0 || d.k_split > 8 || (d.k_split > 1 && (!is_narrow(d.tile) || d.tile == 0)))
    return fail(CAKE_ERR_INVALID_ARGUMENT, "k_split must be 0 to 8, and above 1 only with tile 16, 32, 64 or 128, got %d", d.k_split);
  if (m < 0 || m > INT32_MAX / 2) return fail(CAKE_ERR_INVALID_ARGUMENT, "m must be 0 to 2^30 - 1, got %lld", (long long)m);
  if (m == 0) return CAKE_OK;
  if (!lhs || !lhs_scales || !rhs || !rhs_scales || !out) return fail(CAKE_ERR_INVALID_ARGUMENT, "cake_scaled_matmul_enqueue: null argument");
  const int osize = d.out_dtype == CAKE_DTYPE_F32 ? 4 : 2;
  const int64_t k_blocks = (d.k + cake::kBlockK - 1) / cake::kBlockK;
  // With a single row its stride says nothing; tensor maps still want a valid one.
  const int64_t pitch = (d.k + 127) / 128 * 128;
  if (m == 1) {
    lhs_row_stride = pitch;
    out_row_stride = d.n;
  }
  if (d.n == 1) rhs_row_stride = pitch;
  if ((reinterpret_cast<uintptr_t>(lhs) | reinterpret_cast<uintptr_t>(rhs)) & 15)
    return fail(CAKE_ERR_INVALID_ARGUMENT, "lhs and rhs must be 16-byte aligned");
  if (lhs_row_stride % 16 || rhs_row_stride % 16 || lhs_row_stride < d.k || rhs_row_stride < d.k)
    return fail(CAKE_ERR_INVALID_ARGUMENT, "lhs and rhs row strides must be multiples of 16 bytes and at least k, got %lld and %lld",
                (long long)lhs_row_stride, (long long)rhs_row_stride);
  if ((m > 1 && lhs_scales_row_stride < k_blocks) || (d.n > 1 && rhs_scales_row_stride < k_blocks))
    return fail(CAKE_ERR_INVALID_ARGUMENT, "a scales row stride is shorter than its %lld scales", (long long)k_blocks);
  if (out_row_stride < d.n) return fail(CAKE_ERR_INVALID_ARGUMENT, "the output row stride is shorter than its row");
  if (reinterpret_cast<uintptr_t>(out) % osize) return fail(CAKE_ERR_INVALID_ARGUMENT, "out is not aligned to its elements");

  if (reinterpret_cast<uintptr_t>(status_device) & 3) return fail(CAKE_ERR_INVALID_ARGUMENT, "status_device must be 4-byte aligned");

  Device device;
  int32_t rc = current_device(&device);
  if (rc) return rc;
  // Tensor stores write whole 16-byte pieces, also where the row ends inside one: only rows of whole pieces
  // leave what lies behind them alone.
  const bool tensor_store = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && out_row_stride * osize % 16 == 0 && d.n * osize % 16 == 0;
  const bool lines = ((reinterpret_cast<uintptr_t>(lhs) | reinterpret_cast<uintptr_t>(rhs) | static_cast<uintptr_t>(lhs_row_stride) | static_cast<uintptr_t>(rhs_row_stride)) & 127) == 0;
  const Choice c = choose(d, m, device.sm_count, lines, tensor_store);
  const bool narrow = is_narrow(c.tile);
  cake::Params p;
  memset(&p, 0, sizeof(p));
  const int64_t rows_a = narrow ? d.n : m, rows_b = narrow ? m : d.n;
  p.rows_a = static_cast<int32_t>(rows_a);
  p.rows_b = static_cast<int32_t>(rows_b);
  const int64_t tile_rows = narrow ? cake::kRowsA : 2 * cake::kRowsA;
  const int64_t tiles_a = (rows_a + tile_rows - 1) / tile_rows, tiles_b = (rows_b + c.tile - 1) / c.tile;
  if (tiles_a * tiles_b * c.split > INT32_MAX / 2)
    return fail(CAKE_ERR_UNSUPPORTED, "%lld x %lld tiles are more than one launch covers", (long long)tiles_a, (long long)tiles_b);
  p.tiles_a = static_cast<int32_t>(tiles_a);
  p.tiles_b = static_cast<int32_t>(tiles_b);
  p.k_blocks = static_cast<int32_t>(k_blocks);
  p.split = c.split;
  p.out_f32 = osize == 4;
  p.scales_a = static_cast<const uint8_t*>(narrow ? rhs_scales : lhs_scales);
  p.scales_b = static_cast<const uint8_t*>(narrow ? lhs_scales : rhs_scales);
  p.scales_a_stride = narrow ? rhs_scales_row_stride : lhs_scales_row_stride;
  p.scales_b_stride = narrow ? lhs_scales_row_stride : rhs_scales_row_stride;
  p.out = out;
  p.out_stride = out_row_stride;
  p.status = status_device;
  p.tma_store = !narrow && tensor_store;

  CUtensorMap map_a, map_b, map_out;
  memset(&map_out, 0, sizeof(map_out));
  rc = encode_operand(&map_a, narrow ? rhs : lhs, rows_a, d.k, narrow ? rhs_row_stride : lhs_row_stride, cake::kRowsA);
  if (rc) return rc;
  rc = encode_operand(&map_b, narrow ? lhs : rhs, rows_b, d.k, narrow ? lhs_row_stride : rhs_row_stride, narrow ? c.tile : c.tile / 2);
  if (rc) return rc;
  if (p.tma_store) {
    const uint64_t dims[2] = {static_cast<uint64_t>(d.n), static_cast<uint64_t>(m)};
    const uint64_t strides[1] = {static_cast<uint64_t>(out_row_stride) * osize};
    const uint32_t box[2] = {32, 32};
    rc = cake::encode_tensor_map_as(&map_out, out, 2, dims, strides, box, osize == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                    osize == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
    if (rc) return rc;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (c.tile) {
    case 16: return launch<16, true>(device, map_a, map_b, map_out, p, s);
    case 32: return launch<32, true>(device, map_a, map_b, map_out, p, s);
    case 64: return launch<64, true>(device, map_a, map_b, map_out, p, s);
    case 128: return launch<128, true>(device, map_a, map_b, map_out, p, s);
    case 192: return launch<192, false>(device, map_a, map_b, map_out, p, s);
    case 224: return launch<224, false>(device, map_a, map_b, map_out, p, s);
    default: return launch<256, false>(device, map_a, map_b, map_out, p, s);
  }
}

}  // extern "C"
