// Low-rank adapters of many requests beside one shared projection (gemm_sm100_lora*):
//   low[m]  = s_g A[m] down_g^T            d_low[m] = s_g dC[m] up_g
//   C[m]   += low[m] up_g^T                dA[m]   += d_low[m] down_g
//   d_down_g = sum_{m of g} d_low[m]^T A[m]        d_up_g = sum_{m of g} dC[m]^T low[m]
// with g the adapter of row m.  Accumulation in fp32; low and d_low are rounded once to the operands'
// 16-bit type, because the products that read them run on 16-bit tensor core operands.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "gemm_tn_sm100.cuh"

namespace gemm_sm100 {

constexpr int kLoraTileRows = 256;   // rows of one slot list: the rows of a pair tile of the GEMM

// Device layout of a plan (32-bit words).  The rows are cut into tiles of 256; a tile's "slots" are the
// distinct adapters among its rows in order of first appearance, each with a 256-bit row mask.  `order`
// lists the rows that have an adapter, grouped by adapter and ascending inside a group; `offsets`
// are the groups' starts.
struct LoraPlanView {
  int* slot_count;       // [tiles]
  int* slot_adapter;     // [tiles][256]
  uint32_t* slot_mask;   // [tiles][256][8]: bit r % 32 of word r / 32 is row r of the tile
  int* row_slot;         // [M]: the row's slot in its tile, -1 for rows without an adapter
  int* order;            // [M]
  int* offsets;          // [adapters + 1]
};

__host__ __device__ inline long lora_plan_tiles(long M) { return (M + kLoraTileRows - 1) / kLoraTileRows; }
__host__ __device__ inline long lora_plan_round(long words) { return (words + 63) / 64 * 64; }

__host__ __device__ inline long lora_plan_words(long M, long adapters) {
  const long tiles = lora_plan_tiles(M);
  return lora_plan_round(tiles) + tiles * kLoraTileRows * 9 + 2 * lora_plan_round(M) + lora_plan_round(adapters + 1);
}

__host__ __device__ inline LoraPlanView lora_plan_view(void* plan, long M) {
  const long tiles = lora_plan_tiles(M);
  LoraPlanView v;
  v.slot_count = static_cast<int*>(plan);
  v.slot_adapter = v.slot_count + lora_plan_round(tiles);
  v.slot_mask = reinterpret_cast<uint32_t*>(v.slot_adapter + tiles * kLoraTileRows);
  v.row_slot = reinterpret_cast<int*>(v.slot_mask + tiles * kLoraTileRows * 8);
  v.order = v.row_slot + lora_plan_round(M);
  v.offsets = v.order + lora_plan_round(M);
  return v;
}

__device__ __forceinline__ int lora_read_id(const void* ids, int ids_are_64, long row, int adapters) {
  const long long id = ids_are_64 ? static_cast<const long long*>(ids)[row] : static_cast<const int*>(ids)[row];
  return id >= 0 && id < adapters ? static_cast<int>(id) : -1;
}

// One launch, 256 threads a block.  Block t < tiles: the slot list of tile t.  Block tiles + g: the rows of
// adapter g in ascending order; their place in `order` is the number of rows of adapters below g,
// which the block counts itself, so that no block waits for another.  Every adapter's block reads all indices from L2, and
// reads them again if the adapter has rows: for 64 adapters and 8192 rows 4 MB of 32-bit indices, 8 MB of 64-bit ones.
// Measured: 128 rows of 16 adapters 4.0 us, 1024 of 64 8.7, 8192 of up to 64 8.9 (the chain of 32 blocks of 256 rows is what
// takes the time), 8192 of 4096 100, 65536 of 64 98.
__global__ void __launch_bounds__(256) lora_plan_kernel(const void* ids, int ids_are_64, int M, int adapters, void* plan) {
  const LoraPlanView v = lora_plan_view(plan, M);
  const int tiles = static_cast<int>(lora_plan_tiles(M));
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  __shared__ int s_id[256];
  __shared__ int s_slot[256];
  __shared__ uint32_t s_mask[256][8];
  __shared__ int s_warp[8];
  __shared__ int s_below[8];
  if (static_cast<int>(blockIdx.x) < tiles) {
    const int tile = blockIdx.x;
    const long row = static_cast<long>(tile) * kLoraTileRows + t;
    const int id = row < M ? lora_read_id(ids, ids_are_64, row, adapters) : -1;
    s_id[t] = id;
    for (int w = 0; w < 8; ++w) s_mask[t][w] = 0;
    __syncthreads();
    int first = t;
    if (id >= 0)
      for (first = 0; s_id[first] != id; ++first) {
      }
    const bool opens = id >= 0 && first == t;
    const uint32_t ballot = __ballot_sync(0xffffffffu, opens);
    if (lane == 0) s_warp[warp] = __popc(ballot);
    __syncthreads();
    int slot = __popc(ballot & ((1u << lane) - 1u));
    int count = 0;
    for (int w = 0; w < 8; ++w) {
      if (w < warp) slot += s_warp[w];
      count += s_warp[w];
    }
    if (opens) s_slot[t] = slot;
    __syncthreads();
    if (id >= 0) atomicOr(&s_mask[s_slot[first]][warp], 1u << lane);   // the same mask in whatever order
    if (row < M) v.row_slot[row] = id >= 0 ? s_slot[first] : -1;
    if (opens) v.slot_adapter[tile * kLoraTileRows + slot] = id;
    if (t == 0) v.slot_count[tile] = count;
    __syncthreads();
    if (t < count)
      for (int w = 0; w < 8; ++w) v.slot_mask[(static_cast<long>(tile) * kLoraTileRows + t) * 8 + w] = s_mask[t][w];
    return;
  }
  const int g = blockIdx.x - tiles;
  int below = 0, own = 0;
  for (long row = t; row < M; row += 256) {
    const int id = lora_read_id(ids, ids_are_64, row, adapters);
    below += id >= 0 && id < g;
    own += id == g;
  }
  for (int o = 16; o > 0; o >>= 1) {
    below += __shfl_xor_sync(0xffffffffu, below, o);
    own += __shfl_xor_sync(0xffffffffu, own, o);
  }
  if (lane == 0) {
    s_below[warp] = below;
    s_warp[warp] = own;
  }
  __syncthreads();
  int base = 0, total = 0;
  for (int w = 0; w < 8; ++w) {
    base += s_below[w];
    total += s_warp[w];
  }
  if (t == 0) {
    v.offsets[g] = base;
    if (g == adapters - 1) v.offsets[adapters] = base + total;
  }
  if (total == 0) return;
  for (long row0 = 0; row0 < M; row0 += 256) {
    const long row = row0 + t;
    const bool mine = row < M && lora_read_id(ids, ids_are_64, row, adapters) == g;
    const uint32_t ballot = __ballot_sync(0xffffffffu, mine);
    __syncthreads();
    if (lane == 0) s_warp[warp] = __popc(ballot);
    __syncthreads();
    int at = base + __popc(ballot & ((1u << lane) - 1u));
    for (int w = 0; w < 8; ++w) {
      if (w < warp) at += s_warp[w];
      base += s_warp[w];
    }
    if (mine) v.order[at] = static_cast<int>(row);
  }
}

// The ranks that make one swizzle row of 32, 64 or 128 bytes in shared memory.
__host__ __device__ constexpr int rank_chunk(int R) { return R <= 16 ? 16 : (R <= 32 ? 32 : 64); }

// ------------------------------------------------------------------------------ low-rank rows
// low[m] = s_g P[m] W_g^T over the long axis L: P = A and W = down [R, L], or (kRankInner) P = dC and W = up
// [L, R].  A tile of 128 rows is one MMA operand; the adapters of the plan's tile (256 rows: this tile's and its
// neighbour's, so an adapter that only the neighbour uses is multiplied in vain) lie side by side along
// the MMA's N, in groups of up to 128 columns, so that P is read once however many adapters a group
// holds, and every row takes its own adapter's columns out of the accumulator.  The work is a read of
// P and, per pair of tiles, of its adapters: bytes, not products, bound it.  L is cut over the CTAs of a cluster, which
// add their partial rows through distributed shared memory in rank order.
// Measured: 8192 x 4096 with rank 16 16.4 to 17.3 us (67.2 MB, 4 TB/s; about 5 us of it are launch, first loads and exchange), with a cold
// L2 19.5 to 21.7; 8192 x 14336 with rank 64 45 us at 5.4 TB/s; 64 x 14336 with 32 adapters of
// rank 64 (61 MB, nearly all adapters) 19.7 us.  Groups of 128 columns because two CTAs with three stages of 32 KB
// then share an SM; the alternative of one product per adapter and row tile reads P once per adapter.
struct LowParams {
  CUtensorMap tmap_p;    // [M, L]: boxes of 64 x p_rows
  CUtensorMap tmap_w;    // [adapters, R, L]: boxes of 64 x R, or [adapters, L, R]: boxes of a chunk of ranks x 64
  const void* plan;
  const float* scales;
  float scale;
  void* out;             // [M, R], pitch ld_out
  long ld_out;
  int M, R, L;
  int p_rows;            // rows per box of P: 128, or fewer when M is
  int splits;            // partial sums of a row: L is cut over as many CTAs, or over half of them with two sums each
  int clusters;          // clusters per tile; the tile's groups are dealt to them
  int group_slots;       // adapters per group
  int groups;            // groups that are taken one to a cluster of `splits` sums; with more, fewer sums of each are formed
  unsigned int* status;
  unsigned long long timeout_ns;
};

// kDeep: six stages and one CTA per SM instead of three and two (chosen by low_grid).
template <bool kDeep>
struct LowConfig {
  static constexpr int kThreads = 192;                 // producer, MMA issuer, four epilogue warps
  static constexpr int kStages = kDeep ? 6 : 3;
  static constexpr int kPBytes = 128 * 64 * 2, kWBytes = 128 * 64 * 2;
  static constexpr int kStageBytes = kPBytes + kWBytes;
  static constexpr int kTmemCols = 256;                // two accumulators of 128 columns
  static constexpr int kMaxFoldedRank = kStages * kStageBytes / (2 * 128 * 4) / 8 * 8 - 8;   // two sets of partial rows in the ring
  static_assert(2 * 128 * (kMaxFoldedRank + 4) * 4 <= kStages * kStageBytes, "partial rows");
  static constexpr int kBarrierBytes = 128;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kBarrierBytes + 128 * 8;
};

template <bool kIsBf16, bool kRankInner, bool kDeep>
__device__ __forceinline__ void lora_low_body(const LowParams& p, const int block) {
  using Cfg = LowConfig<kDeep>;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t smem_p = base, smem_w = base + kStages * Cfg::kPBytes;
  uint8_t* bar_mem = smem_raw + (base - smem_u32(smem_raw)) + kStages * Cfg::kStageBytes;
  const uint32_t full = smem_u32(bar_mem), empty = full + 8u * kStages, done = empty + 8u * kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_mem + 8 * (2 * kStages + 1));
  volatile uint32_t* abort_flag = tmem_slot + 1;
  int* row_slot = reinterpret_cast<int*>(bar_mem + Cfg::kBarrierBytes);
  float* row_factor = reinterpret_cast<float*>(row_slot + 128);
  const int warp = threadIdx.x >> 5;
  const uint32_t lane = lane_id();
  const int rank = static_cast<int>(cluster_ctarank());
  uint32_t cluster_size;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(cluster_size));
  const int unit = block / static_cast<int>(cluster_size);
  const int tile = unit / p.clusters, group0 = unit % p.clusters;
  WaitCtx ctx{abort_flag, smem_u32(const_cast<const uint32_t*>(abort_flag)), p.status, p.timeout_ns};

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    prefetch_tensormap(&p.tmap_p);
    prefetch_tensormap(&p.tmap_w);
    for (int b = 0; b < 2 * kStages + 1; ++b) mbar_init(full + 8u * b, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(tmem_slot), Cfg::kTmemCols);
    tmem_relinquish<1>();
    tc_fence_before_sync();
  }
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();
  // only now: the product kernel behind this one relies on everything before this kernel being complete
  grid_launch_dependents();

  const LoraPlanView v = lora_plan_view(const_cast<void*>(p.plan), p.M);
  const int tile256 = tile >> 1;
  const int slots = v.slot_count[tile256];
  const int* adapters = v.slot_adapter + tile256 * kLoraTileRows;
  const int k_blocks = (p.L + 63) / 64;
  const int R = p.R;
  // columns of the accumulator per adapter: the ranks, or whole chunks of them
  const int chunk = rank_chunk(R), slot_cols = kRankInner ? (R + chunk - 1) / chunk * chunk : R;
  const int groups = slots == 0 ? 1 : (slots + p.group_slots - 1) / p.group_slots;   // (no slot: zeros are written)
  // A tile with more groups than clusters: the cluster takes up to `splits` groups at once and forms fewer partial sums of
  // each (one exchange instead of one per group: 2048 x (4096 + 4096), 16 adapters of rank 32 in every tile, 38 us one after
  // another).  `sums` follows from the problem alone, for it is the order in which a row is added up; where the CTAs are
  // half as many, each has every second of its K blocks in a second accumulator.
  // (All of these are powers of two.  The clusters of a shared launch may be larger than `splits`.)
  int sums = p.splits;
  for (int taken = p.groups; sums > 1 && taken < groups; taken *= 2) sums >>= 1;
  int parts_log = __ffs(min(sums, static_cast<int>(cluster_size))) - 1;
  if (1 << parts_log == sums && sums > 1 && static_cast<int>(cluster_size >> parts_log) * p.clusters < groups) --parts_log;
  const int parts = 1 << parts_log, at_once = static_cast<int>(cluster_size >> parts_log);
  const int part = rank & (parts - 1), leader = rank - part;
  const uint32_t second = parts < sums ? 128u : 0u;    // column of the second accumulator
  // The CTAs of a part take the K blocks in turn: what they read of a row of P at any moment is contiguous.
  const int steps = (k_blocks - part + parts - 1) >> parts_log;
  const int pitch = R + 4;                             // floats per partial row: 16-byte accesses without bank conflicts
  uint32_t step = 0;                                   // ring position, running on over the groups
  uint32_t parity = 0;
  if (warp >= 2) {
    // every row's slot and factor, while the first operands are on their way
    const int row = (warp & 3) * 32 + static_cast<int>(lane);
    const long m = static_cast<long>(tile) * 128 + row;
    const int slot = m < p.M ? v.row_slot[m] : -1;
    row_slot[row] = slot;
    row_factor[row] = slot >= 0 && p.scales ? p.scale * p.scales[adapters[slot]] : p.scale;
    __syncwarp();
  }
#pragma unroll 1
  for (int first = group0 * at_once; first < groups; first += p.clusters * at_once) {
    const int group = first + (rank >> parts_log);
    const int slot0 = group * p.group_slots;
    const int n_slots = min(p.group_slots, slots - slot0);   // (none left: the CTA only takes part in the exchange)
    const bool ok = *abort_flag == 0;
    if (n_slots > 0 && ok) {
      if (warp == 0) {
        const uint64_t pol = policy_evict_normal();
        const bool issuer = elect_one();
        const uint32_t w_bytes = static_cast<uint32_t>(slot_cols) * 128u;
        const uint32_t bytes = static_cast<uint32_t>(p.p_rows) * 128u + n_slots * w_bytes;
        const int my_adapter = static_cast<int>(lane) < n_slots ? adapters[slot0 + lane] : 0;
        uint32_t at = step;
        for (int kb = part; kb < k_blocks; kb += parts, ++at) {
          const uint32_t s = at % kStages;
          if (!wait_bounded(empty + 8u * s, ((at / kStages) & 1u) ^ 1u, ctx, kStatusTimeoutProducer)) break;
          if (issuer) {
            mbar_arrive_expect_tx(full + 8u * s, bytes);
            tma_load_2d<1>(smem_p + s * Cfg::kPBytes, &p.tmap_p, full + 8u * s, kb * 64, tile * 128, pol);
          }
          for (int j = 0; j < n_slots; ++j) {
            const int g = __shfl_sync(0xffffffffu, my_adapter, j);
            const uint32_t dst = smem_w + s * Cfg::kWBytes + j * w_bytes;
            if (issuer) {
              if constexpr (!kRankInner) {
                tma_load_3d<1>(dst, &p.tmap_w, full + 8u * s, kb * 64, 0, g, pol);
              } else {
                for (int r = 0; r < R; r += chunk) tma_load_3d<1>(dst + r * 128, &p.tmap_w, full + 8u * s, r, kb * 64, g, pol);
              }
            }
          }
          __syncwarp();
        }
      } else if (warp == 1) {
        const bool issuer = elect_one();
        const int n = (n_slots * slot_cols + 15) / 16 * 16;
        const uint32_t idesc = make_idesc_f16(kIsBf16 ? 1u : 0u, 128, static_cast<uint32_t>(n), kRankInner ? 1u : 0u, 0);
        uint32_t at = step;
        for (int i = 0; i < steps; ++i, ++at) {
          const uint32_t s = at % kStages;
          if (!wait_bounded(full + 8u * s, (at / kStages) & 1u, ctx, kStatusTimeoutMma)) break;
          tc_fence_after_sync();
          if (issuer) {
            const uint32_t acc = tmem + (i & 1 ? second : 0u);
            const bool begun = i > (second != 0u ? 1 : 0);
            const uint64_t dp = make_smem_desc_sw128(smem_p + s * Cfg::kPBytes);
            if constexpr (!kRankInner) {
              const uint64_t dw = make_smem_desc_sw128(smem_w + s * Cfg::kWBytes);
#pragma unroll
              for (int k = 0; k < 4; ++k) umma_f16<1>(acc, dp + 2u * k, dw + 2u * k, idesc, begun || k > 0);
            } else {
              const uint64_t dw = make_smem_desc_rows_mn(smem_w + s * Cfg::kWBytes, chunk * 2u, chunk * 128u);
#pragma unroll
              for (int k = 0; k < 4; ++k) umma_f16<1>(acc, dp + 2u * k, dw + 2u * chunk * k, idesc, begun || k > 0);
            }
            umma_commit<1>(empty + 8u * s);
            if (i == steps - 1) umma_commit<1>(done);
          }
          __syncwarp();
        }
      } else {
        // Every row's own columns, into the partial rows (the idle ring: all its loads have been consumed).
        const int q = warp & 3;
        const int row = q * 32 + static_cast<int>(lane);
        const int mine = row_slot[row] - slot0;
        if (wait_bounded(done, parity, ctx, kStatusTimeoutEpilogue)) {
          tc_fence_after_sync();
          const uint32_t dst = base + static_cast<uint32_t>(row * pitch) * 4u, lanes = tmem + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
          for (int j = 0; j < n_slots; ++j) {
            if (!__any_sync(0xffffffffu, mine == j)) continue;
            for (int r = 0; r < R; r += 8) {
              uint32_t x[8], y[8];
              tmem_ld_32x8(lanes + j * slot_cols + r, x);
              if (second != 0u) tmem_ld_32x8(lanes + second + j * slot_cols + r, y);
              tmem_ld_wait();
              if (mine == j) {
                const uint32_t to = dst + r * 4u, to2 = to + 128u * 4u * static_cast<uint32_t>(pitch);
                st_shared_v4(to, x[0], x[1], x[2], x[3]);
                st_shared_v4(to + 16u, x[4], x[5], x[6], x[7]);
                if (second != 0u) {
                  st_shared_v4(to2, y[0], y[1], y[2], y[3]);
                  st_shared_v4(to2 + 16u, y[4], y[5], y[6], y[7]);
                }
              }
            }
          }
          tc_fence_before_sync();
        }
      }
      step += static_cast<uint32_t>(steps);
      parity ^= 1u;
    }
    // every CTA's partial rows are written
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    // This CTA's share of the rows, summed over the parts' sums in their order.
    const int share = 128 >> parts_log, quads = R / 4;
    for (int i = threadIdx.x; i < share * quads; i += Cfg::kThreads) {
      const int row = part * share + i / quads, r = i % quads * 4;
      const long m = static_cast<long>(tile) * 128 + row;
      if (m >= p.M) break;
      const int slot = row_slot[row];
      uint16_t* out = static_cast<uint16_t*>(p.out) + m * p.ld_out + r;
      if (slot < 0) {
        if (group == 0) *reinterpret_cast<uint2*>(out) = make_uint2(0u, 0u);
        continue;
      }
      if (slot < slot0 || slot >= slot0 + n_slots || !ok) continue;
      const uint32_t src = base + static_cast<uint32_t>(row * pitch + r) * 4u;
      float4 x[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < sums)
          x[c] = ld_cluster_v4(map_to_cta(src + (c < parts ? 0u : 128u * static_cast<uint32_t>(pitch) * 4u),
                                          static_cast<uint32_t>(leader + (c < parts ? c : c - parts))));
      float4 sum = x[0];
#pragma unroll
      for (int c = 1; c < 8; ++c)
        if (c < sums) sum.x += x[c].x, sum.y += x[c].y, sum.z += x[c].z, sum.w += x[c].w;
      const float f = row_factor[row];
      *reinterpret_cast<uint2*>(out) =
          make_uint2(pack2<kIsBf16>(__float_as_uint(sum.x * f), __float_as_uint(sum.y * f)),
                     pack2<kIsBf16>(__float_as_uint(sum.z * f), __float_as_uint(sum.w * f)));
    }
    // the partial rows may go (to the next group's loads, or with the CTA); the plain reads and writes of the
    // ring come before the next group's asynchronous ones
    fence_proxy_async_smem();
    cluster_arrive();
    cluster_wait();
  }

  if (*abort_flag != 0) {
#pragma unroll 1
    for (int i = 0; i < 200; ++i) __nanosleep(1000);   // a wait gave up: loads in flight land before the memory goes
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem, Cfg::kTmemCols);
  }
}

template <bool kIsBf16, bool kRankInner, bool kDeep>
__global__ void __launch_bounds__(192, kDeep ? 1 : 2) lora_low_kernel(const __grid_constant__ LowParams p) {
  lora_low_body<kIsBf16, kRankInner, kDeep>(p, static_cast<int>(blockIdx.x));
}

// Both kinds of rows in one launch, for a backward pass that computes the low rows again: the first `blocks` CTAs
// low, the others d_low.  Each adds its rows up as a launch of its own does, so that they have the same bits.
template <bool kIsBf16, bool kDeep>
__global__ void __launch_bounds__(192, kDeep ? 1 : 2)
lora_low_pair_kernel(const __grid_constant__ LowParams low, const __grid_constant__ LowParams d_low, const int blocks) {
  if (static_cast<int>(blockIdx.x) < blocks)
    lora_low_body<kIsBf16, false, kDeep>(low, static_cast<int>(blockIdx.x));
  else
    lora_low_body<kIsBf16, true, kDeep>(d_low, static_cast<int>(blockIdx.x) - blocks);
}

// ------------------------------------------------------------------------------ adapters' gradients
// out_g[i, r] = sum over the rows m of adapter g of P[m, i] Q[m, r]: d_down (P = A, Q = d_low, stored as [R, D])
// and d_up (P = dC, Q = low, stored as [D, R]).  128 columns i of P are the MMA's M, the ranks its N, and the
// rows are contracted: P and Q go to the tensor core as they lie in memory, as MN-major operands.  The rows of
// an adapter may be anywhere in the batch, so threads gather them (plan order) with 16-byte asynchronous
// copies into the swizzled tiles; places behind the last row are filled with zeros in both operands and read
// nothing.  One read of P bounds it: 8192 x (4096 + 4096) with rank 16 takes 29.7 us (134.8 MB from DRAM, 4.5 TB/s), 8192 x
// (14336 + 4096) with 8 adapters of rank 64 97 us (3.1 TB/s; Q, read again for every column tile, is half of P there).
// Work: a column tile of one adapter, whose rows are cut over `splits` CTAs of a cluster of four (1, 2 or 4: the
// fewest with at most `split_rows` rows each), which add their partial sums through distributed shared
// memory in rank order.  The cluster takes 4 / splits neighbouring tiles at once, and a grid that fills the
// device walks over all adapters' groups of tiles.
struct GradSide {
  const uint16_t* P;
  const uint16_t* Q;
  uint16_t* out;
  long ldp, ldq;
  int D;                 // columns of P; 0: this gradient is not wanted
  int rank_outer;        // 1: out is [R, D], 0: [D, R]
};
struct GradParams {
  GradSide side[2];
  const void* plan;
  int M, R, adapters;
  int tiles0, tiles;     // column tiles of side 0, and of both sides
  int split_rows;
  unsigned int* status;
  unsigned long long timeout_ns;
};

constexpr int kGradCluster = 4;
template <int kRanks>   // R rounded up to whole chunks: 16, 32, 64 or 128
struct GradConfig {
  static constexpr int kThreads = 160;                 // four warps gather and store, one issues
  static constexpr int kRows = 64;                     // rows per ring stage
  static constexpr int kStages = kRanks <= 16 ? 4 : 3;
  static constexpr int kBlockBytes = kRows * 128;      // 64 columns of a stage
  static constexpr int kPBytes = 2 * kBlockBytes, kQBytes = kRows * kRanks * 2;
  static constexpr int kChunk = rank_chunk(kRanks);
  static constexpr int kStageBytes = kPBytes + kQBytes;
  static constexpr int kTmemCols = kRanks < 32 ? 32 : kRanks;
  static constexpr int kCtasPerSm = kRanks <= 64 ? 3 : 2;
  // the partial sums of a cut tile lie in the ring: 128 columns x (R + 4), or R x (128 + 4) floats
  static_assert(kStages * kStageBytes >= 128 * (kRanks + 4) * 4 && kStages * kStageBytes >= kRanks * 132 * 4, "partial sums");
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + 128;
  static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 233472, "shared memory of an SM");
};

template <bool kIsBf16, int kRanks>
__global__ void __launch_bounds__(160, GradConfig<kRanks>::kCtasPerSm)
lora_grad_kernel(const __grid_constant__ GradParams p) {
  using Cfg = GradConfig<kRanks>;
  constexpr int kStages = Cfg::kStages, kRows = Cfg::kRows;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t smem_p = base, smem_q = base + kStages * Cfg::kPBytes;
  uint8_t* bar_mem = smem_raw + (base - smem_u32(smem_raw)) + kStages * Cfg::kStageBytes;
  const uint32_t full = smem_u32(bar_mem), empty = full + 8u * kStages, done = empty + 8u * kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_mem + 8 * (2 * kStages + 1));
  volatile uint32_t* abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5;
  const uint32_t lane = lane_id();
  const int rank = static_cast<int>(cluster_ctarank());
  const int cluster = static_cast<int>(blockIdx.x) / kGradCluster, clusters = static_cast<int>(gridDim.x) / kGradCluster;
  WaitCtx ctx{abort_flag, smem_u32(const_cast<const uint32_t*>(abort_flag)), p.status, p.timeout_ns};

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int b = 0; b < kStages; ++b) {
      mbar_init(full + 8u * b, 128);
      mbar_init(empty + 8u * b, 1);
    }
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == 4) {
    tmem_alloc<1>(smem_u32(tmem_slot), Cfg::kTmemCols);
    tmem_relinquish<1>();
    tc_fence_before_sync();
  }
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_launch_dependents();
  grid_dependency_wait();

  const LoraPlanView v = lora_plan_view(const_cast<void*>(p.plan), p.M);
  const int R = p.R;
  uint32_t n = 0;                                        // ring position, running on over the units
  uint32_t rounds = 0;                                   // uses of the accumulator so far
  // The adapters' groups of tiles, one adapter after another, are the units of the grid; clusters take them in
  // turn.  Every warp finds its units by itself, 32 adapters at a time.
  int u = cluster, batch_start = 0;
  int empties = 0;
  const long zeros = (static_cast<long>(p.side[0].D) + p.side[1].D) * R / 8;     // 16-byte pieces per adapter
  const int fill = static_cast<int>(min(static_cast<long>(gridDim.x), zeros / (Cfg::kThreads * 4) + 1));
#pragma unroll 1
  for (int g0 = 0; g0 < p.adapters; g0 += 32) {
    int my_first = 0, my_last = 0, my_splits = 1, my_end = 0;
    if (g0 + static_cast<int>(lane) < p.adapters) {
      my_first = v.offsets[g0 + lane];
      my_last = v.offsets[g0 + lane + 1];
      while (my_splits < kGradCluster && my_last - my_first > p.split_rows * my_splits) my_splits *= 2;
      if (my_last > my_first) my_end = (p.tiles * my_splits + kGradCluster - 1) / kGradCluster;
    }
    for (int o = 1; o < 32; o *= 2) {
      const int below = __shfl_up_sync(0xffffffffu, my_end, o);
      if (static_cast<int>(lane) >= o) my_end += below;
    }
    my_end += batch_start;                               // where this lane's adapter ends in the grid's units
    // Adapters without rows have no units.  Their zeros are contiguous memory, written by `fill` CTAs per adapter, the
    // next ones for every further adapter; a lane finds out whether this CTA writes for its adapter.
    const bool empty_here = my_last == my_first && g0 + static_cast<int>(lane) < p.adapters;
    const uint32_t all_empty = __ballot_sync(0xffffffffu, empty_here);
    const int order = empties + __popc(all_empty & ((1u << lane) - 1u));
    empties += __popc(all_empty);
    const int grid = static_cast<int>(gridDim.x);
    const int turn = static_cast<int>((static_cast<long>(grid) + blockIdx.x - static_cast<long>(order) * fill % grid) % grid);
    for (uint32_t mine = __ballot_sync(0xffffffffu, empty_here && turn < fill); mine != 0; mine &= mine - 1) {
      const int from = __ffs(static_cast<int>(mine)) - 1;
      const long g = g0 + from;
      const int part = __shfl_sync(0xffffffffu, turn, from);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const long pieces = static_cast<long>(p.side[x].D) * R / 8;          // of 16 bytes
        uint4* out = reinterpret_cast<uint4*>(p.side[x].out + g * p.side[x].D * R);
        for (long i = static_cast<long>(part) * Cfg::kThreads + threadIdx.x; i < pieces; i += static_cast<long>(fill) * Cfg::kThreads)
          out[i] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    const int batch_end = __shfl_sync(0xffffffffu, my_end, 31);
#pragma unroll 1
    for (; u < batch_end; u += clusters) {
      const int owner = __popc(__ballot_sync(0xffffffffu, my_end <= u));
      const int g = g0 + owner;
      const int first = __shfl_sync(0xffffffffu, my_first, owner), last = __shfl_sync(0xffffffffu, my_last, owner);
      const int splits = __shfl_sync(0xffffffffu, my_splits, owner), group_tiles = kGradCluster / splits;
      const int start_of = __shfl_sync(0xffffffffu, my_end, owner > 0 ? owner - 1 : 0);
      const int start = owner > 0 ? start_of : batch_start;
      const int tile = (u - start) * group_tiles + rank / splits, part = rank % splits;
      const bool work = tile < p.tiles && *abort_flag == 0;
      const GradSide& side = p.side[tile < p.tiles0 ? 0 : 1];
      const int col0 = (tile < p.tiles0 ? tile : tile - p.tiles0) * 128;
      const int blocks = (last - first + kRows - 1) / kRows;
      const int shift = __popc(splits - 1);
      auto block_of = [&](int c) { return static_cast<int>((static_cast<long>(blocks) * c) >> shift); };
      const int b0 = block_of(part), b1 = block_of(part + 1);
      const int pitch = side.rank_outer ? 128 + 4 : R + 4;   // floats per row of the partial sums: [r][i] or [i][r]
      if (work && b1 > b0) {
        if (warp < 4) {
          // Thread: 16-byte piece `piece` of the rows tid / 16 + 8 k of every block, and the same piece of Q
          // where Q has it; two 64-column blocks of P, 128-byte swizzle.
          const int tid = threadIdx.x, piece = tid & 15, r0 = tid >> 4;
          const bool col_ok = col0 + piece * 8 < side.D, q_ok = piece * 8 < R;
          const uint16_t* src_p = side.P + (col_ok ? col0 + piece * 8 : 0);
          const uint16_t* src_q = side.Q + (q_ok ? piece * 8 : 0);
          const long ldp = side.ldp, ldq = side.ldq;
          // row t of a block sits at t * 128, its piece c at c ^ (t % 8); t % 8 == r0 for all of this thread's rows
          const uint32_t place = static_cast<uint32_t>((piece >> 3) * Cfg::kBlockBytes + r0 * 128 + (((piece & 7) ^ r0) << 4));
          // Q likewise, in rows of one chunk of ranks with the swizzle of that width
          constexpr int kPieces = Cfg::kChunk / 8;
          const int turn = kPieces == 8 ? r0 : (kPieces == 4 ? r0 >> 1 : r0 >> 2);
          const uint32_t place_q = static_cast<uint32_t>((piece / kPieces) * (kRows * Cfg::kChunk * 2) + r0 * Cfg::kChunk * 2 +
                                                         (((piece % kPieces) ^ turn) << 4));
          // The rows' places in the batch, kRows / 4 per warp and block: a lane loads one of the next two blocks'
          // entries, two blocks ahead of their use (one block ahead, their latency was every block's time).
          auto fetch_rows = [&](int b) {
            const int e = static_cast<int>(lane) & 15;
            const int block = b + (static_cast<int>(lane) >> 4), at = first + block * kRows + warp * 2 + (e >> 3) + 8 * (e & 7);
            return block < b1 && at < last ? v.order[at] : -1;
          };
          int rows_now = fetch_rows(b0), rows_next = fetch_rows(b0 + 2);
          int taken = 0;                                 // stages filled in this unit
          for (int b = b0; b < b1; ++b, ++taken) {
            const uint32_t at = n + static_cast<uint32_t>(taken), s = at % kStages;
            if (!wait_bounded(empty + 8u * s, ((at / kStages) & 1u) ^ 1u, ctx, kStatusTimeoutProducer)) break;
            const uint32_t dst_p = smem_p + s * Cfg::kPBytes + place, dst_q = smem_q + s * Cfg::kQBytes + place_q;
#pragma unroll
            for (int k = 0; k < kRows / 8; ++k) {
              const int row = __shfl_sync(0xffffffffu, rows_now, (taken & 1) * 16 + static_cast<int>(lane >> 4) * 8 + k);
              const bool live = row >= 0;
              const long m = live ? row : 0;
              cp_async_16(dst_p + k * 1024u, src_p + m * ldp, live && col_ok);
              if (q_ok) cp_async_16(dst_q + k * (8u * Cfg::kChunk * 2u), src_q + m * ldq, live);
            }
            cp_async_arrive(full + 8u * s);
            if (taken & 1) {
              rows_now = rows_next;
              rows_next = fetch_rows(b + 3);
            }
          }
          __syncwarp();
          if (wait_bounded(done, rounds & 1u, ctx, kStatusTimeoutEpilogue)) {
            // the partial sums, into the idle ring
            tc_fence_after_sync();
            const int i = warp * 32 + static_cast<int>(lane);
            for (int r = 0; r < R; r += 8) {
              uint32_t x[8];
              tmem_ld_32x8(tmem + (static_cast<uint32_t>(warp * 32) << 16) + r, x);
              tmem_ld_wait();
              if (splits == 1) {
                // nobody to add: straight to memory
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = pack2<kIsBf16>(x[2 * e], x[2 * e + 1]);
                uint16_t* out = side.out + static_cast<long>(g) * side.D * R;
                if (col0 + i < side.D) {
                  if (side.rank_outer) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                      out[static_cast<long>(r + e) * side.D + col0 + i] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
                  } else {
                    *reinterpret_cast<uint4*>(out + static_cast<long>(col0 + i) * R + r) = make_uint4(w[0], w[1], w[2], w[3]);
                  }
                }
              } else if (side.rank_outer) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  asm volatile("st.shared.b32 [%0], %1;" ::"r"(base + static_cast<uint32_t>((r + e) * pitch + i) * 4u), "r"(x[e])
                               : "memory");
              } else {
                const uint32_t dst = base + static_cast<uint32_t>(i * pitch + r) * 4u;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                             : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 16u), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
                             : "memory");
              }
            }
            tc_fence_before_sync();
          }
        } else {
          const bool issuer = elect_one();
          const uint32_t idesc = make_idesc_f16(kIsBf16 ? 1u : 0u, 128, static_cast<uint32_t>((R + 15) / 16 * 16), 1u, 1u);
          uint32_t at = n;
          for (int b = b0; b < b1; ++b, ++at) {
            const uint32_t s = at % kStages;
            if (!wait_bounded(full + 8u * s, (at / kStages) & 1u, ctx, kStatusTimeoutMma)) break;
            // The copies are generic-proxy writes.  The fence stands here, behind the barrier: a gathering
            // thread's own fence would wait for every copy it has in flight.
            fence_proxy_async_smem();
            tc_fence_after_sync();
            if (issuer) {
              const uint64_t dp = make_smem_desc_sw128_mn(smem_p + s * Cfg::kPBytes, Cfg::kBlockBytes);
              const uint64_t dq = make_smem_desc_rows_mn(smem_q + s * Cfg::kQBytes, Cfg::kChunk * 2u, kRows * Cfg::kChunk * 2u);
#pragma unroll
              for (int k = 0; k < kRows / 16; ++k) umma_f16<1>(tmem, dp + 128u * k, dq + 2u * Cfg::kChunk * k, idesc, b > b0 || k > 0);
              umma_commit<1>(empty + 8u * s);
              if (b == b1 - 1) umma_commit<1>(done);
            }
            __syncwarp();
          }
        }
        n += static_cast<uint32_t>(b1 - b0);
        ++rounds;
      }
      __syncthreads();
      if (splits > 1) {
        cluster_arrive();
        cluster_wait();
      }
      if (work && splits > 1) {
        // This CTA's share of its tile's sums, four neighbours at a time, added over the parts in rank order.
        const int per_row = (side.rank_outer ? 128 : R) / 4, quads = 32 * R, leader = rank - part;
        const int q0 = quads * part / splits, q1 = quads * (part + 1) / splits;
        uint16_t* out = side.out + static_cast<long>(g) * side.D * R;
        uint32_t live = 0;                                 // (a part without rows has left nothing)
        for (int c = 0; c < splits; ++c) live |= block_of(c) != block_of(c + 1) ? 1u << c : 0u;
        for (int q = q0 + static_cast<int>(threadIdx.x); q < q1; q += Cfg::kThreads) {
          const int y = q / per_row, x = q % per_row * 4;
          const int i = col0 + (side.rank_outer ? x : y);
          if (i >= side.D) continue;
          float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          const uint32_t src = base + static_cast<uint32_t>(y * pitch + x) * 4u;
          float4 t[kGradCluster];
#pragma unroll
          for (int c = 0; c < kGradCluster; ++c) {
            t[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if ((live >> c) & 1u)
              t[c] = ld_cluster_v4(map_to_cta(src, static_cast<uint32_t>(leader + c)));
          }
#pragma unroll
          for (int c = 0; c < kGradCluster; ++c) sum.x += t[c].x, sum.y += t[c].y, sum.z += t[c].z, sum.w += t[c].w;
          const long at = side.rank_outer ? static_cast<long>(y) * side.D + i : static_cast<long>(i) * R + x;
          *reinterpret_cast<uint2*>(out + at) = make_uint2(pack2<kIsBf16>(__float_as_uint(sum.x), __float_as_uint(sum.y)),
                                                           pack2<kIsBf16>(__float_as_uint(sum.z), __float_as_uint(sum.w)));
        }
      }
      // the ring goes back to the copies
      if (splits > 1) {
        cluster_arrive();
        cluster_wait();
      } else {
        __syncthreads();
      }
    }
    batch_start = batch_end;
  }

  if (*abort_flag != 0) {
#pragma unroll 1
    for (int t = 0; t < 200; ++t) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem, Cfg::kTmemCols);
  }
}

}  // namespace gemm_sm100
