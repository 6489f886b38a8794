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
  int* row_adapter;      // [M]: -1 for rows without an adapter
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
  v.row_adapter = reinterpret_cast<int*>(v.slot_mask + tiles * kLoraTileRows * 8);
  v.order = v.row_adapter + lora_plan_round(M);
  v.offsets = v.order + lora_plan_round(M);
  return v;
}

__device__ __forceinline__ int lora_read_id(const void* ids, int ids_are_64, long row, int adapters) {
  const long long id = ids_are_64 ? static_cast<const long long*>(ids)[row] : static_cast<const int*>(ids)[row];
  return id >= 0 && id < adapters ? static_cast<int>(id) : -1;
}

// One launch, 256 threads a block.  Block t < tiles: the slot list of tile t.  Block tiles + g: the rows of
// adapter g in ascending order; their place in `order` is the number of rows of adapters below g,
// which the block counts itself, so that no block waits for another (adapters x M ids read from L2:
// 2 MB for 64 adapters and 8192 rows).
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
    if (row < M) v.row_adapter[row] = id;
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

// ------------------------------------------------------------------------------ simple kernels
template <bool kIsBf16>
__device__ __forceinline__ float lora_to_float(uint16_t bits) {
  if constexpr (kIsBf16) return __uint_as_float(static_cast<uint32_t>(bits) << 16);
  __half h;
  memcpy(&h, &bits, 2);
  return __half2float(h);
}
template <bool kIsBf16>
__device__ __forceinline__ uint16_t lora_from_float(float x) {
  uint16_t bits;
  if constexpr (kIsBf16) {
    const __nv_bfloat16 h = __float2bfloat16_rn(x);
    memcpy(&bits, &h, 2);
  } else {
    const __half h = __float2half_rn(x);
    memcpy(&bits, &h, 2);
  }
  return bits;
}

// out[m, r] = s_g sum_l P[m, l] W_g[r, l], the element (r, l) of W_g at W + g * stride_g + r * stride_r + l * stride_l.
// One warp per (row, r).
template <bool kIsBf16>
__global__ void lora_low_simple_kernel(const uint16_t* P, long ldp, const uint16_t* W, long stride_g, long stride_r,
                                       long stride_l, const float* scales, float scale, uint16_t* out, long ld_out, int M,
                                       int R, int L, void* plan) {
  const LoraPlanView v = lora_plan_view(plan, M);
  const long item = (static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (item >= static_cast<long>(M) * R) return;
  const long m = item / R;
  const int r = static_cast<int>(item % R), lane = threadIdx.x & 31;
  const int g = v.row_adapter[m];
  float sum = 0.0f;
  if (g >= 0) {
    const uint16_t* w = W + g * stride_g + r * stride_r;
    for (int l = lane; l < L; l += 32) sum += lora_to_float<kIsBf16>(P[m * ldp + l]) * lora_to_float<kIsBf16>(w[l * stride_l]);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    sum *= scales ? scale * scales[g] : scale;
  }
  if (lane == 0) out[m * ld_out + r] = lora_from_float<kIsBf16>(sum);
}

// out_g[i, r] = sum over the rows m of adapter g of P[m, i] Q[m, r], stored at out + g * D * R + i * stride_i + r * stride_r.
// One thread per element.
template <bool kIsBf16>
__global__ void lora_grad_simple_kernel(const uint16_t* P, long ldp, const uint16_t* Q, long ldq, uint16_t* out, long stride_i,
                                        long stride_r, int M, int D, int R, void* plan) {
  const LoraPlanView v = lora_plan_view(plan, M);
  const long item = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (item >= static_cast<long>(D) * R) return;
  const int g = blockIdx.y;
  const long i = item % D, r = item / D;
  float sum = 0.0f;
  const int end = v.offsets[g + 1];
  for (int at = v.offsets[g]; at < end; ++at) {
    const long m = v.order[at];
    sum += lora_to_float<kIsBf16>(P[m * ldp + i]) * lora_to_float<kIsBf16>(Q[m * ldq + r]);
  }
  out[static_cast<long>(g) * D * R + i * stride_i + r * stride_r] = lora_from_float<kIsBf16>(sum);
}

}  // namespace gemm_sm100
