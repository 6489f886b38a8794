// Host side of the low-rank adapter entry points (gemm_sm100_lora* in include/gemm_sm100.h): argument
// checks, launches.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <utility>

#include "gemm_host_sm100.cuh"
#include "lora_sm100.cuh"

namespace {

using namespace gemm_sm100;
using namespace gemm_sm100::host;

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// What a 16-bit matrix of `cols` columns has to fulfil; `rows` <= 1 leaves the pitch unused but checked all the same.
int check_matrix(const void* p, long cols, long ld) {
  if (!p) return GEMM_SM100_ERR_NULL_POINTER;
  if (ld < cols) return GEMM_SM100_ERR_BAD_SHAPE;
  if (misaligned(p) || ld % 8 != 0) return GEMM_SM100_ERR_BAD_ALIGNMENT;
  return GEMM_SM100_OK;
}

int check_common(const gemm_sm100_lora_args& a) {
  if (a.M < 0 || a.N <= 0 || a.K <= 0 || a.K % 8 != 0) return GEMM_SM100_ERR_BAD_SHAPE;
  if (a.R < 8 || a.R % 8 != 0 || a.R > GEMM_SM100_LORA_MAX_RANK) return GEMM_SM100_ERR_BAD_SHAPE;
  if (a.adapters < 1 || a.adapters > GEMM_SM100_LORA_MAX_ADAPTERS) return GEMM_SM100_ERR_BAD_SHAPE;
  if (a.dtype != GEMM_SM100_BF16 && a.dtype != GEMM_SM100_FP16) return GEMM_SM100_ERR_UNSUPPORTED_DTYPE;
  return GEMM_SM100_OK;
}

int check_down(const gemm_sm100_lora_args& a) {
  const int rc = check_matrix(a.down, a.K, a.ld_down);
  if (rc != GEMM_SM100_OK) return rc;
  if (a.stride_down < static_cast<long>(a.R - 1) * a.ld_down + a.K && a.adapters > 1) return GEMM_SM100_ERR_BAD_SHAPE;
  return a.stride_down % 8 != 0 ? GEMM_SM100_ERR_BAD_ALIGNMENT : GEMM_SM100_OK;
}

int check_up(const gemm_sm100_lora_args& a) {
  const int rc = check_matrix(a.up, a.R, a.ld_up);
  if (rc != GEMM_SM100_OK) return rc;
  if (a.stride_up < static_cast<long>(a.N - 1) * a.ld_up + a.R && a.adapters > 1) return GEMM_SM100_ERR_BAD_SHAPE;
  return a.stride_up % 8 != 0 ? GEMM_SM100_ERR_BAD_ALIGNMENT : GEMM_SM100_OK;
}

const uint16_t* u16(const void* p) { return static_cast<const uint16_t*>(p); }
uint16_t* u16(void* p) { return static_cast<uint16_t*>(p); }

// Device state and tensor map encoder.
int ready(DeviceState** st, int* cuda_error_out) {
  std::lock_guard<std::mutex> lock(g_mutex);
  const int rc = device_state(st, cuda_error_out);
  return rc != GEMM_SM100_OK ? rc : get_encoder(cuda_error_out);
}


// Tensor map of a 16-bit array of two or three dimensions, innermost first, whose rows of `box[0]` elements
// land in shared memory with the swizzle of that width.  (L2 fetches of 128 bytes: with 256, 64 adapters of rank 16 beside
// 128 x 14336 x 512 took 28.7 us instead of 27.7.)
int encode_rows(CUtensorMap* map, const void* base, int dtype, int rank, const long (&dims)[3], const long (&pitches)[2],
                const int (&box)[3], int* cuda_error_out) {
  const cuuint64_t d[3] = {static_cast<cuuint64_t>(dims[0]), static_cast<cuuint64_t>(dims[1]), static_cast<cuuint64_t>(dims[2])};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(pitches[0]) * 2u, static_cast<cuuint64_t>(pitches[1]) * 2u};
  const cuuint32_t b[3] = {static_cast<cuuint32_t>(box[0]), static_cast<cuuint32_t>(box[1]), static_cast<cuuint32_t>(box[2])};
  const cuuint32_t ones[3] = {1u, 1u, 1u};
  const CUtensorMapSwizzle swizzle = box[0] == 64 ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : (box[0] == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
  const CUtensorMapDataType type =
      dtype == GEMM_SM100_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = g_encode(map, type, static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, strides, b, ones,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? GEMM_SM100_OK : set_cuda_error(cuda_error_out, cudaErrorInvalidValue);
}

// Tile configurations with an adapter kernel: those the planner chooses by itself, and the layouts' four for B as [K, N].
constexpr unsigned kProductConfigs = (1u << 0) | (1u << 1) | (1u << 2) | (1u << 3) | (1u << 7) | (1u << 9) | (1u << 10) |
                                     (1u << 11) | (1u << 12) | (1u << 13) | (1u << 14) | (1u << 15);
constexpr unsigned kProductConfigsKN = 0xfu;
// those whose K can be cut inside a cluster
constexpr bool has_cluster_split(int config) { return config == 0 || config == 2 || config == 11 || config == 12; }

// The product of the rows with the shared weight and, in the same accumulator, with their adapters.
struct AdapterOperands {
  const void* low;
  long ld_low;
  const void* W;          // [adapters, N, R], or [adapters, R, N] with p.b_is_kn
  long ld_w, stride_w;
  int R, adapters;
  const void* plan;
};

template <class Cfg, int kCfgIndex, bool kBIsKN>
auto product_kernel(bool split_k) {
  auto kernel = gemm_lora_kernel<Cfg, false, kBIsKN>;
  if constexpr (has_cluster_split(kCfgIndex)) {
    if (split_k) kernel = gemm_lora_kernel<Cfg, true, kBIsKN>;
  }
  return kernel;
}

// One-time set-up of an instantiation on a device: its shared-memory limit, and how many CTAs of it are co-resident.
template <int kCfgIndex, bool kIsBf16, bool kBIsKN>
int product_limit(bool split_k, DeviceState& st, int* limit, int* cuda_error_out) {
  using Cfg = LoraConfig<ConfigOf<kCfgIndex, kIsBf16>>;
  static int max_ctas[kMaxDevices][2];
  std::lock_guard<std::mutex> lock(g_mutex);
  int& known = max_ctas[st.device][split_k ? 1 : 0];
  if (known == 0) {
    const auto kernel = product_kernel<Cfg, kCfgIndex, kBIsKN>(split_k);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
    if (e != cudaSuccess) return set_cuda_error(cuda_error_out, e);
    int held = 0;
    if (Cfg::kCtaGroup == 1) {
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, Cfg::kThreads, Cfg::kSmemBytes);
      held *= st.sm_count;
    } else {
      cudaLaunchConfig_t qc = {};
      qc.gridDim = dim3(static_cast<unsigned>(st.sm_count - st.sm_count % 2));
      qc.blockDim = dim3(Cfg::kThreads);
      qc.dynamicSmemBytes = Cfg::kSmemBytes;
      cudaLaunchAttribute qa[1];
      qa[0].id = cudaLaunchAttributeClusterDimension;
      qa[0].val.clusterDim.x = 2;
      qa[0].val.clusterDim.y = 1;
      qa[0].val.clusterDim.z = 1;
      qc.attrs = qa;
      qc.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&held, kernel, &qc);
      held *= 2;
    }
    if (e != cudaSuccess) return set_cuda_error(cuda_error_out, e);
    if (held < 1) return set_cuda_error(cuda_error_out, cudaErrorLaunchOutOfResources);
    known = held < st.sm_count ? held : st.sm_count - st.sm_count % Cfg::kCtaGroup;
  }
  *limit = known;
  return GEMM_SM100_OK;
}

template <int kCfgIndex, bool kIsBf16, bool kBIsKN>
int launch_product_config(const Problem& p, const AdapterOperands& o, const Plan& plan, DeviceState& st, cudaStream_t stream,
                          int* cuda_error_out) {
  using Cfg = LoraConfig<ConfigOf<kCfgIndex, kIsBf16>>;
  const auto kernel = product_kernel<Cfg, kCfgIndex, kBIsKN>(plan.split_k);
  int limit = 0;
  int rc = product_limit<kCfgIndex, kIsBf16, kBIsKN>(plan.split_k, st, &limit, cuda_error_out);
  if (rc) return rc;

  TileParams tp = base_tile_params<Cfg>(p, st);
  int b_box = Cfg::kBRows;
  if (plan.tiles_n > 0) {
    tp.n_tiles = plan.tiles_n;
    tp.bal_q = plan.bal_q;
    tp.bal_rem = plan.bal_rem;
    tp.bal_start = plan.bal_start;
    b_box = 64 / Cfg::kCtaGroup;
    tp.b_box_rows = b_box;
  }
  if (p.M < Cfg::kARows) tp.a_box_rows = static_cast<int>(ceil_div(p.M, 8) * 8);
  tp.k_rotate = k_order_for(p, plan.split_k);
  if (plan.split_k) {
    tp.sk_factor = plan.split_factor;
    tp.sk_cluster = 1;
  }
  CUtensorMap map_a, map_b, map_c;
  rc = encode_2d(&map_a, p.A, p.dtype, p.M, p.K, p.lda, tp.a_box_rows, cuda_error_out, Cfg::kKSub);
  if (rc) return rc;
  rc = kBIsKN ? encode_2d(&map_b, p.B, p.dtype, p.K, p.N, p.ldb, 64, cuda_error_out)
              : encode_2d(&map_b, p.B, p.dtype, p.N, p.K, p.ldb, b_box, cuda_error_out, Cfg::kKSub);
  if (rc) return rc;
  rc = encode_2d(&map_c, p.C, p.dtype, p.M, tma_store_cols(p.N), p.ldc, 32, cuda_error_out);
  if (rc) return rc;
  LoraParams lora;
  std::memset(&lora, 0, sizeof(lora));
  lora.R = o.R;
  lora.chunk = rank_chunk(o.R);
  lora.chunks = static_cast<int>(ceil_div(o.R, lora.chunk));
  rc = encode_rows(&lora.tmap_low, o.low, p.dtype, 2, {o.R, p.M, 1}, {o.ld_low, 0}, {lora.chunk, tp.a_box_rows, 1}, cuda_error_out);
  if (rc) return rc;
  rc = kBIsKN ? encode_rows(&lora.tmap_w, o.W, p.dtype, 3, {p.N, o.R, o.adapters}, {o.ld_w, o.stride_w}, {64, lora.chunk, 1},
                            cuda_error_out)
              : encode_rows(&lora.tmap_w, o.W, p.dtype, 3, {o.R, p.N, o.adapters}, {o.ld_w, o.stride_w},
                            {lora.chunk, b_box, 1}, cuda_error_out);
  if (rc) return rc;
  const LoraPlanView view = lora_plan_view(const_cast<void*>(o.plan), p.M);
  lora.slot_count = view.slot_count;
  lora.slot_adapter = view.slot_adapter;
  lora.slot_mask = view.slot_mask;

  long ctas = plan.ctas;
  if (ctas > limit && !plan.split_k) ctas = limit;
  const cudaError_t e = launch_kernel<Cfg>(kernel, ctas, plan.split_k ? plan.split_factor * Cfg::kCtaGroup : Cfg::kCtaGroup,
                                           stream, map_a, map_b, map_c, tp, lora);
  return e == cudaSuccess ? GEMM_SM100_OK : set_cuda_error(cuda_error_out, e);
}

// Forced choices go to the planner.
bool choice_forced() {
  return g_opt_tile_config >= 0 || g_opt_split_k >= 0 || g_opt_sk_cluster >= 0 || g_opt_tiles_n > 0 || g_opt_max_ctas > 0;
}

// ---- low-rank rows: how they are cut
void low_shape(LowParams* p, int M, int R, int L, bool rank_inner) {
  p->M = M, p->R = R, p->L = L;
  p->group_slots = 128 / (rank_inner ? static_cast<int>(ceil_div(R, rank_chunk(R))) * rank_chunk(R) : R);
}

// How a problem is cut.  Two CTAs fit on an SM.  L is cut over as many CTAs of a cluster as leave them all at work at once;
// what is free beyond that takes groups of adapters of the same tile (how many a tile really has is
// known on the device only: a CTA without a group has nothing to do).  The cut is the order in which a row is added up,
// so it depends on the problem alone and not on what shares its launch: a backward pass gives the same bits
// whether the low rows were kept or not, and whichever gradients are wanted.
void cut_low(LowParams* p, int adapters, int sm_count) {
  const int M = p->M;
  const long tiles = ceil_div(M, 128), k_blocks = ceil_div(p->L, 64), room = 2L * sm_count;
  p->splits = 8;
  while (p->splits > 1 && (tiles * p->splits > room || p->splits > k_blocks)) p->splits /= 2;
  const long tile_rows = M < kLoraTileRows ? M : kLoraTileRows;
  const long most_groups = ceil_div(adapters < tile_rows ? adapters : tile_rows, p->group_slots);
  const long groups = room / (tiles * p->splits);
  p->groups = static_cast<int>(groups < 1 ? 1 : (groups > most_groups ? most_groups : groups));
}

// ---- product: which tiles
// Tiles for few rows (at most 128, K a multiple of 64), where the shared planner, which does not know what adapter
// stages cost on a tile, is up to 40 % off.  From forced runs of every configuration (M 2 to 128, N 128 to 16384, K 256 to 28672,
// 4 to 16 adapters of rank 16 and 64), planner's choice against this one:
//  * more than half as many 128-column tiles as SMs, at most one each: those, whole (32 x 10240 x 5120 39.9 against
//    30.7 us, 64 x 12288 x 8192 59.8 / 57.0, 4 x 16384 x 2048 19.6 / 17.7; 64-column tiles would need two waves);
//  * fewer, and K at most twice N or at most 2048: 64-column tiles, whole (1 x 4096 x 4096 18.7 / 14.9, 64 x 4096 x 4096 23.2 /
//    18.4, 16 x 5120 x 8192 34.2 / 28.8, 2 x 512 x 2048 12.5 / 9.3, 64 x 256 x 256 10.6 / 9.3; for 65 to 128 rows there is no such tile);
//  * K longer: tiles cut in four, inside clusters.  The kernel of the low rows (`low_ctas`, two on an SM) still holds SMs when
//    this one starts, and what has no room beside it waits for it.  So 128-column tiles where they fit into seven eighths of
//    the SMs together with it (the rest is left over in the GPCs: 29 tiles with 32 CTAs are 9 % faster by themselves, 30 of them
//    13 to 19 % slower), else 256-column tiles where those do (64 x 3584 x 14336 with 16 adapters of rank 64 45.8 against 38.5 us),
//    else, when either has to wait, up to 33 128-column tiles again (64 x 4096 x 14336 with 64 adapters 65.9 / 59.0).  Of 756 lines
//    (M 16 to 128, N 512 to 4224, K 8704 to 28672, 1 to 64 adapters of rank 16 or 64, by themselves and behind a GEMM) the choice is on
//    average 0.3 % slower than the better of the two.
bool few_row_plan(int M, int N, int K, long low_ctas, int sm_count, Plan* out) {
  if (M > 128 || K % 64 != 0 || choice_forced()) return false;
  const long t64 = ceil_div(N, 64), t128 = ceil_div(N, 128), t256 = ceil_div(N, 256);
  Plan plan;
  if (2 * t128 > sm_count) {
    if (t128 > sm_count) return false;
    plan.config = 12;
    plan.ctas = static_cast<int>(t128);
  } else if (K <= 2L * N || K <= 2048) {
    if (M > 64) return false;
    plan.config = M <= 16 ? 13 : 14;
    plan.ctas = static_cast<int>(t64);
  } else {
    if (t256 > 33) return false;                           // all clusters at once
    auto beside = [&](long tiles) { return 4 * tiles + low_ctas / 2 <= sm_count * 7 / 8; };
    plan.config = beside(t128) || (t128 <= 33 && !beside(t256)) ? 12 : 2;
    plan.split_k = plan.cluster = true;
    plan.split_factor = 4;
    plan.ctas = static_cast<int>((plan.config == 12 ? t128 : t256) * 4);
  }
  *out = plan;
  return true;
}

// Tiles for more than 128 rows whose output still is less than a wave: up to 1024 rows, dA with K up to 8192 up to 1792 (beyond
// 1024 rows in the mean 7 % faster for one adapter, 6 % for runs of four, 2 % slower for 16 in every tile: 1300 x 1536 x 1024 43.2, 37.9, 44.5 ->
// 36.8, 34.4, 45.4; longer contractions 1 % slower in the mean, 12 % faster to 11 % slower).  With more and narrower rows the same
// counts of tiles lost up to 13 %: 9000 x 64 x 512 36.4 -> 41.1, 2048 x 1024 x 1024 30.7 -> 32.4, dA 3000 x 768 x 14336 173 -> 189.  The planner counts on all SMs, but the kernel
// of the low rows still holds some when this one starts: CTAs beyond about 100 (fewer for clusters, which want neighbouring
// SMs) wait for it, and the whole product with them.  About half of the SMs, busy from the start, are then the
// better choice.  Forced runs of every configuration (M 129 to 1024, output columns 512 to 12288, K 512 to 16384), and the choice below
// against the planner's as part of a longer sequence (dA: a training step; forward: behind a 2048 x 2048 x 2048 GEMM of 17 us), in us
// for one adapter of rank 64 / runs of four of rank 32 / 16 of rank 16 in every tile.  M x output columns x K:
//  [K,N] operand (dA):
//  * 64 to 74 CTAs of 256 x 256 pair tiles: those, whole (512 x 4352 x 1024 46.1, 41.7, 49.3 -> 37.5, 33.4, 40.4; 256 x 8704 x 4096
//    74.7, 74.8, 89.1 -> 70.9, 70.1, 80.2); with 64 to 66 the planner's clusters of four all fit and are as good from K = 5120.
//    At K = 4096 twelve of 15 lines are faster whole, three slower (700 x 2688 61.3, 56.6, 73.1 -> 56.7, 52.7, 66.1; 512 x 4096
//    60.7, 56.0, 74.0 -> 63.0, 58.0, 67.6; 1024 x 2048 64.9, 58.9, 69.4 -> 61.2, 55.4, 72.2);
//  * 14 to 16 such tiles, K 4096 up to 8192: cut in two (1024 x 1024 x 4096 58.0, 50.1, 59.7 -> 51.6, 46.9, 58.0; at K = 8192 2 % slower,
//    with 18 to 28 tiles 3 to 8 %);
//  * 7 to 9, more than 256 rows, K from 8192: 128 x 256 tiles cut in four instead of the planner's clusters of eight (1024 x 512 x
//    8192 62.4, 55.9, 85.0 -> 59.2, 53.6, 84.6; 512 x 1024 x 8192 52.6, 48.8, 68.6 -> 52.4, 48.9, 59.9).
//  [N,K] operand (K a multiple of 64 for 128-column tiles):
//  * up to 74 CTAs of 256 x 256 pair tiles, from 64 to 72 CTAs on by the rows, K at most 2048 (1024 from 513 rows on): those,
//    whole (512 x 4352 x 1024 31.5, 30.7, 34.5 -> 29.2, 29.0, 31.9; 1024 x 2048 x 1024 31.1, 30.1, 34.9 -> 29.1, 28.7, 35.9, and with
//    16 adapters at K = 2048 38.4 -> 41.7);
//  * 68 to 74 CTAs of 256 x 128 pair tiles, K from 8192: those, whole (256 x 4608 x 8192 58.0, 58.9, 60.5 -> 51.4, 52.1, 54.8);
//  * 13 to 20 such tiles, K from 4096: cut in two (512 x 1024 x 4096 40.4, 39.6, 42.6 -> 34.6, 34.8, 36.2; 256 x 2048 x 14336 56.3, 57.4,
//    62.5 -> 53.9, 54.2, 56.3);
// (12 such tiles stay with the planner: 128 x 128 tiles cut in four are up to 17 % faster or 7 % slower without a size that
// tells which: 256 x 1536 x 14336 42.8, 43.8, 57.9 -> 45.8, 46.5, 48.3; 512 x 768 x 14336 49.4, 48.8, 58.3 -> 44.6, 44.9, 60.8.)
bool half_wave_plan(int M, int N, int K, bool b_is_kn, int sm_count, Plan* out) {
  if (M <= 128 || M > (b_is_kn && K <= 8192 ? 1792 : 1024) || choice_forced()) return false;
  const long rows = ceil_div(M, 256), wide = rows * ceil_div(N, 256), narrow = rows * ceil_div(N, 128);
  const long half = sm_count / 4;                          // pair tiles on half of the SMs
  int config = -1, factor = 1;
  if (b_is_kn) {
    if (wide <= half && (wide > 33 || (wide >= 32 && K <= 4096))) {
      config = 0;
    } else if (wide >= 14 && wide <= 16 && K >= 4096 && K < 8192) {
      config = 0;
      factor = 2;
    } else if (wide >= 7 && wide <= 9 && M > 256 && K >= 8192) {
      config = 2;
      factor = 4;
    }
  } else if (wide >= 32 + (M <= 512 ? 2 : 0) + (M <= 256 ? 2 : 0) && wide <= half &&
             K <= (M > 512 ? 1024 : 2048)) {
    config = 0;
  } else if (K % 64 == 0) {
    if (narrow >= 34 && narrow <= half && K >= 8192) {
      config = 11;
    } else if (narrow >= 13 && narrow <= 20 && K >= 4096) {
      config = 11;
      factor = 2;
    }
  }
  if (config < 0) return false;
  Plan plan;
  plan.config = config;
  const ConfigInfo& c = kConfigs[config];
  plan.ctas = static_cast<int>(ceil_div(M, 128L * c.cta_group) * ceil_div(N, static_cast<long>(c.mma_n) * c.halves) * factor *
                               c.cta_group);
  if (factor > 1) {
    plan.split_k = plan.cluster = true;
    plan.split_factor = factor;
  }
  *out = plan;
  return true;
}

// What carries out a product, and in `rule` what chose it.
Plan product_plan(int M, int N, int K, bool b_is_kn, int R, int adapters, int sm_count, const char** rule) {
  Plan plan;
  *rule = "few rows";
  if (!b_is_kn) {
    LowParams low;
    low_shape(&low, M, R, K, /*rank_inner=*/false);
    cut_low(&low, adapters, sm_count);
    if (few_row_plan(M, N, K, ceil_div(M, 128) * low.splits * low.groups, sm_count, &plan)) return plan;
  }
  *rule = "less than a wave";
  if (half_wave_plan(M, N, K, b_is_kn, sm_count, &plan)) return plan;
  *rule = "planner";
  return plan_for(M, N, K, sm_count, /*allow_split=*/true, b_is_kn ? kProductConfigsKN : kProductConfigs,
                  /*allow_balance=*/!b_is_kn, /*allow_workspace=*/false);
}

template <bool kIsBf16>
int launch_product(const Problem& p, const AdapterOperands& o, const Plan& plan, cudaStream_t stream, int* cuda_error_out) {
  DeviceState* st = nullptr;
  const int rc = ready(&st, cuda_error_out);
  if (rc != GEMM_SM100_OK) return rc;
  if (p.b_is_kn) {
    switch (plan.config) {
      case 0: return launch_product_config<0, kIsBf16, true>(p, o, plan, *st, stream, cuda_error_out);
      case 1: return launch_product_config<1, kIsBf16, true>(p, o, plan, *st, stream, cuda_error_out);
      case 2: return launch_product_config<2, kIsBf16, true>(p, o, plan, *st, stream, cuda_error_out);
      default: return launch_product_config<3, kIsBf16, true>(p, o, plan, *st, stream, cuda_error_out);
    }
  }
  switch (plan.config) {
    case 0: return launch_product_config<0, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 1: return launch_product_config<1, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 2: return launch_product_config<2, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 3: return launch_product_config<3, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 7: return launch_product_config<7, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 9: return launch_product_config<9, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 10: return launch_product_config<10, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 11: return launch_product_config<11, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 12: return launch_product_config<12, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 13: return launch_product_config<13, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 14: return launch_product_config<14, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    case 15: return launch_product_config<15, kIsBf16, false>(p, o, plan, *st, stream, cuda_error_out);
    default: return GEMM_SM100_ERR_BAD_OPTION;
  }
}

// Launch in clusters of `cluster` CTAs; a programmatic dependent of the kernel before it like the GEMM's kernels.
template <class Kernel, class... Params>
cudaError_t launch_cluster(Kernel kernel, long ctas, int cluster, int threads, int smem_bytes, cudaStream_t stream,
                           const Params&... params) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = g_opt_pdl.load() != 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, params...);
}

// The dynamic shared-memory limit of a kernel, set once per device.
template <class Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, bool (&done)[kMaxDevices], int device) {
  std::lock_guard<std::mutex> lock(g_mutex);
  if (done[device]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done[device] = true;
  return e;
}

template <bool kIsBf16, bool kRankInner, bool kDeep>
cudaError_t allow_low(DeviceState& st) {
  static bool allowed[kMaxDevices];
  return allow_smem(lora_low_kernel<kIsBf16, kRankInner, kDeep>, LowConfig<kDeep>::kSmemBytes, allowed, st.device);
}
template <bool kIsBf16, bool kDeep>
cudaError_t allow_low_pair(DeviceState& st) {
  static bool allowed[kMaxDevices];
  return allow_smem(lora_low_pair_kernel<kIsBf16, kDeep>, LowConfig<kDeep>::kSmemBytes, allowed, st.device);
}

// Parameters of the low-rank rows of P [M, L] through W: down [adapters, R, L], or (rank_inner) up [adapters, L, R].
int low_params(LowParams* out_params, const gemm_sm100_lora_args& a, bool rank_inner, const void* P, long ldp, const void* W,
               long ld_w, long stride_w, int L, void* out, long ld_out, const DeviceState& st, int* cuda_error_out) {
  LowParams& p = *out_params;
  std::memset(&p, 0, sizeof(p));
  p.p_rows = a.M >= 128 ? 128 : static_cast<int>(ceil_div(a.M, 8) * 8);
  int rc = encode_rows(&p.tmap_p, P, a.dtype, 2, {L, a.M, 1}, {ldp, 0}, {64, p.p_rows, 1}, cuda_error_out);
  if (rc) return rc;
  rc = rank_inner ? encode_rows(&p.tmap_w, W, a.dtype, 3, {a.R, L, a.adapters}, {ld_w, stride_w}, {rank_chunk(a.R), 64, 1},
                                cuda_error_out)
                  : encode_rows(&p.tmap_w, W, a.dtype, 3, {L, a.R, a.adapters}, {ld_w, stride_w}, {64, a.R, 1}, cuda_error_out);
  if (rc) return rc;
  p.plan = a.plan;
  p.scales = a.scales;
  p.scale = a.scale;
  p.out = out;
  p.ld_out = ld_out;
  low_shape(&p, a.M, a.R, L, rank_inner);
  p.status = st.status_ptr;
  p.timeout_ns = static_cast<unsigned long long>(g_opt_timeout_ms.load()) * 1000000ull;
  return GEMM_SM100_OK;
}

// CTAs of a launch that `problems` share.  Two that do not fit on the SMs together get half of the CTAs each, with up to two
// partial sums per CTA; whole, in two waves, the backward pass with recomputed low rows takes 138.5 instead of 134.7 us
// (4096 x 4096 x 4096, eight adapters of rank 64) and 94.1 instead of 89.3 (2048 x 4096 x 4096, 16 of rank 32 in every tile).
//
// Deep ring (six stages, one CTA per SM) or short (three, two CTAs): the deep one is faster by itself, but takes twice the SMs,
// and the product kernel `behind` (no CTAs: none) starts on those that are left.  So it is taken where the product would
// have to wait in any case and the launch keeps to half of the SMs: in a sweep of 1224 pairs of times (M 16 to 2048, N and K 1024 to
// 14336, 1 to 64 adapters; forward behind a GEMM and alone, backward with low rows kept and in one launch) 218 pairs, 1 % slower to 11 %
// faster, 2.9 % faster in the mean (64 x 8192 x 14336 with 16 adapters of rank 64 66.7 -> 62.0 us, 1100 x 2048 x 8192 with one 51.7 ->
// 49.7, 128 x 4096 x 8192 with eight 33.9 -> 31.5).  And where a launch of up to 32 CTAs and the product fit beside one another: 332 pairs,
// 2.6 % slower to 3.6 % faster, 0.1 % in the mean (a training step of 114 x 17328 x 2912 with ten of rank 24 102 -> 89 us).  Elsewhere the deep ring costs up to 30 %: 700 x 1024 x 8192 with one adapter 26.1 ->
// 31.8 us, 16 x 8192 x 8192 with eight 33.2 -> 39.7, 64 x 4096 x 14336 with 32 46.6 -> 53.9.  On more than half of
// the SMs it depends on the rows' order, which the host does not know: backward pass of 1024 x 8192 x 1024 with two adapters of rank 128,
// rows in order 51.1 -> 49.1 (half of the CTAs have no adapters), mixed 51.5 -> 56.6.  (Not measured below eight K blocks per CTA.)
struct LowGrid {
  int cluster;           // CTAs of a cluster
  long ctas[2];          // of each problem
  bool deep;
};
// SMs that the product behind wants: its CTAs, one per SM, and an eighth more where clusters of four or more of them have to
// find room in the GPCs.
int wanted_sms(const Plan& plan, int sm_count) {
  const int cluster = plan.split_k ? plan.split_factor * kConfigs[plan.config].cta_group : 1;
  return plan.ctas + (cluster >= 4 ? sm_count / 8 : 0);
}

LowGrid low_grid(LowParams* const* params, int problems, int adapters, const Plan& behind, int sm_count) {
  LowGrid g = {1, {0, 0}, false};
  const long tiles = ceil_div(params[0]->M, 128);
  long wanted = 0;
  for (int i = 0; i < problems; ++i) {
    cut_low(params[i], adapters, sm_count);
    wanted += tiles * params[i]->splits * params[i]->groups;
  }
  const bool fold = problems > 1 && wanted > 2L * sm_count && params[0]->R <= LowConfig<false>::kMaxFoldedRank;
  for (int i = 0; i < problems; ++i) {
    const int ctas = fold && params[i]->groups == 1 ? params[i]->splits / 2 : params[i]->splits;
    if (ctas > g.cluster) g.cluster = ctas;
  }
  bool long_runs = false;
  long total = 0;
  for (int i = 0; i < problems; ++i) {
    LowParams& p = *params[i];
    p.clusters = static_cast<int>(ceil_div(static_cast<long>(p.groups) * p.splits, (fold ? 2L : 1L) * g.cluster));
    g.ctas[i] = tiles * p.clusters * g.cluster;
    total += g.ctas[i];
    if (ceil_div(p.L, 64) >= 8L * g.cluster) long_runs = true;
  }
  const bool no_room = 2 * total <= sm_count && total + 2L * wanted_sms(behind, sm_count) > 2L * sm_count;
  const bool room_for_both = total <= 32 && total + wanted_sms(behind, sm_count) <= sm_count;
  g.deep = long_runs && (no_room || room_for_both);
  const long forced = g_opt_lora_ring.load();
  if (forced >= 0) g.deep = forced != 0;
  return g;
}

template <bool kIsBf16, bool kRankInner>
int launch_low(const gemm_sm100_lora_args& a, const void* P, long ldp, const void* W, long ld_w, long stride_w, int L, void* out,
               long ld_out, const Plan& behind, cudaStream_t stream, int* cuda_error_out) {
  DeviceState* st = nullptr;
  int rc = ready(&st, cuda_error_out);
  if (rc != GEMM_SM100_OK) return rc;
  LowParams p;
  rc = low_params(&p, a, kRankInner, P, ldp, W, ld_w, stride_w, L, out, ld_out, *st, cuda_error_out);
  if (rc != GEMM_SM100_OK) return rc;
  LowParams* const one[1] = {&p};
  const LowGrid g = low_grid(one, 1, a.adapters, behind, st->sm_count);
  const long ctas = g.ctas[0];
  cudaError_t e = g.deep ? allow_low<kIsBf16, kRankInner, true>(*st) : allow_low<kIsBf16, kRankInner, false>(*st);
  if (e == cudaSuccess)
    e = g.deep ? launch_cluster(lora_low_kernel<kIsBf16, kRankInner, true>, ctas, g.cluster, LowConfig<true>::kThreads,
                                LowConfig<true>::kSmemBytes, stream, p)
               : launch_cluster(lora_low_kernel<kIsBf16, kRankInner, false>, ctas, g.cluster, LowConfig<false>::kThreads,
                                LowConfig<false>::kSmemBytes, stream, p);
  return e == cudaSuccess ? GEMM_SM100_OK : set_cuda_error(cuda_error_out, e);
}

// low (from A and down) and d_low (from dC and up) in one launch.
template <bool kIsBf16>
int launch_low_pair(const gemm_sm100_lora_args& a, void* low, long ld_low, const void* dC, long ld_dc, void* d_low, long ld_d_low,
                    const Plan& behind, cudaStream_t stream, int* cuda_error_out) {
  DeviceState* st = nullptr;
  int rc = ready(&st, cuda_error_out);
  if (rc != GEMM_SM100_OK) return rc;
  LowParams p, q;
  rc = low_params(&p, a, false, a.A, a.lda, a.down, a.ld_down, a.stride_down, a.K, low, ld_low, *st, cuda_error_out);
  if (rc == GEMM_SM100_OK)
    rc = low_params(&q, a, true, dC, ld_dc, a.up, a.ld_up, a.stride_up, a.N, d_low, ld_d_low, *st, cuda_error_out);
  if (rc != GEMM_SM100_OK) return rc;
  LowParams* const both[2] = {&p, &q};
  const LowGrid g = low_grid(both, 2, a.adapters, behind, st->sm_count);
  const int first = static_cast<int>(g.ctas[0]);
  const long ctas = g.ctas[0] + g.ctas[1];
  cudaError_t e = g.deep ? allow_low_pair<kIsBf16, true>(*st) : allow_low_pair<kIsBf16, false>(*st);
  if (e == cudaSuccess)
    e = g.deep ? launch_cluster(lora_low_pair_kernel<kIsBf16, true>, ctas, g.cluster, LowConfig<true>::kThreads,
                                LowConfig<true>::kSmemBytes, stream, p, q, first)
               : launch_cluster(lora_low_pair_kernel<kIsBf16, false>, ctas, g.cluster, LowConfig<false>::kThreads,
                                LowConfig<false>::kSmemBytes, stream, p, q, first);
  return e == cudaSuccess ? GEMM_SM100_OK : set_cuda_error(cuda_error_out, e);
}

template <bool kIsBf16, int kRanks>
cudaError_t allow_grad(DeviceState& st) {
  static bool allowed[kMaxDevices];
  return allow_smem(lora_grad_kernel<kIsBf16, kRanks>, GradConfig<kRanks>::kSmemBytes, allowed, st.device);
}

// Both adapters' gradients in one launch.
template <bool kIsBf16, int kRanks>
int launch_grad(const gemm_sm100_lora_args& a, const GradSide& down, const GradSide& up, cudaStream_t stream,
                int* cuda_error_out) {
  using Cfg = GradConfig<kRanks>;
  DeviceState* st = nullptr;
  const int rc = ready(&st, cuda_error_out);
  if (rc != GEMM_SM100_OK) return rc;
  auto kernel = lora_grad_kernel<kIsBf16, kRanks>;
  cudaError_t e = allow_grad<kIsBf16, kRanks>(*st);
  if (e != cudaSuccess) return set_cuda_error(cuda_error_out, e);
  GradParams p;
  std::memset(&p, 0, sizeof(p));
  p.side[0] = down;
  p.side[1] = up;
  p.plan = a.plan;
  p.M = a.M, p.R = a.R, p.adapters = a.adapters;
  p.tiles0 = static_cast<int>(ceil_div(down.D, 128));
  p.tiles = p.tiles0 + static_cast<int>(ceil_div(up.D, 128));
  p.status = st->status_ptr;
  p.timeout_ns = static_cast<unsigned long long>(g_opt_timeout_ms.load()) * 1000000ull;
  // How far to cut the rows: the rows may all belong to one adapter, so the cut that finishes that case first
  // sets the number of rows a CTA takes at once; adapters with fewer rows are cut less.
  // (Nine tenths of the CTAs that the SMs hold: a cluster sits inside one GPC, and what is left over there must not make
  // a second wave.)  The cut is the order in which a gradient is added up: it is chosen for both gradients' tiles, also
  // where only one of them is wanted, so that this one has the same bits then.
  const long clusters = static_cast<long>(st->sm_count) * Cfg::kCtasPerSm * 9 / (10 * kGradCluster);
  const long both = ceil_div(a.K, 128) + ceil_div(a.N, 128);
  int splits = 1;
  double best = 1e300;
  for (int c = 1; c <= kGradCluster; c *= 2) {
    const double t = static_cast<double>(ceil_div(ceil_div(both, kGradCluster / c), clusters)) *
                     (static_cast<double>(ceil_div(a.M, c)) + 128.0);      // (a unit costs about two blocks of rows besides)
    if (t < best) best = t, splits = c;
  }
  p.split_rows = static_cast<int>(ceil_div(a.M, splits));
  if (p.split_rows < 128) p.split_rows = 128;
  // as many units as there can be (those of adapters without rows write zeros instead)
  const long units = ceil_div(static_cast<long>(p.tiles) * splits, kGradCluster) * a.adapters;
  e = launch_cluster(kernel, (units < clusters ? units : clusters) * kGradCluster, kGradCluster, Cfg::kThreads, Cfg::kSmemBytes,
                     stream, p);
  return e == cudaSuccess ? GEMM_SM100_OK : set_cuda_error(cuda_error_out, e);
}

template <int kCfgIndex, bool kIsBf16>
int prepare_config(DeviceState& st, int* cuda_error_out) {
  int limit = 0, rc = GEMM_SM100_OK;
  for (int split = 0; split < (has_cluster_split(kCfgIndex) ? 2 : 1) && rc == GEMM_SM100_OK; ++split) {
    if constexpr (((kProductConfigs >> kCfgIndex) & 1u) != 0)
      rc = product_limit<kCfgIndex, kIsBf16, false>(split != 0, st, &limit, cuda_error_out);
    if constexpr (((kProductConfigsKN >> kCfgIndex) & 1u) != 0)
      if (rc == GEMM_SM100_OK) rc = product_limit<kCfgIndex, kIsBf16, true>(split != 0, st, &limit, cuda_error_out);
  }
  return rc;
}

template <bool kIsBf16, int... kIndices>
int prepare_type(DeviceState& st, int* cuda_error_out, std::integer_sequence<int, kIndices...>) {
  int rc = GEMM_SM100_OK;
  (void)((rc = prepare_config<kIndices, kIsBf16>(st, cuda_error_out), rc == GEMM_SM100_OK) && ...);
  if (rc != GEMM_SM100_OK) return rc;
  cudaError_t e = allow_low<kIsBf16, false, false>(st);
  if (e == cudaSuccess) e = allow_low<kIsBf16, false, true>(st);
  if (e == cudaSuccess) e = allow_low<kIsBf16, true, false>(st);
  if (e == cudaSuccess) e = allow_low<kIsBf16, true, true>(st);
  if (e == cudaSuccess) e = allow_low_pair<kIsBf16, false>(st);
  if (e == cudaSuccess) e = allow_low_pair<kIsBf16, true>(st);
  if (e == cudaSuccess) e = allow_grad<kIsBf16, 16>(st);
  if (e == cudaSuccess) e = allow_grad<kIsBf16, 32>(st);
  if (e == cudaSuccess) e = allow_grad<kIsBf16, 64>(st);
  if (e == cudaSuccess) e = allow_grad<kIsBf16, 128>(st);
  return e == cudaSuccess ? GEMM_SM100_OK : set_cuda_error(cuda_error_out, e);
}

// The low-rank rows of A; the caller has checked what all calls share.
int low_rows(const gemm_sm100_lora_args& a, void* low, long ld_low, const Plan& behind, cudaStream_t stream, int* cuda_error_out) {
  if (!a.plan) return GEMM_SM100_ERR_NULL_POINTER;
  int rc = check_matrix(a.A, a.K, a.lda);
  if (rc || (rc = check_down(a)) || (rc = check_matrix(low, a.R, ld_low))) return rc;
  return (a.dtype == GEMM_SM100_BF16 ? launch_low<true, false> : launch_low<false, false>)(
      a, a.A, a.lda, a.down, a.ld_down, a.stride_down, a.K, low, ld_low, behind, stream, cuda_error_out);
}

}  // namespace

namespace gemm_sm100 {
namespace host {

int lora_prepare(DeviceState& st, int* cuda_error_out) {
  cudaFuncAttributes attributes;
  const cudaError_t e = cudaFuncGetAttributes(&attributes, lora_plan_kernel);   // loads it
  if (e != cudaSuccess) return set_cuda_error(cuda_error_out, e);
  const int rc = prepare_type<true>(st, cuda_error_out, std::make_integer_sequence<int, kNumConfigs>{});
  return rc ? rc : prepare_type<false>(st, cuda_error_out, std::make_integer_sequence<int, kNumConfigs>{});
}

}  // namespace host
}  // namespace gemm_sm100

extern "C" {

size_t gemm_sm100_lora_plan_bytes(int M, int adapters) {
  if (M < 0 || adapters < 1 || adapters > GEMM_SM100_LORA_MAX_ADAPTERS) return 0;
  return static_cast<size_t>(lora_plan_words(M, adapters)) * sizeof(int);
}

int gemm_sm100_lora_plan(const void* ids, int ids_are_64, int M, int adapters, void* plan, size_t plan_bytes,
                         void* cuda_stream, int* cuda_error_out) {
  if (cuda_error_out) *cuda_error_out = 0;
  if (M < 0 || adapters < 1 || adapters > GEMM_SM100_LORA_MAX_ADAPTERS) return GEMM_SM100_ERR_BAD_SHAPE;
  if (!plan || (M > 0 && !ids)) return GEMM_SM100_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(ids) & (ids_are_64 ? 7u : 3u)) != 0) return GEMM_SM100_ERR_BAD_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(plan) & 255u) || plan_bytes < gemm_sm100_lora_plan_bytes(M, adapters))
    return GEMM_SM100_ERR_WORKSPACE;
  const unsigned blocks = static_cast<unsigned>(lora_plan_tiles(M) + adapters);
  lora_plan_kernel<<<blocks, 256, 0, static_cast<cudaStream_t>(cuda_stream)>>>(ids, ids_are_64, M, adapters, plan);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GEMM_SM100_OK : set_cuda_error(cuda_error_out, e);
}

int gemm_sm100_lora_describe_plan(int M, int N, int K, int R, int adapters, int gradient, char* buf, size_t buf_bytes) {
  if (!buf || buf_bytes == 0) return GEMM_SM100_ERR_NULL_POINTER;
  gemm_sm100_lora_args a = {};
  a.M = M, a.N = N, a.K = K, a.R = R, a.adapters = adapters;
  const int rc = check_common(a);
  if (rc != GEMM_SM100_OK || M == 0 || (gradient && N % 8 != 0)) return rc != GEMM_SM100_OK ? rc : GEMM_SM100_ERR_BAD_SHAPE;
  const char* rule;
  // (dA is an [M, K] output with N contracted)
  const Plan plan = product_plan(M, gradient ? K : N, gradient ? N : K, gradient != 0, R, adapters, current_sm_count(), &rule);
  const int n = std::snprintf(buf, buf_bytes, "%s: ", rule);
  if (n <= 0 || static_cast<size_t>(n) >= buf_bytes) return GEMM_SM100_OK;
  describe(plan, gradient ? K : N, buf + n, buf_bytes - n);
  LowParams low;
  std::memset(&low, 0, sizeof(low));
  low_shape(&low, M, R, gradient ? N : K, gradient != 0);
  LowParams* const one[1] = {&low};
  const LowGrid grid = low_grid(one, 1, adapters, plan, current_sm_count());
  const size_t used = std::strlen(buf);
  std::snprintf(buf + used, buf_bytes - used, "; low rows: %ld ctas in clusters of %d, %s ring", grid.ctas[0], grid.cluster,
                grid.deep ? "deep" : "short");
  return GEMM_SM100_OK;
}

int gemm_sm100_lora_low(const gemm_sm100_lora_args* args, void* low, long ld_low, void* cuda_stream, int* cuda_error_out) {
  if (cuda_error_out) *cuda_error_out = 0;
  if (!args) return GEMM_SM100_ERR_NULL_POINTER;
  const int rc = check_common(*args);
  if (rc != GEMM_SM100_OK || args->M == 0) return rc;
  return low_rows(*args, low, ld_low, /*behind=*/Plan{}, static_cast<cudaStream_t>(cuda_stream), cuda_error_out);
}

int gemm_sm100_lora(const gemm_sm100_lora_args* args, void* C, long ldc, void* low, long ld_low, void* cuda_stream,
                    int* cuda_error_out) {
  if (cuda_error_out) *cuda_error_out = 0;
  if (!args) return GEMM_SM100_ERR_NULL_POINTER;
  const gemm_sm100_lora_args& a = *args;
  int rc = check_common(a);
  if (rc != GEMM_SM100_OK) return rc;
  if (a.M == 0) return GEMM_SM100_OK;
  if ((rc = check_matrix(a.B, a.K, a.ldb)) || (rc = check_up(a)) || (rc = check_matrix(C, a.N, ldc))) return rc;
  const char* rule;
  const Plan plan = product_plan(a.M, a.N, a.K, /*b_is_kn=*/false, a.R, a.adapters, current_sm_count(), &rule);
  rc = low_rows(a, low, ld_low, plan, static_cast<cudaStream_t>(cuda_stream), cuda_error_out);
  if (rc != GEMM_SM100_OK) return rc;
  const Problem p{a.A, a.B, C, a.M, a.N, a.K, a.lda, a.ldb, ldc, a.dtype};
  const AdapterOperands o{low, ld_low, a.up, a.ld_up, a.stride_up, a.R, a.adapters, a.plan};
  return (a.dtype == GEMM_SM100_BF16 ? launch_product<true> : launch_product<false>)(
      p, o, plan, static_cast<cudaStream_t>(cuda_stream), cuda_error_out);
}

int gemm_sm100_lora_backward(const gemm_sm100_lora_args* args, const void* dC, long ld_dc, void* low, long ld_low,
                             int recompute_low, void* d_low, long ld_d_low, void* dA, long ld_da, void* d_down, void* d_up, void* cuda_stream,
                             int* cuda_error_out) {
  if (cuda_error_out) *cuda_error_out = 0;
  if (!args) return GEMM_SM100_ERR_NULL_POINTER;
  const gemm_sm100_lora_args& a = *args;
  int rc = check_common(a);
  if (rc != GEMM_SM100_OK) return rc;
  if (a.N % 8 != 0) return GEMM_SM100_ERR_BAD_SHAPE;
  if (!dA && !d_down && !d_up) return GEMM_SM100_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  cudaError_t e = cudaSuccess;
  if (misaligned(d_down) || misaligned(d_up)) return GEMM_SM100_ERR_BAD_ALIGNMENT;
  if (a.M == 0) {
    const size_t bytes = static_cast<size_t>(a.adapters) * a.R * 2;
    if (d_down) e = cudaMemsetAsync(d_down, 0, bytes * a.K, stream);
    if (e == cudaSuccess && d_up) e = cudaMemsetAsync(d_up, 0, bytes * a.N, stream);
    return e == cudaSuccess ? GEMM_SM100_OK : set_cuda_error(cuda_error_out, e);
  }
  if (!a.plan) return GEMM_SM100_ERR_NULL_POINTER;
  if ((rc = check_matrix(dC, a.N, ld_dc))) return rc;
  if (d_down && (rc = check_matrix(a.A, a.K, a.lda))) return rc;
  if (d_up && (rc = check_matrix(low, a.R, ld_low))) return rc;
  if (dA && ((rc = check_matrix(a.B, a.K, a.ldb)) || (rc = check_down(a)) || (rc = check_matrix(dA, a.K, ld_da)))) return rc;
  const bool bf16 = a.dtype == GEMM_SM100_BF16;
  const bool again = recompute_low != 0 && d_up != nullptr;
  if (again && ((rc = check_matrix(a.A, a.K, a.lda)) || (rc = check_down(a)))) return rc;
  Plan plan;
  if (dA) {
    const char* rule;
    plan = product_plan(a.M, a.K, a.N, /*b_is_kn=*/true, a.R, a.adapters, current_sm_count(), &rule);
  }
  if (dA || d_down) {
    if ((rc = check_up(a)) || (rc = check_matrix(d_low, a.R, ld_d_low))) return rc;
    if (again)
      rc = (bf16 ? launch_low_pair<true> : launch_low_pair<false>)(a, low, ld_low, dC, ld_dc, d_low, ld_d_low, plan, stream,
                                                                       cuda_error_out);
    else
      rc = (bf16 ? launch_low<true, true> : launch_low<false, true>)(a, dC, ld_dc, a.up, a.ld_up, a.stride_up, a.N, d_low,
                                                                     ld_d_low, plan, stream, cuda_error_out);
  } else if (again) {
    rc = low_rows(a, low, ld_low, /*behind=*/plan, stream, cuda_error_out);
  }
  if (rc != GEMM_SM100_OK) return rc;
  if (dA) {
    const Problem p{dC, a.B, dA, a.M, a.K, a.N, ld_dc, a.ldb, ld_da, a.dtype, /*b_is_kn=*/true};
    const AdapterOperands o{d_low, ld_d_low, a.down, a.ld_down, a.stride_down, a.R, a.adapters, a.plan};
    rc = (bf16 ? launch_product<true> : launch_product<false>)(p, o, plan, stream, cuda_error_out);
    if (rc != GEMM_SM100_OK) return rc;
  }
  if (!d_down && !d_up) return GEMM_SM100_OK;
  const GradSide down{u16(a.A), u16(d_low), u16(d_down), a.lda, ld_d_low, d_down ? a.K : 0, 1};
  const GradSide up{u16(dC), u16(low), u16(d_up), ld_dc, ld_low, d_up ? a.N : 0, 0};
  if (a.R <= 16) return (bf16 ? launch_grad<true, 16> : launch_grad<false, 16>)(a, down, up, stream, cuda_error_out);
  if (a.R <= 32) return (bf16 ? launch_grad<true, 32> : launch_grad<false, 32>)(a, down, up, stream, cuda_error_out);
  if (a.R <= 64) return (bf16 ? launch_grad<true, 64> : launch_grad<false, 64>)(a, down, up, stream, cuda_error_out);
  return (bf16 ? launch_grad<true, 128> : launch_grad<false, 128>)(a, down, up, stream, cuda_error_out);
}

}  // extern "C"
