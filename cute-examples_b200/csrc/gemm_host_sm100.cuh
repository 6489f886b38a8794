// What the host launchers share: the table of tile configurations, process-wide options, the tensor
// map encoder, the plan of a launch, and the launch itself.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstring>
#include <mutex>

#include "../../include/gemm_sm100.h"
#include "gemm_tn_sm100.cuh"

namespace gemm_sm100 {
namespace host {

constexpr int kMaxDevices = 64;
constexpr int kNumConfigs = 16;

struct ConfigInfo {
  int cta_group, mma_n, halves, stages, epi_warps;
  int a_rows = 128;    // rows of A loaded per stage: the configuration only takes problems of at most that many rows
  int epi_bufs = 0;    // staging buffers per epilogue warp (0: 8 / epi_warps)
  int k_sub = 1;       // 64-element K blocks per stage (2: one 3-D TMA box per operand tile and stage)
};
constexpr ConfigInfo kConfigs[kNumConfigs] = {
    {2, 256, 1, 6, 4},   // 256 x 256 pair tile, alternating accumulator slots
    {2, 256, 2, 4, 8},   // 256 x 512 pair tile, both slots, 8 epilogue warps
    {1, 256, 1, 4, 4},   // 128 x 256 single-CTA tile
    {1, 128, 1, 4, 4},   // 128 x 128 single-CTA tile
    {2, 256, 2, 4, 4},
    {2, 256, 1, 6, 8},
    {1, 256, 1, 4, 8},
    // 256 x 128 pair tile: fewest operand bytes per SM among the small tiles.  Five stages: with
    // operand boxes this small the ring delivers FEWER bytes per clock the more loads it keeps in
    // flight (trace counters with the MMAs switched off, 8192 x 4096 x 4096: 0.48 of the MMA rate
    // with 4 stages, 0.47 with 5, 0.44 with 6, 0.35 with 8), and few-tile problems ran 13-20 % faster
    // with 5 stages than with 8.
    {2, 128, 1, 5, 4},
    {2, 192, 1, 6, 4},   // 256 x 192 pair tile: for tile counts that quantise badly with 256 columns
    // 128 x 256 tiles for problems of at most 16 / 64 rows: only those rows of A are loaded, and the
    // shared memory saved holds more stages (6 / 5 x 32 KiB of B in flight per SM instead of 4)
    {1, 256, 1, 6, 4, 16, 1},
    {1, 256, 1, 5, 4, 64, 1},
    // 256 x 128 pair tile with two K blocks per stage (K % 64 == 0 only): half as many, twice as
    // large TMA boxes as configuration 7
    {2, 128, 1, 4, 4, 128, 0, 2},
    // 128 x 128 single-CTA tile with two K blocks per stage, for problems of at most 128 rows whose
    // columns give too few 256-wide tiles: twice the tiles of configuration 2, half-size partial tiles
    {1, 128, 1, 3, 4, 128, 0, 2},
    // 128 x 64 tiles for problems of at most 16 / 64 rows and several thousand columns: four K blocks
    // (512 bytes of every row) per TMA box, short A
    {1, 64, 1, 5, 4, 16, 1, 4},
    {1, 64, 1, 3, 4, 64, 1, 4},
    // configuration 9 with two K blocks per box (K % 64 == 0): 16 x 28672 x 8192 74.5 against 75.6 us
    {1, 256, 1, 3, 4, 16, 1, 2},
};

template <int kIndex, bool kIsBf16>
using ConfigOf = GemmConfig<kConfigs[kIndex].cta_group, kConfigs[kIndex].mma_n, kConfigs[kIndex].halves,
                            kConfigs[kIndex].stages, kConfigs[kIndex].epi_warps, kIsBf16, kConfigs[kIndex].a_rows,
                            kConfigs[kIndex].epi_bufs, kConfigs[kIndex].k_sub>;

struct DeviceState {
  bool ready = false;
  int device = 0;
  int sm_count = 0;
  int cc_major = 0;
  unsigned int* status_ptr = nullptr;
  void* static_scratch = nullptr;      // device address of g_static_scratch on this device
  int max_ctas[kNumConfigs][2] = {};   // persistent grid limit per config and dtype
  bool attr_set[kNumConfigs][2] = {};
};

inline std::mutex g_mutex;
inline DeviceState g_dev[kMaxDevices];
// Process-wide knobs.  Written by gemm_sm100_set_option / gemm_sm100_set_trace_buffer, read by
// launches on any thread: atomics, so a concurrent change is seen whole or not at all.
inline std::atomic<long> g_opt_tile_config{-1};
inline std::atomic<long> g_opt_timeout_ms{2000};
inline std::atomic<long> g_opt_max_ctas{0};
inline std::atomic<long> g_opt_debug_flags{0};
inline std::atomic<long> g_opt_group_m{0};
inline std::atomic<long> g_opt_k_rotate{-1};   // 0 never, 1 always, -1 (default) when there is a single tile row: 3 % on the few-row shapes, 2 = serpentine
inline std::atomic<long> g_opt_sk_cluster{-1};  // cluster K-split (partial sums through distributed shared memory): -1 planner, 0 never, 1 always where an even split of 2 or 4 is made
inline std::atomic<long> g_opt_lora_ring{-1};   // ring of the kernel of the low-rank rows: -1 by the launch, 0 short, 1 deep
inline std::atomic<long> g_opt_pdl{1};        // 1: launch with programmatic stream serialization (overlap with the previous kernel's tail)
inline std::atomic<long> g_opt_early_prefetch{1};   // with pdl: L2 prefetch of the first stages before waiting for the previous kernel
inline std::atomic<long> g_opt_tiles_n{0};    // > 0: force this many tiles per tile row (tests), when the configuration allows the widths
inline std::atomic<long> g_opt_balance{1};    // 1: the planner may choose a balanced column tiling; 0: uniform tiles only
inline std::atomic<long> g_opt_split_k{-1};   // -1 automatic, 0 never, 1 whenever the configuration allows it
// Clusters of 2, 4 and 8 CTAs (one CTA per SM) the device holds at once, from the occupancy query.
inline std::atomic<int> g_held_clusters[3] = {};
// Bumped by every gemm_sm100_set_option: cached plans of an older generation are stale.
inline std::atomic<unsigned> g_opt_generation{1};

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn g_encode = nullptr;

inline int set_cuda_error(int* out, cudaError_t e) {
  if (out) *out = static_cast<int>(e);
  return GEMM_SM100_ERR_CUDA;
}

// Looks the driver's tensor-map encoder up once (no link-time dependency on libcuda).
inline int get_encoder(int* cuda_error_out) {
  if (g_encode) return GEMM_SM100_OK;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult qres;
  cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
  if (e != cudaSuccess) return set_cuda_error(cuda_error_out, e);
  if (qres != cudaDriverEntryPointSuccess || fn == nullptr)
    return set_cuda_error(cuda_error_out, cudaErrorSymbolNotFound);
  g_encode = reinterpret_cast<EncodeTiledFn>(fn);
  return GEMM_SM100_OK;
}

// Columns of C the TMA stores cover: whole 16-byte pieces only (the kernel writes the last N % 8
// columns with plain stores); never 0, which is not a valid extent (the map is unused then).
inline long tma_store_cols(long n) { return n >= 8 ? (n & ~7L) : 8; }

// Tensor map of a row-major 2-D array of 16-bit elements: `rows` x `cols`, pitch `ld`
// elements, box `box_rows` x 64 columns, 128-byte swizzle (64 x 2 B = one swizzle row).
// With k_sub > 1 (cols a multiple of 64) the same array is described as 3-D: 64 elements x rows x
// 64-element K blocks (128 bytes apart), box 64 x box_rows x k_sub, so that one copy brings k_sub K
// blocks of the rows, each as its own K-major tile.
inline int encode_2d(CUtensorMap* map, const void* base, int dtype, long rows, long cols, long ld,
              int box_rows, int* cuda_error_out, int k_sub = 1) {
  const bool blocks = k_sub > 1;
  const cuuint64_t dims[3] = {blocks ? 64u : static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(cols / 64)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * 2u, 128u};
  const cuuint32_t box[3] = {64u, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(k_sub)};
  const cuuint32_t elem_strides[3] = {1u, 1u, 1u};
  const CUtensorMapDataType dt =
      dtype == GEMM_SM100_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = g_encode(map, dt, blocks ? 3 : 2, const_cast<void*>(base), dims, strides, box, elem_strides,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_cuda_error(cuda_error_out, cudaErrorInvalidValue);
  return GEMM_SM100_OK;
}

// State of the current device, made on first use; the caller holds g_mutex.
int device_state(DeviceState** out, int* cuda_error_out);

struct Problem {
  const void* A;
  const void* B;
  void* C;
  int M, N, K;
  long lda, ldb, ldc;
  int dtype;
  bool b_is_kn = false;   // B given as [K, N] (pitch ldb >= N) instead of [N, K]
  bool a_is_km = false;   // A given as [K, M] (pitch lda >= M) instead of [M, K]
  float alpha = 1.0f;     // C = alpha * op(A) op(B) + beta * C (only the layout kernels apply them)
  float beta = 0.0f;
};

inline long ceil_div(long a, long b) { return (a + b - 1) / b; }

struct Plan {
  int config = 0;
  // Column tiling (TileParams::bal_q / bal_rem): tiles_n tiles per tile row; 0 = uniform tiles.
  int tiles_n = 0, bal_q = 0, bal_rem = 0, bal_start = 0;
  bool split_k = false;
  int ctas = 0;              // grid size
  size_t flag_bytes = 0;     // K-split: arrival counters (one per CTA), padded to 256 bytes
  size_t partial_bytes = 0;  // K-split: one fp32 partial tile per CTA
  int partial_rows = 128;    // K-split: rows kept per partial tile
  int split_factor = 0;      // K-split: > 1 = every tile cut into this many equal K ranges
  bool cluster = false;      // even split whose contributors form a cluster and exchange partial sums in shared memory
};

// One-time set-up of every adapter kernel on the device (part of gemm_sm100_init).
int lora_prepare(DeviceState& st, int* cuda_error_out);

// The plan of a problem under the current options, cached per thread.  `allow_workspace` false: no K-split
// that needs a workspace; `config_mask`: the configurations the caller has kernels for.
Plan plan_for(int M, int N, int K, int sm_count, bool allow_split = true, unsigned config_mask = ~0u,
              bool allow_balance = true, bool allow_workspace = true);

// A plan for an output of N columns in words.
void describe(const Plan& plan, int N, char* buf, size_t buf_bytes);

// SMs of the current device (those of a B200 where there is none).
int current_sm_count();

inline int grid_cap(const ConfigInfo& c, int sm_count) {
  long cap = sm_count - sm_count % c.cta_group;
  if (g_opt_max_ctas > 0 && g_opt_max_ctas < cap) cap = g_opt_max_ctas - g_opt_max_ctas % c.cta_group;
  if (cap < c.cta_group) cap = c.cta_group;
  return static_cast<int>(cap);
}

inline int default_group_m(int m_tiles) {
  return g_opt_group_m.load() > 0 ? static_cast<int>(g_opt_group_m.load()) : (m_tiles >= 16 ? 16 : 8);
}

// Tile counts, rasterisation and wait limit of one launch (everything that does not depend on
// the schedule variant).
template <class Cfg>
TileParams base_tile_params(const Problem& p, const DeviceState& st) {
  TileParams tp;
  tp.M = p.M;
  tp.N = p.N;
  tp.K = p.K;
  tp.m_tiles = static_cast<int>(ceil_div(p.M, 128L * Cfg::kCtaGroup));
  tp.n_tiles = static_cast<int>(ceil_div(p.N, Cfg::kBlockN));
  tp.k_blocks = static_cast<int>(ceil_div(p.K, Cfg::kBlockK));
  // Rasterisation group: 16 tile rows when the problem has that many (measured best from 8192
  // to 32768 rows: the A panel of a group is reused by more B tiles), else 8.
  tp.group_m = default_group_m(tp.m_tiles);
  tp.bal_q = Cfg::kBlockN / 64;
  tp.bal_rem = 0;
  tp.bal_start = 0;
  tp.b_box_rows = Cfg::kBRows;
  tp.a_box_rows = Cfg::kARows;
  tp.early_prefetch = (g_opt_pdl.load() != 0 && g_opt_early_prefetch.load() != 0) ? 1 : 0;
  tp.status = st.status_ptr;
  tp.timeout_ns = static_cast<unsigned long long>(g_opt_timeout_ms.load()) * 1000000ull;
  tp.trace = nullptr;
  tp.debug_flags = 0;
  tp.sk_flags = nullptr;
  tp.sk_partials = nullptr;
  tp.sk_rows = 128;
  tp.sk_factor = 0;
  tp.sk_cluster = 0;
  tp.k_rotate = 0;
  tp.alpha = p.alpha;
  tp.beta = p.beta;
  tp.c_ptr = p.C;
  tp.ldc = p.ldc;
  return tp;
}

// Order of a tile's K blocks (TileParams::k_rotate) for this problem under the "k_rotate" option.
// Automatic (-1): rotation only in the memory-bound few-row regime (at most 128 rows, thousands of
// columns).  Other problems keep K ascending, so that the same rows give the same bits whether
// they are computed in one call or in row panels, and in every operand layout.
inline int k_order_for(const Problem& p, bool split_k) {
  const long k_order = g_opt_k_rotate.load();
  const bool few_rows = p.M <= 128 && p.N >= 2048 && !split_k;
  return k_order == 2 ? 2 : ((k_order == 1 || (k_order < 0 && few_rows)) ? 1 : 0);
}

// Cluster launch of `kernel` on `ctas` CTAs of Cfg::kThreads threads.
template <class Cfg, class Kernel, class... Args>
cudaError_t launch_kernel(Kernel kernel, long ctas, int cluster_ctas, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  unsigned n = 0;
  if (cluster_ctas > 1) {                              // single-CTA tiles are launched without a cluster
    attrs[n].id = cudaLaunchAttributeClusterDimension;
    attrs[n].val.clusterDim.x = static_cast<unsigned>(cluster_ctas);
    attrs[n].val.clusterDim.y = 1;
    attrs[n].val.clusterDim.z = 1;
    ++n;
  }
  if (g_opt_pdl.load() != 0) {
    // Programmatic dependent launch: this kernel's CTAs may be scheduled while the previous kernel
    // of the stream drains (if that kernel allows it, as these kernels do at their start); they
    // set up barriers and tensor memory and then wait for it to complete before touching global
    // memory.  Back-to-back GEMMs lose a few microseconds less between launches.
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace host
}  // namespace gemm_sm100
