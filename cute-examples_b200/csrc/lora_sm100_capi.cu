// Host side of the low-rank adapter entry points (gemm_sm100_lora* in include/gemm_sm100.h): argument
// checks, launches.
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/gemm_sm100.h"
#include "lora_sm100.cuh"

namespace {

using namespace gemm_sm100;

int cuda_failed(int* out, cudaError_t e) {
  if (out) *out = static_cast<int>(e);
  return GEMM_SM100_ERR_CUDA;
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
long ceil_div(long a, long b) { return (a + b - 1) / b; }

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

template <bool kIsBf16>
void launch_low(const gemm_sm100_lora_args& a, const void* P, long ldp, const void* W, long stride_g, long stride_r,
                long stride_l, int L, void* out, long ld_out, cudaStream_t stream) {
  const long warps = static_cast<long>(a.M) * a.R;
  lora_low_simple_kernel<kIsBf16><<<static_cast<unsigned>(ceil_div(warps, 8)), 256, 0, stream>>>(
      u16(P), ldp, u16(W), stride_g, stride_r, stride_l, a.scales, a.scale, u16(out), ld_out, a.M, a.R, L,
      const_cast<void*>(a.plan));
}

template <bool kIsBf16>
void launch_product(const gemm_sm100_lora_args& a, const void* A, long lda, long stride_bn, long stride_bl, const void* low,
                    long ld_low, const void* W, long stride_g, long stride_n, long stride_r, int N, int L, void* C, long ldc,
                    cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(ceil_div(N, 16)), static_cast<unsigned>(ceil_div(a.M, 16)));
  lora_product_simple_kernel<kIsBf16><<<grid, dim3(16, 16), 0, stream>>>(
      u16(A), lda, u16(a.B), stride_bn, stride_bl, u16(low), ld_low, u16(W), stride_g, stride_n, stride_r, u16(C), ldc, a.M, N,
      L, a.R, const_cast<void*>(a.plan));
}

template <bool kIsBf16>
void launch_grad(const gemm_sm100_lora_args& a, const void* P, long ldp, const void* Q, long ldq, void* out, long stride_i,
                 long stride_r, int D, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<long>(D) * a.R, 256)), static_cast<unsigned>(a.adapters));
  lora_grad_simple_kernel<kIsBf16><<<grid, 256, 0, stream>>>(u16(P), ldp, u16(Q), ldq, u16(out), stride_i, stride_r, a.M, D,
                                                             a.R, const_cast<void*>(a.plan));
}

}  // namespace

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
  return e == cudaSuccess ? GEMM_SM100_OK : cuda_failed(cuda_error_out, e);
}

int gemm_sm100_lora_low(const gemm_sm100_lora_args* args, void* low, long ld_low, void* cuda_stream, int* cuda_error_out) {
  if (cuda_error_out) *cuda_error_out = 0;
  if (!args) return GEMM_SM100_ERR_NULL_POINTER;
  const gemm_sm100_lora_args& a = *args;
  int rc = check_common(a);
  if (rc != GEMM_SM100_OK) return rc;
  if (a.M == 0) return GEMM_SM100_OK;
  if (!a.plan) return GEMM_SM100_ERR_NULL_POINTER;
  if ((rc = check_matrix(a.A, a.K, a.lda)) || (rc = check_down(a)) || (rc = check_matrix(low, a.R, ld_low))) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  auto launch = a.dtype == GEMM_SM100_BF16 ? launch_low<true> : launch_low<false>;
  launch(a, a.A, a.lda, a.down, a.stride_down, a.ld_down, 1, a.K, low, ld_low, stream);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GEMM_SM100_OK : cuda_failed(cuda_error_out, e);
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
  rc = gemm_sm100_lora_low(args, low, ld_low, cuda_stream, cuda_error_out);
  if (rc != GEMM_SM100_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  auto launch = a.dtype == GEMM_SM100_BF16 ? launch_product<true> : launch_product<false>;
  launch(a, a.A, a.lda, a.ldb, 1, low, ld_low, a.up, a.stride_up, a.ld_up, 1, a.N, a.K, C, ldc, stream);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GEMM_SM100_OK : cuda_failed(cuda_error_out, e);
}

int gemm_sm100_lora_backward(const gemm_sm100_lora_args* args, const void* dC, long ld_dc, const void* low, long ld_low,
                             void* d_low, long ld_d_low, void* dA, long ld_da, void* d_down, void* d_up, void* cuda_stream,
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
    return e == cudaSuccess ? GEMM_SM100_OK : cuda_failed(cuda_error_out, e);
  }
  if (!a.plan) return GEMM_SM100_ERR_NULL_POINTER;
  if ((rc = check_matrix(dC, a.N, ld_dc))) return rc;
  if (d_down && (rc = check_matrix(a.A, a.K, a.lda))) return rc;
  if (d_up && (rc = check_matrix(low, a.R, ld_low))) return rc;
  if (dA && ((rc = check_matrix(a.B, a.K, a.ldb)) || (rc = check_down(a)) || (rc = check_matrix(dA, a.K, ld_da)))) return rc;
  const bool bf16 = a.dtype == GEMM_SM100_BF16;
  if (dA || d_down) {
    if ((rc = check_up(a)) || (rc = check_matrix(d_low, a.R, ld_d_low))) return rc;
    (bf16 ? launch_low<true> : launch_low<false>)(a, dC, ld_dc, a.up, a.stride_up, 1, a.ld_up, a.N, d_low, ld_d_low, stream);
  }
  if (dA)
    (bf16 ? launch_product<true> : launch_product<false>)(a, dC, ld_dc, 1, a.ldb, d_low, ld_d_low, a.down, a.stride_down, 1,
                                                          a.ld_down, a.K, a.N, dA, ld_da, stream);
  if (d_down) (bf16 ? launch_grad<true> : launch_grad<false>)(a, a.A, a.lda, d_low, ld_d_low, d_down, 1, a.K, a.K, stream);
  if (d_up) (bf16 ? launch_grad<true> : launch_grad<false>)(a, dC, ld_dc, low, ld_low, d_up, a.R, 1, a.N, stream);
  e = cudaGetLastError();
  return e == cudaSuccess ? GEMM_SM100_OK : cuda_failed(cuda_error_out, e);
}

}  // extern "C"
