// harp_gemm_s8: C[M, N] = (A B^T) * sa[m] * sb[n] + bias[n] with A [M, K] and
// B [N, K] in signed 8-bit integers, a scale for each row of A (token) and of B
// (output channel), 32-bit integer sums and a bf16 or fp32 result.
//
// The integer sum is exact (K <= 131071 keeps 128 * 128 * K below 2^31), so the
// result is one rounding of the sum to fp32, two products and an addition, and
// does not depend on the order of the K loop.
#include "common.cuh"
#include "gemm_sm100.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

namespace harp {

namespace {

using bf16 = __nv_bfloat16;

struct S8Args {
  int M, N, K;
  const int8_t* A;
  long lda;
  const int8_t* B;
  long ldb;
  const float* sa;
  const float* sb;
  const void* bias;
  int bias_f32;
  void* C;
  long ldc;
  int c_f32;
  int* err;
};

__device__ __forceinline__ float bias_at(const S8Args& a, int n) {
  if (a.bias == nullptr) return 0.f;
  return a.bias_f32 ? reinterpret_cast<const float*>(a.bias)[n]
                    : __bfloat162float(reinterpret_cast<const bf16*>(a.bias)[n]);
}

// CUDA-core kernel for operands TMA cannot address (rows that do not start on
// 16-byte boundaries) and for K = 0.
__global__ void __launch_bounds__(256) gemm_s8_simt(const S8Args a) {
  __shared__ int As[32][33];
  __shared__ int Bs[32][33];
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;  // 32 x 8 threads
  const int m0 = blockIdx.y * 32, n0 = blockIdx.x * 32;
  int acc[4] = {0, 0, 0, 0};
  for (int k0 = 0; k0 < a.K; k0 += 32) {
    for (int r = ty; r < 32; r += 8) {
      const int k = k0 + tx;
      As[r][tx] = (m0 + r < a.M && k < a.K) ? (int)a.A[(long)(m0 + r) * a.lda + k] : 0;
      Bs[r][tx] = (n0 + r < a.N && k < a.K) ? (int)a.B[(long)(n0 + r) * a.ldb + k] : 0;
    }
    __syncthreads();
#pragma unroll 8
    for (int kk = 0; kk < 32; ++kk) {
      const int b = Bs[tx][kk];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += As[ty + 8 * i][kk] * b;
    }
    __syncthreads();
  }
  const int n = n0 + tx;
  if (n >= a.N) return;
  const float sb = a.sb[n], bias = bias_at(a, n);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty + 8 * i;
    if (m >= a.M) continue;
    const float v = (float)acc[i] * a.sa[m] * sb + bias;
    if (a.c_f32) reinterpret_cast<float*>(a.C)[(long)m * a.ldc + n] = v;
    else reinterpret_cast<bf16*>(a.C)[(long)m * a.ldc + n] = __float2bfloat16(v);
  }
}

void check_scales(const at::Tensor& s, const at::Tensor& rows, const char* name) {
  TORCH_CHECK(s.is_cuda() && s.device() == rows.device() && s.scalar_type() == at::kFloat && s.dim() == 1 &&
                  s.size(0) == rows.size(0) && (s.size(0) <= 1 || s.stride(0) == 1),
              "harp gemm_s8: ", name, " must be a dense fp32 vector with a scale for each row, on the operands' device");
}

}  // namespace

void gemm_s8(const at::Tensor& A, const at::Tensor& sa, const at::Tensor& B, const at::Tensor& sb,
             const c10::optional<at::Tensor>& bias, at::Tensor& C, at::Tensor& err) {
  TORCH_CHECK(A.is_cuda() && B.is_cuda() && C.is_cuda() && err.is_cuda(), "harp gemm_s8: CUDA tensors required");
  TORCH_CHECK(A.device() == B.device() && A.device() == C.device() && A.device() == err.device(),
              "harp gemm_s8: operands on one device");
  TORCH_CHECK(A.scalar_type() == at::kChar && B.scalar_type() == at::kChar, "harp gemm_s8: int8 operands");
  TORCH_CHECK(A.dim() == 2 && B.dim() == 2 && C.dim() == 2, "harp gemm_s8: 2-D operands");
  const int64_t M = A.size(0), N = B.size(0), K = A.size(1);
  TORCH_CHECK(B.size(1) == K, "harp gemm_s8: A has ", std::to_string(K), " columns and B ", std::to_string(B.size(1)));
  TORCH_CHECK(C.size(0) == M && C.size(1) == N, "harp gemm_s8: C shape");
  TORCH_CHECK(K <= 131071, "harp gemm_s8: K = ", std::to_string(K), " could overflow the 32-bit sums (at most 131071)");
  TORCH_CHECK(M <= 0x7FFFFF00 && N <= 0x7FFFFF00, "harp gemm_s8: M and N below 2^31");
  TORCH_CHECK((A.stride(1) == 1 || K <= 1) && (B.stride(1) == 1 || K <= 1) && (C.stride(1) == 1 || N <= 1),
              "harp gemm_s8: unit inner stride");
  TORCH_CHECK(C.scalar_type() == at::kBFloat16 || C.scalar_type() == at::kFloat, "harp gemm_s8: bf16 or fp32 output");
  TORCH_CHECK(err.scalar_type() == at::kInt && err.numel() >= 4, "harp gemm_s8: error word");
  check_scales(sa, A, "a_scale");
  check_scales(sb, B, "b_scale");
  if (bias.has_value())
    TORCH_CHECK(bias->is_cuda() && bias->device() == A.device() && bias->dim() == 1 && bias->size(0) == N &&
                    (N <= 1 || bias->stride(0) == 1) &&
                    (bias->scalar_type() == at::kBFloat16 || bias->scalar_type() == at::kFloat),
                "harp gemm_s8: bias must be a dense bf16 or fp32 vector of ", std::to_string(N), " values on the operands' device");
  if (M == 0 || N == 0) return;
  const at::cuda::CUDAGuard guard(A.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  S8Args a;
  a.M = (int)M; a.N = (int)N; a.K = (int)K;
  a.A = reinterpret_cast<const int8_t*>(A.data_ptr());
  a.lda = A.stride(0);
  a.B = reinterpret_cast<const int8_t*>(B.data_ptr());
  a.ldb = B.stride(0);
  a.sa = sa.data_ptr<float>();
  a.sb = sb.data_ptr<float>();
  a.bias = bias.has_value() ? bias->data_ptr() : nullptr;
  a.bias_f32 = bias.has_value() && bias->scalar_type() == at::kFloat;
  a.C = C.data_ptr();
  a.ldc = C.stride(0);
  a.c_f32 = C.scalar_type() == at::kFloat;
  a.err = err.data_ptr<int>();
  dim3 grid((unsigned)((N + 31) / 32), (unsigned)((M + 31) / 32));
  TORCH_CHECK(grid.y <= 65535, "harp gemm_s8: too many rows for the CUDA-core path");
  gemm_s8_simt<<<grid, 256, 0, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launch();
}

}  // namespace harp
