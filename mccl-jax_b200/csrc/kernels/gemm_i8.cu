// gemm_i8.cu — products of 8-bit integers with a scale per row of each operand:
//     C[i][j] = act(f32(sum_k A[i][k] B[j][k]) * a_scale[i] * b_scale[j] + bias[j])
// with the sum exact in 32-bit integers, and the raw sums themselves (s32 C).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kernels.h"
#include "../../../include/b200_kernels.h"

namespace b200k {
namespace {

enum : int { kOutF32 = 0, kOutBF16 = 1, kOutF16 = 2, kOutS32 = 3 };

// What follows the integer sum.  Null scales are 1, a null bias 0.
struct Epilogue {
  const float* a_scale;
  const float* b_scale;
  const float* bias;
  int gelu;
};

// The tanh form of GELU, 0.5 v (1 + tanh u) with u = sqrt(2 / pi) (v + 0.044715 v^3), as v / (1 + e^-2u):
// the same function without the cancellation in 1 + tanh(u) for u < 0.
__device__ __forceinline__ float gelu_tanh(float v) {
  constexpr float kU = -2.0f * 0.7978845608028654f * 1.4426950408889634f;   // -2 sqrt(2 / pi) log2(e)
  const float e = exp2f(kU * v * fmaf(0.044715f * v, v, 1.0f));
  return __fdividef(v, 1.0f + e);
}

__device__ __forceinline__ float finish(int acc, float sa, float sb, float bias, int gelu) {
  const float v = fmaf((float)acc * sa, sb, bias);
  return gelu ? gelu_tanh(v) : v;
}

template <int OUT>
__device__ __forceinline__ void store_one(void* C, long long at, int acc, float v) {
  if (OUT == kOutF32) ((float*)C)[at] = v;
  else if (OUT == kOutBF16) ((__nv_bfloat16*)C)[at] = __float2bfloat16_rn(v);
  else if (OUT == kOutF16) ((__half*)C)[at] = __float2half_rn(v);
  else ((int*)C)[at] = acc;
}

// 64 x 64 tiles, 16 k at a time, 4 x 4 sums per thread, one byte per load: any size, pitch and address.
template <int OUT>
__global__ void __launch_bounds__(256) gemm_i8_simt_kernel(const int8_t* __restrict__ A, long long lda, const int8_t* __restrict__ B,
                                                           long long ldb, void* __restrict__ C, long long ldc, int M, int N, int K,
                                                           const Epilogue ep) {
  __shared__ int As[64][5], Bs[64][5];           // 16 bytes a row, and a word apart from the next bank
  const long long m0 = (long long)blockIdx.y * 64, n0 = (long long)blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 16) {
    for (int e = threadIdx.x; e < 64 * 16; e += 256) {
      const int row = e >> 4, k = k0 + (e & 15);
      ((int8_t*)As[row])[e & 15] = m0 + row < M && k < K ? A[(m0 + row) * lda + k] : (int8_t)0;
      ((int8_t*)Bs[row])[e & 15] = n0 + row < N && k < K ? B[(n0 + row) * ldb + k] : (int8_t)0;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(As[ty + 16 * i][w], Bs[tx + 16 * j][w], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long m = m0 + ty + 16 * i;
    if (m >= M) continue;
    const float sa = ep.a_scale ? ep.a_scale[m] : 1.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long n = n0 + tx + 16 * j;
      if (n >= N) continue;
      const float v = OUT == kOutS32 ? 0.f
                                     : finish(acc[i][j], sa, ep.b_scale ? ep.b_scale[n] : 1.f, ep.bias ? ep.bias[n] : 0.f, ep.gelu);
      store_one<OUT>(C, m * ldc + n, acc[i][j], v);
    }
  }
}

int OutCodeI8(int type) {
  return type == B200_DT_F32 ? kOutF32 : type == B200_DT_BF16 ? kOutBF16 : type == B200_DT_F16 ? kOutF16 : type == B200_DT_S32 ? kOutS32 : -1;
}

}  // namespace

size_t GemmI8ScratchBytes(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K) { return 0; }

int GemmI8(const void* A, int64_t lda, const void* B, int64_t ldb, const float* a_scale, const float* b_scale, const float* bias,
           void* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int out_type, int act, void* scratch, size_t scratch_bytes,
           cudaStream_t st) {
  const int out = OutCodeI8(out_type);
  if (out < 0 || M < 0 || N < 0 || K < 0 || M > INT32_MAX || N > INT32_MAX || K > kGemmI8MaxK || lda < K || ldb < K || ldc < N)
    return -1;
  if (act < 0 || act > 1 || (out == kOutS32 && (a_scale || b_scale || bias || act))) return -1;
  if (M == 0 || N == 0) return 0;
  const int es = out == kOutBF16 || out == kOutF16 ? 2 : 4;
  if ((K && (!A || !B)) || !C || (uintptr_t)C % es || (uintptr_t)a_scale % 4 || (uintptr_t)b_scale % 4 || (uintptr_t)bias % 4) return -1;
  if ((M + 63) / 64 > 65535) return -1;
  const Epilogue ep = {a_scale, b_scale, bias, act};
  const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64));
  const int8_t *a = (const int8_t*)A, *b = (const int8_t*)B;
  if (out == kOutF32) gemm_i8_simt_kernel<kOutF32><<<grid, 256, 0, st>>>(a, lda, b, ldb, C, ldc, (int)M, (int)N, (int)K, ep);
  else if (out == kOutBF16) gemm_i8_simt_kernel<kOutBF16><<<grid, 256, 0, st>>>(a, lda, b, ldb, C, ldc, (int)M, (int)N, (int)K, ep);
  else if (out == kOutF16) gemm_i8_simt_kernel<kOutF16><<<grid, 256, 0, st>>>(a, lda, b, ldb, C, ldc, (int)M, (int)N, (int)K, ep);
  else gemm_i8_simt_kernel<kOutS32><<<grid, 256, 0, st>>>(a, lda, b, ldb, C, ldc, (int)M, (int)N, (int)K, ep);
  CountLaunches();
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace b200k

extern "C" size_t b200_gemm_i8_scratch_bytes(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K) {
  return b200k::GemmI8ScratchBytes(A, lda, B, ldb, M, N, K);
}

extern "C" int b200_gemm_i8(const void* A, int64_t lda, const void* B, int64_t ldb, const float* a_scale, const float* b_scale,
                            const float* bias, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int out_type, int act,
                            void* scratch, size_t scratch_bytes, void* stream) {
  return b200k::GemmI8(A, lda, B, ldb, a_scale, b_scale, bias, C, ldc, M, N, K, out_type, act, scratch, scratch_bytes,
                       (cudaStream_t)stream);
}
