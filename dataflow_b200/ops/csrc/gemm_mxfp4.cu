// Product of two operands in the microscaled 4-bit format: D (M, N) = A (M, K) x B (N, K)^T (+ bias) (+ addend).
//
//   D[m, n] = sum over blocks b of 32:  2^(sa[m, b] + sb[n, b] - 254) * sum_i a[m, 32 b + i] b[n, 32 b + i]
//
// Plain form on the ordinary arithmetic units: 32 x 32 outputs per block, operands decoded into shared memory.
#include "lowbit.h"
#include "lowbit_common.cuh"

namespace dfb {
namespace {

__global__ void __launch_bounds__(1024) gemm_mxfp4_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ sa,
                                                           const uint8_t* __restrict__ B, const uint8_t* __restrict__ sb, void* D, long long ldd,
                                                           int d_f32, const void* add, long long ld_add, const bf16* __restrict__ bias,
                                                           long long M, long long N, int K) {
  __shared__ float as[32][33], bs[32][33];
  const long long m0 = blockIdx.x * 32LL, n0 = blockIdx.y * 32LL;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, tile_cols = mx_tile_cols(K);
  float acc = 0.f;
  for (int b = 0; b < K / 32; ++b) {
    const long long m = m0 + ty, n = n0 + ty;
    const int k = b * 32 + tx;
    as[ty][tx] = m < M ? mx_value((A[m * (K >> 1) + (k >> 1)] >> (4 * (k & 1))) & 15u) * mx_scale_value(sa[mx_scale_at(m, b, tile_cols)]) : 0.f;
    bs[ty][tx] = n < N ? mx_value((B[n * (K >> 1) + (k >> 1)] >> (4 * (k & 1))) & 15u) * mx_scale_value(sb[mx_scale_at(n, b, tile_cols)]) : 0.f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32; ++i) acc += as[ty][i] * bs[tx][i];
    __syncthreads();
  }
  const long long m = m0 + ty, n = n0 + tx;
  if (m >= M || n >= N) return;
  if (bias) acc += bf2f(bias[n]);
  if (d_f32) {
    if (add) acc += reinterpret_cast<const float*>(add)[m * ld_add + n];
    reinterpret_cast<float*>(D)[m * ldd + n] = acc;
  } else {
    if (add) acc += bf2f(reinterpret_cast<const bf16*>(add)[m * ld_add + n]);
    reinterpret_cast<bf16*>(D)[m * ldd + n] = f2bf(acc);
  }
}

}  // namespace

int gemm_mxfp4(const void* A, const void* sa, const void* B, const void* sb, void* D, long long ldd, int d_f32, const void* add,
               long long ld_add, const void* bias, long long M, long long N, int K, int num_sms, cudaStream_t s) {
  if (!M || !N) return 0;
  const long long gx = (M + 31) / 32, gy = (N + 31) / 32;
  if (gx > 0x7fffffffLL || gy > 65535) return -3;
  gemm_mxfp4_kernel<<<dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), 1024, 0, s>>>(
      (const uint8_t*)A, (const uint8_t*)sa, (const uint8_t*)B, (const uint8_t*)sb, D, ldd, d_f32, add, ld_add, (const bf16*)bias, M, N, K);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

int gemm_mxfp4_last_error() { return 0; }

}  // namespace dfb
