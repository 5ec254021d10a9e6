// The microscaled 4-bit format: quantisation of a matrix along its rows or along its columns, and back.
//
// Blocks of 32 elements along the contraction share X = 2^(floor(log2 amax) - 2) (one e8m0 byte); an element is
// e2m1(x / X), rounded to nearest even and saturating at 6.  Bound by memory: 2 bytes read and 0.53 written per element.
#include "lowbit.h"
#include "lowbit_common.cuh"

namespace dfb {
namespace {

DFB_DEVICE float to_float(float x) { return x; }
DFB_DEVICE float to_float(bf16 x) { return bf2f(x); }

// one thread per (row, block of 32), the padding of the scale tiles included
template <typename T, bool TRANS>
__global__ void __launch_bounds__(256) quant_mxfp4_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q,
                                                           uint8_t* __restrict__ tiles, long long rows, int K) {
  const int tile_cols = mx_tile_cols(K), blocks = tile_cols * 4;
  const long long rows_pad = (rows + 127) / 128 * 128;
  const long long idx = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
  // neighbouring threads: neighbouring blocks of a row, or neighbouring rows of a transposed matrix
  const long long row = TRANS ? idx % rows_pad : idx / blocks;
  const int b = static_cast<int>(TRANS ? idx / rows_pad : idx % blocks);
  if (row >= rows_pad || b >= blocks) return;
  uint32_t sb = 0;
  if (row < rows && b < K / kMxBlock) {
    float f[32], amax = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const long long k = b * 32 + i;
      f[i] = to_float(TRANS ? x[k * ldx + row] : x[row * ldx + k]);
      amax = fmaxf(amax, mx_abs(f[i]));
    }
    sb = mx_scale_byte(amax);
    const float inv = mx_scale_inv(sb);
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] *= inv;
    *reinterpret_cast<uint4*>(q + row * (K >> 1) + b * 16) = make_uint4(mx_pack8(f), mx_pack8(f + 8), mx_pack8(f + 16), mx_pack8(f + 24));
  }
  tiles[mx_scale_at(row, b, tile_cols)] = static_cast<uint8_t>(sb);
}

// one thread per eight elements
template <typename T>
__global__ void __launch_bounds__(256) dequant_mxfp4_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ tiles,
                                                             T* __restrict__ y, long long rows, int K) {
  const long long idx = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
  const int nvec = K >> 3;
  const long long row = idx / nvec;
  const int v = static_cast<int>(idx % nvec);
  if (row >= rows) return;
  const uint32_t c = *reinterpret_cast<const uint32_t*>(q + row * (K >> 1) + v * 4);
  const float s = mx_scale_value(tiles[mx_scale_at(row, v >> 2, mx_tile_cols(K))]);
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = mx_value((c >> (4 * i)) & 15u) * s;
  T* yp = y + row * K + v * 8;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(yp) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(yp + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    st8(yp, pack8(f));
  }
}

}  // namespace

int quant_mxfp4(const void* x, long long ldx, int x_f32, int transposed, void* q, void* tiles, long long rows, int K, cudaStream_t s) {
  if (!rows) return 0;
  const long long n = (rows + 127) / 128 * 128 * mx_tile_cols(K) * 4, grid = (n + 255) / 256;
  if (grid > 0x7fffffffLL) return -3;
  auto go = [&](auto kernel, auto* p) { kernel<<<static_cast<unsigned>(grid), 256, 0, s>>>(p, ldx, (uint8_t*)q, (uint8_t*)tiles, rows, K); };
  if (x_f32) {
    if (transposed) go(quant_mxfp4_kernel<float, true>, (const float*)x);
    else go(quant_mxfp4_kernel<float, false>, (const float*)x);
  } else {
    if (transposed) go(quant_mxfp4_kernel<bf16, true>, (const bf16*)x);
    else go(quant_mxfp4_kernel<bf16, false>, (const bf16*)x);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

int dequant_mxfp4(const void* q, const void* tiles, void* y, int y_f32, long long rows, int K, cudaStream_t s) {
  const long long n = rows * (K >> 3), grid = (n + 255) / 256;
  if (!n) return 0;
  if (grid > 0x7fffffffLL) return -3;
  if (y_f32) dequant_mxfp4_kernel<float><<<static_cast<unsigned>(grid), 256, 0, s>>>((const uint8_t*)q, (const uint8_t*)tiles, (float*)y, rows, K);
  else dequant_mxfp4_kernel<bf16><<<static_cast<unsigned>(grid), 256, 0, s>>>((const uint8_t*)q, (const uint8_t*)tiles, (bf16*)y, rows, K);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // namespace dfb
