// The microscaled 4-bit format: quantisation of a matrix along its rows or along its columns, and back.
//
// Blocks of 32 elements along the contraction share X = 2^(floor(log2 amax) - 2) (one e8m0 byte); an element is
// e2m1(x / X), rounded to nearest even and saturating at 6.  Bound by memory: 2 bytes read and 0.53 written per element.
#include "lowbit.h"
#include "lowbit_common.cuh"

namespace dfb {
namespace {

// Eight elements as they lie in memory.  A load that may not be whole (FULL false) goes element by element, zeros past `live`;
// the two forms are chosen once per block, so that a whole block's loads stand one behind the other without a branch between.
template <typename T>
struct Raw8 { T v[8]; };
template <>
struct Raw8<bf16> { bf16x8 v; };
template <>
struct Raw8<float> { float4 a, b; };
template <bool FULL>
DFB_DEVICE Raw8<bf16> load8(const bf16* p, int live) {
  Raw8<bf16> r;
  if constexpr (FULL) {
    r.v = ld8(p);
  } else {
    bf16* e = reinterpret_cast<bf16*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < live ? p[i] : f2bf(0.f);
  }
  return r;
}
template <bool FULL>
DFB_DEVICE Raw8<float> load8(const float* p, int live) {
  Raw8<float> r;
  if constexpr (FULL) {
    r.a = *reinterpret_cast<const float4*>(p);
    r.b = *reinterpret_cast<const float4*>(p + 4);
  } else {
    float* e = reinterpret_cast<float*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < live ? p[i] : 0.f;
  }
  return r;
}
// Largest magnitudes as bits, which order like the numbers, with NaN above infinity.  bf16: two neighbours in one instruction.
DFB_DEVICE uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
DFB_DEVICE uint32_t words(const Raw8<bf16>& r, int j) { return *reinterpret_cast<const uint32_t*>(&r.v.v[j]); }
DFB_DEVICE float amax8(const Raw8<bf16>& r) {
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) a = max_u16x2(a, words(r, j) & 0x7fff7fffu);
  return __uint_as_float(max(a << 16, a & 0xffff0000u));
}
DFB_DEVICE float amax8(const Raw8<float>& r) {
  const float f[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  return mx_amax8(f);
}
DFB_DEVICE void widen(const Raw8<bf16>& r, float* f) { unpack8(r.v, f); }
DFB_DEVICE void widen(const Raw8<float>& r, float* f) {
  f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w;
  f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
}

// Along the rows: eight elements per lane, four lanes per block of 32; a warp takes 256 elements of kUnroll rows, all loads in
// flight at once.  The grid covers the padded scale tiles (whole 128 rows x 256 elements).
constexpr int kUnroll = 4;
template <typename T, bool FULL>
DFB_DEVICE void quant_rows(const T* x, long long ldx, uint8_t* q, uint8_t* tiles, long long rows, int K) {
  const int tile_cols = mx_tile_cols(K), k = blockIdx.x * 256 + (threadIdx.x & 31) * 8;
  const long long row0 = blockIdx.y * (8LL * kUnroll) + (threadIdx.x >> 5) * kUnroll;
  const int left = static_cast<int>(rows - row0 < kUnroll ? (rows > row0 ? rows - row0 : 0) : kUnroll);
  const T* xp = x + row0 * ldx + k;
  uint8_t* qp = q + row0 * (K >> 1) + (k >> 1);
  uint8_t* tile = tiles + mx_scale_at(row0, k >> 5, tile_cols);      // kUnroll rows inside a group of 32: 16 bytes apart
  Raw8<T> raw[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) raw[u] = load8<FULL>(xp + u * ldx, FULL || u < left ? K - k : 0);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    float f[8];
    widen(raw[u], f);
    const uint32_t sb = mx_scale_byte(mx_amax4lanes(amax8(raw[u])));
    if (FULL || (u < left && k < K)) *reinterpret_cast<uint32_t*>(qp + u * static_cast<long long>(K >> 1)) = mx_scale_pack8(f, mx_scale_inv(sb));
    const uint32_t word = mx_scale_word(sb);
    if ((threadIdx.x & 15) == 0) *reinterpret_cast<uint32_t*>(tile + u * 16) = word;
  }
}
template <typename T>
__global__ void __launch_bounds__(256) quant_mxfp4_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q,
                                                           uint8_t* __restrict__ tiles, long long rows, int K, bool vec) {
  if (vec && (blockIdx.y + 1) * (8LL * kUnroll) <= rows && static_cast<int>(blockIdx.x + 1) * 256 <= K) quant_rows<T, true>(x, ldx, q, tiles, rows, K);
  else quant_rows<T, false>(x, ldx, q, tiles, rows, K);
}

// Along the columns (x stored (K, rows)): a block takes 64 rows x 256 elements of K, warp w the 32 elements of block w.  A lane
// reads 8 neighbouring rows' values of 8 consecutive k, so that it ends with one whole word of codes per row; the words turn
// around in shared memory and leave as 128-byte rows.
template <typename T, bool FULL>
DFB_DEVICE void quant_cols(const T* x, long long ldx, long long rows, int K, uint32_t (*codes)[33], uint8_t (*scales)[8]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane & 7, sub = lane >> 3;
  const int kb = blockIdx.y * 256 + warp * 32 + sub * 8;
  const long long n = blockIdx.x * 64LL + grp * 8;
  const int live = kb < K ? static_cast<int>(rows - n < 8 ? (rows > n ? rows - n : 0) : 8) : 0;
  Raw8<T> raw[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) raw[k] = load8<FULL>(x + (kb + k) * ldx + n, live);
  float f[8][8], amax[8];                      // [k][row]
#pragma unroll
  for (int k = 0; k < 8; ++k) widen(raw[k], f[k]);
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) a = max_u16x2(a, words(raw[k], j) & 0x7fff7fffu);
      a = max_u16x2(a, __shfl_xor_sync(0xffffffffu, a, 8));
      a = max_u16x2(a, __shfl_xor_sync(0xffffffffu, a, 16));
      amax[2 * j] = __uint_as_float(a << 16);
      amax[2 * j + 1] = __uint_as_float(a & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float g[8] = {f[0][r], f[1][r], f[2][r], f[3][r], f[4][r], f[5][r], f[6][r], f[7][r]};
      float a = mx_amax8(g);
      a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 8));
      amax[r] = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 16));
    }
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const float g[8] = {f[0][r], f[1][r], f[2][r], f[3][r], f[4][r], f[5][r], f[6][r], f[7][r]};
    const uint32_t sb = mx_scale_byte(amax[r]);
    codes[grp * 8 + r][warp * 4 + sub] = mx_scale_pack8(g, mx_scale_inv(sb));
    if (sub == 0) scales[grp * 8 + r][warp] = static_cast<uint8_t>(sb);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) quant_mxfp4_cols_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q,
                                                                uint8_t* __restrict__ tiles, long long rows, int K, bool vec) {
  __shared__ uint32_t codes[64][33];           // 33: the eight row groups of a store fall on different banks
  __shared__ __align__(4) uint8_t scales[64][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tile_cols = mx_tile_cols(K), k0 = blockIdx.y * 256;
  const long long n0 = blockIdx.x * 64LL;
  if (vec && n0 + 64 <= rows && k0 + 256 <= K) quant_cols<T, true>(x, ldx, rows, K, codes, scales);
  else quant_cols<T, false>(x, ldx, rows, K, codes, scales);
  __syncthreads();
  for (int r = warp; r < 64; r += 8)
    if (n0 + r < rows && k0 + lane * 8 < K) *reinterpret_cast<uint32_t*>(q + (n0 + r) * (K >> 1) + (k0 >> 1) + lane * 4) = codes[r][lane];
  if (threadIdx.x < 128) {                     // four scale bytes of a row are one word of a tile
    const int r = threadIdx.x >> 1, half = threadIdx.x & 1;
    *reinterpret_cast<uint32_t*>(tiles + mx_scale_at(n0 + r, (k0 >> 5) + half * 4, tile_cols)) =
        *reinterpret_cast<const uint32_t*>(&scales[r][half * 4]);
  }
}

// The same walk backwards: a warp takes 256 elements of kUnroll rows.
template <typename T>
__global__ void __launch_bounds__(256) dequant_mxfp4_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ tiles,
                                                             T* __restrict__ y, long long rows, int K) {
  const int tile_cols = mx_tile_cols(K), k = blockIdx.y * 256 + (threadIdx.x & 31) * 8;
  const long long row0 = blockIdx.x * (8LL * kUnroll) + (threadIdx.x >> 5) * kUnroll;
  if (k >= K || row0 >= rows) return;
  const int left = static_cast<int>(rows - row0 < kUnroll ? rows - row0 : kUnroll);
  const uint8_t* qp = q + row0 * (K >> 1) + (k >> 1);
  const uint8_t* tile = tiles + mx_scale_at(row0, k >> 5, tile_cols);
  uint32_t c[kUnroll], sb[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    c[u] = sb[u] = 0;
    if (u < left) {
      c[u] = *reinterpret_cast<const uint32_t*>(qp + u * static_cast<long long>(K >> 1));
      sb[u] = tile[u * 16];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (u >= left) break;
    const float s = mx_scale_value(sb[u]);
    float f[8];
    mx_unpack8(c[u], f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= s;
    T* yp = y + row0 * K + k + u * static_cast<long long>(K);
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(yp) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(yp + 4) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      st8(yp, pack8(f));
    }
  }
}

}  // namespace

int quant_mxfp4(const void* x, long long ldx, int x_f32, int transposed, void* q, void* tiles, long long rows, int K, cudaStream_t s) {
  if (!rows) return 0;
  const int es = x_f32 ? 4 : 2, segs = mx_tile_cols(K) / 2;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * es) % 16 == 0;       // every row starts on 16 bytes
  const long long rows_pad = (rows + 127) / 128 * 128;
  const long long gx = rows_pad / (transposed ? 64 : 8 * kUnroll);
  if (gx > 0x7fffffffLL || segs > 65535) return -3;
  // along the rows the segments of a row come first (y: groups of 32 rows); along the columns the row tiles
  if (!transposed && gx > 65535) {           // more rows than a grid's second axis holds: in slices of whole tiles
    const long long part = 65535 / 4 * 128;  // a multiple of 128 rows
    for (long long r = 0; r < rows; r += part) {
      const int rc = quant_mxfp4(static_cast<const char*>(x) + r * ldx * es, ldx, x_f32, 0, static_cast<char*>(q) + r * (K / 2),
                                 static_cast<char*>(tiles) + (r >> 7) * mx_tile_cols(K) * 512LL, rows - r < part ? rows - r : part, K, s);
      if (rc) return rc;
    }
    return 0;
  }
  const dim3 grid = transposed ? dim3(static_cast<unsigned>(gx), segs) : dim3(segs, static_cast<unsigned>(gx));
  auto go = [&](auto kernel, auto* p) { kernel<<<grid, 256, 0, s>>>(p, ldx, (uint8_t*)q, (uint8_t*)tiles, rows, K, vec); };
  if (x_f32) {
    if (transposed) go(quant_mxfp4_cols_kernel<float>, (const float*)x);
    else go(quant_mxfp4_kernel<float>, (const float*)x);
  } else {
    if (transposed) go(quant_mxfp4_cols_kernel<bf16>, (const bf16*)x);
    else go(quant_mxfp4_kernel<bf16>, (const bf16*)x);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

int dequant_mxfp4(const void* q, const void* tiles, void* y, int y_f32, long long rows, int K, cudaStream_t s) {
  if (!rows) return 0;
  const long long gx = (rows + 8 * kUnroll - 1) / (8 * kUnroll);
  const int segs = mx_tile_cols(K) / 2;
  if (gx > 0x7fffffffLL || segs > 65535) return -3;
  const dim3 grid(static_cast<unsigned>(gx), segs);
  if (y_f32) dequant_mxfp4_kernel<float><<<grid, 256, 0, s>>>((const uint8_t*)q, (const uint8_t*)tiles, (float*)y, rows, K);
  else dequant_mxfp4_kernel<bf16><<<grid, 256, 0, s>>>((const uint8_t*)q, (const uint8_t*)tiles, (bf16*)y, rows, K);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // namespace dfb
