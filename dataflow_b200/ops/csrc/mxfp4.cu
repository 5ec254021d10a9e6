// The microscaled 4-bit format: quantisation of a matrix along its rows or along its columns, and back.
//
// Blocks of 32 elements along the contraction share X = 2^(floor(log2 amax) - 2) (one e8m0 byte); an element is
// e2m1(x / X), rounded to nearest even and saturating at 6.  Bound by memory, 2 bytes read and 0.53 written per element of bf16:
// 8192 x 4096 along the rows 16.3 us (0.8 of the copy rate, ramps included), 4096 x 14336 along the columns 29.6 us (0.77: what
// registers hold of a block's loads), 14336 x 4096 back 21.9 us (the copy rate).
#include "lowbit.h"
#include "lowbit_common.cuh"

namespace dfb {
namespace {

// Sixteen elements as they lie in memory.  How they are fetched is chosen once per block, so that its loads stand one behind the
// other without a branch between: 32 bytes at a time (8192 x 4096 along the rows 16.5 us; 16 bytes at a time 20.6), 16 bytes where
// rows do not start on 32, or element by element, zeros past `live`.
enum Fetch { kElements, k16Bytes, k32Bytes };
template <typename T>
struct Raw {
  uint32_t u[4 * sizeof(T)];
};
template <int HOW, typename T>
DFB_DEVICE Raw<T> fetch16(const T* p, int live) {
  Raw<T> r;
  if constexpr (HOW == k32Bytes) {
#pragma unroll
    for (int i = 0; i < 4 * static_cast<int>(sizeof(T)); i += 8) load32(reinterpret_cast<const uint32_t*>(p) + i, r.u + i);
  } else if constexpr (HOW == k16Bytes) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) *reinterpret_cast<uint4*>(r.u + 4 * i) = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (sizeof(T) == 4) {
        r.u[i] = i < live ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
      } else {
        if (!(i & 1)) r.u[i >> 1] = 0;
        if (i < live) r.u[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
      }
    }
  }
  return r;
}
// elements 8 h .. 8 h + 7 in fp32
template <typename T>
DFB_DEVICE void widen8(const Raw<T>& r, int h, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4) f[i] = __uint_as_float(r.u[8 * h + i]);
    else f[i] = __uint_as_float(i & 1 ? r.u[4 * h + (i >> 1)] & 0xffff0000u : r.u[4 * h + (i >> 1)] << 16);
  }
}
// Largest magnitudes as bits, which order like the numbers, with NaN above infinity.  bf16: two neighbours in one instruction.
DFB_DEVICE uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
DFB_DEVICE float amax16(const Raw<T>& r) {
  uint32_t a = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) a = max(a, r.u[i] & 0x7fffffffu);
    return __uint_as_float(a);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max_u16x2(a, r.u[i] & 0x7fff7fffu);
    return __uint_as_float(max(a << 16, a & 0xffff0000u));
  }
}

// Along the rows: sixteen elements per lane, two lanes per block of 32; a warp takes 256 elements of two rows, kUnroll times, all
// loads in flight at once.  The grid covers the padded scale tiles (whole 128 rows x 256 elements).
constexpr int kUnroll = 2;
constexpr int kRowsPerBlock = 8 * 2 * kUnroll;
template <typename T, int HOW>
DFB_DEVICE void quant_rows(const T* x, long long ldx, uint8_t* q, uint8_t* tiles, long long rows, int K) {
  const int lane = threadIdx.x & 31, tile_cols = mx_tile_cols(K), k = blockIdx.x * 256 + (lane & 15) * 16;
  const long long row0 = blockIdx.y * static_cast<long long>(kRowsPerBlock) + (threadIdx.x >> 5) * (2 * kUnroll) + (lane >> 4);
  const T* xp = x + row0 * ldx + k;
  uint8_t* qp = q + row0 * (K >> 1) + (k >> 1);
  uint8_t* tile = tiles + mx_scale_at(row0, k >> 5, tile_cols);      // the block's rows lie in one group of 32: 16 bytes apart
  Raw<T> raw[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) raw[u] = fetch16<HOW>(xp + 2 * u * ldx, row0 + 2 * u < rows ? K - k : 0);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t sb = mx_scale_byte(mx_amax_lanes<2>(amax16(raw[u])));
    const float inv = mx_scale_inv(sb);
    float f[8];
    uint2 c;
    widen8(raw[u], 0, f);
    c.x = mx_scale_pack8(f, inv);
    widen8(raw[u], 1, f);
    c.y = mx_scale_pack8(f, inv);
    if (HOW != kElements || (row0 + 2 * u < rows && k < K)) *reinterpret_cast<uint2*>(qp + 2 * u * static_cast<long long>(K >> 1)) = c;
    const uint32_t word = mx_scale_word<2>(sb);
    if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(tile + 2 * u * 16) = word;
  }
}
template <typename T>
__global__ void __launch_bounds__(256) quant_mxfp4_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q,
                                                           uint8_t* __restrict__ tiles, long long rows, int K, int how) {
  const bool whole = (blockIdx.y + 1) * static_cast<long long>(kRowsPerBlock) <= rows && static_cast<int>(blockIdx.x + 1) * 256 <= K;
  if (whole && how == k32Bytes) quant_rows<T, k32Bytes>(x, ldx, q, tiles, rows, K);
  else if (whole && how == k16Bytes) quant_rows<T, k16Bytes>(x, ldx, q, tiles, rows, K);
  else quant_rows<T, kElements>(x, ldx, q, tiles, rows, K);
}

// Along the columns (x stored (K, rows)): a block takes 128 rows x 256 elements of K, two tiles of scales; warp w the 32 elements
// of block w.  A lane reads 16 neighbouring rows' values of 8 consecutive k, so that it ends with one whole word of codes per row;
// the words turn around in shared memory and leave as 128-byte rows.
template <typename T, int HOW>
DFB_DEVICE void quant_cols(const T* x, long long ldx, long long rows, int K, uint32_t (*codes)[32], uint8_t* scales) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane & 7, sub = lane >> 3;
  const int kb = blockIdx.y * 256 + warp * 32 + sub * 8;
  const long long n = blockIdx.x * 128LL + grp * 16;
  const int live = kb < K ? static_cast<int>(rows - n < 16 ? (rows > n ? rows - n : 0) : 16) : 0;
  constexpr int kParts = sizeof(T) == 4 ? 2 : 1;           // fp32: eight rows' values at a time, for the registers
#pragma unroll 1
  for (int part = 0; part < kParts; ++part) {
    constexpr int W = 16 / kParts;
    uint32_t raw[8][W * sizeof(T) / 4];                    // [k][rows]
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (sizeof(T) == 2) {
        const Raw<T> r = fetch16<HOW>(x + (kb + k) * ldx + n, live);
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[k][i] = r.u[i];
      } else {
        const T* p = x + (kb + k) * ldx + n + part * 8;
        if constexpr (HOW == k32Bytes) {
          load32(p, raw[k]);
        } else if constexpr (HOW == k16Bytes) {
          *reinterpret_cast<uint4*>(raw[k]) = reinterpret_cast<const uint4*>(p)[0];
          *reinterpret_cast<uint4*>(raw[k] + 4) = reinterpret_cast<const uint4*>(p)[1];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) raw[k][i] = part * 8 + i < live ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < W * static_cast<int>(sizeof(T)) / 4; ++j) {
      uint32_t a = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) a = sizeof(T) == 4 ? max(a, raw[k][j] & 0x7fffffffu) : max_u16x2(a, raw[k][j] & 0x7fff7fffu);
#pragma unroll
      for (int o = 8; o <= 16; o <<= 1) {
        const uint32_t b = __shfl_xor_sync(0xffffffffu, a, o);
        a = sizeof(T) == 4 ? max(a, b) : max_u16x2(a, b);
      }
#pragma unroll
      for (int h = 0; h < 4 / static_cast<int>(sizeof(T)); ++h) {
        const int r = grp * 16 + (sizeof(T) == 4 ? part * 8 + j : 2 * j + h);
        const uint32_t sb = mx_scale_byte(__uint_as_float(sizeof(T) == 4 ? a : h ? a & 0xffff0000u : a << 16));
        float g[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = __uint_as_float(sizeof(T) == 4 ? raw[k][j] : h ? raw[k][j] & 0xffff0000u : raw[k][j] << 16);
        codes[r][(warp * 4 + sub) ^ (grp << 2)] = mx_scale_pack8(g, mx_scale_inv(sb));
        if (sub == 0) scales[(warp >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (warp & 3)] = static_cast<uint8_t>(sb);
      }
    }
  }
}
template <typename T>
__global__ void __launch_bounds__(256) quant_mxfp4_cols_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q,
                                                                uint8_t* __restrict__ tiles, long long rows, int K, int how) {
  __shared__ uint32_t codes[128][32];          // words exchanged by row group: the eight groups of a store fall on different banks
  __shared__ __align__(16) uint8_t scales[1024];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k0 = blockIdx.y * 256;
  const long long n0 = blockIdx.x * 128LL;
  const bool whole = n0 + 128 <= rows && k0 + 256 <= K;
  if (whole && how == k32Bytes) quant_cols<T, k32Bytes>(x, ldx, rows, K, codes, scales);
  else if (whole && how == k16Bytes) quant_cols<T, k16Bytes>(x, ldx, rows, K, codes, scales);
  else quant_cols<T, kElements>(x, ldx, rows, K, codes, scales);
  __syncthreads();
  for (int r = warp; r < 128; r += 8)
    if (n0 + r < rows && k0 + lane * 8 < K) *reinterpret_cast<uint32_t*>(q + (n0 + r) * (K >> 1) + (k0 >> 1) + lane * 4) = codes[r][lane ^ ((r >> 4) << 2)];
  if (threadIdx.x < 64)                        // the two tiles of scales are neighbours
    reinterpret_cast<uint4*>(tiles + mx_scale_at(n0, k0 >> 5, mx_tile_cols(K)))[threadIdx.x] = reinterpret_cast<const uint4*>(scales)[threadIdx.x];
}

// The walk along the rows backwards: sixteen elements per lane, stored 32 bytes at a time.
template <typename T>
__global__ void __launch_bounds__(256) dequant_mxfp4_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ tiles,
                                                             T* __restrict__ y, long long rows, int K) {
  const int lane = threadIdx.x & 31, tile_cols = mx_tile_cols(K), k = blockIdx.x * 256 + (lane & 15) * 16;
  const long long row0 = blockIdx.y * static_cast<long long>(kRowsPerBlock) + (threadIdx.x >> 5) * (2 * kUnroll) + (lane >> 4);
  if (k >= K) return;
  const uint8_t* qp = q + row0 * (K >> 1) + (k >> 1);
  const uint8_t* tile = tiles + mx_scale_at(row0, k >> 5, tile_cols);
  uint2 c[kUnroll];
  uint32_t sb[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    c[u] = make_uint2(0, 0);
    sb[u] = 0;
    if (row0 + 2 * u < rows) {
      c[u] = *reinterpret_cast<const uint2*>(qp + 2 * u * static_cast<long long>(K >> 1));
      sb[u] = tile[2 * u * 16];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (row0 + 2 * u >= rows) break;
    const float2 s = both(mx_scale_value(sb[u]));
    float f[16];
    mx_unpack8(c[u].x, f);
    mx_unpack8(c[u].y, f + 8);
    uint32_t out[4 * sizeof(T)];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = mul2(make_float2(f[2 * i], f[2 * i + 1]), s);
      if constexpr (sizeof(T) == 4) {
        out[2 * i] = __float_as_uint(v.x);
        out[2 * i + 1] = __float_as_uint(v.y);
      } else {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
        out[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    uint32_t* yp = reinterpret_cast<uint32_t*>(y + (row0 + 2 * u) * K + k);
#pragma unroll
    for (int i = 0; i < 4 * static_cast<int>(sizeof(T)); i += 8) store32(yp + i, out + i);
  }
}

}  // namespace

int quant_mxfp4(const void* x, long long ldx, int x_f32, int transposed, void* q, void* tiles, long long rows, int K, cudaStream_t s) {
  if (!rows) return 0;
  const int es = x_f32 ? 4 : 2, segs = mx_tile_cols(K) / 2;
  auto starts_on = [&](int bytes) { return reinterpret_cast<uintptr_t>(x) % bytes == 0 && (ldx * es) % bytes == 0; };
  const int how = starts_on(32) ? k32Bytes : starts_on(16) ? k16Bytes : kElements;
  const long long rows_pad = (rows + 127) / 128 * 128;
  const long long gx = rows_pad / (transposed ? 128 : kRowsPerBlock);
  if (gx > 0x7fffffffLL || segs > 65535) return -3;
  // along the rows the segments of a row come first (y: groups of 32 rows); along the columns the row tiles
  if (!transposed && gx > 65535) {           // more rows than a grid's second axis holds: in slices of whole tiles
    const long long part = 65535LL * kRowsPerBlock / 128 * 128;
    for (long long r = 0; r < rows; r += part) {
      const int rc = quant_mxfp4(static_cast<const char*>(x) + r * ldx * es, ldx, x_f32, 0, static_cast<char*>(q) + r * (K / 2),
                                 static_cast<char*>(tiles) + (r >> 7) * mx_tile_cols(K) * 512LL, rows - r < part ? rows - r : part, K, s);
      if (rc) return rc;
    }
    return 0;
  }
  const dim3 grid = transposed ? dim3(static_cast<unsigned>(gx), segs) : dim3(segs, static_cast<unsigned>(gx));
  auto go = [&](auto kernel, auto* p) { kernel<<<grid, 256, 0, s>>>(p, ldx, (uint8_t*)q, (uint8_t*)tiles, rows, K, how); };
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
  const long long gy = (rows + kRowsPerBlock - 1) / kRowsPerBlock;
  const int segs = mx_tile_cols(K) / 2;
  if (gy > 65535) {                          // more rows than a grid's second axis holds: in slices of whole tiles
    const long long part = 65535LL * kRowsPerBlock / 128 * 128;
    for (long long r = 0; r < rows; r += part) {
      const int rc = dequant_mxfp4(static_cast<const char*>(q) + r * (K / 2), static_cast<const char*>(tiles) + (r >> 7) * mx_tile_cols(K) * 512LL,
                                   static_cast<char*>(y) + r * K * (y_f32 ? 4 : 2), y_f32, rows - r < part ? rows - r : part, K, s);
      if (rc) return rc;
    }
    return 0;
  }
  const dim3 grid(segs, static_cast<unsigned>(gy));
  if (y_f32) dequant_mxfp4_kernel<float><<<grid, 256, 0, s>>>((const uint8_t*)q, (const uint8_t*)tiles, (float*)y, rows, K);
  else dequant_mxfp4_kernel<bf16><<<grid, 256, 0, s>>>((const uint8_t*)q, (const uint8_t*)tiles, (bf16*)y, rows, K);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // namespace dfb
