// Device helpers of the narrow formats: e2m1 and e4m3 conversion, e8m0 block scales and their tiled storage.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace dfb {

constexpr int kMxBlock = 32;
constexpr float kE4M3Top = 448.f;
constexpr float kMinScale = 0x1p-120f;      // floor of an fp32 scale: its reciprocal stays finite

// Two fp32 operations in one instruction, each rounded to nearest like its scalar form.
DFB_DEVICE unsigned long long as_u64(float2 a) { return *reinterpret_cast<unsigned long long*>(&a); }
DFB_DEVICE float2 as_f2(unsigned long long a) { return *reinterpret_cast<float2*>(&a); }
DFB_DEVICE float2 both(float a) { return make_float2(a, a); }
DFB_DEVICE float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(as_u64(a)), "l"(as_u64(b)));
  return as_f2(r);
}
DFB_DEVICE float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(as_u64(a)), "l"(as_u64(b)), "l"(as_u64(c)));
  return as_f2(r);
}
DFB_DEVICE float min_nan(float a, float b, float c) {      // the smallest one, or NaN if any is
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

DFB_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Byte of (row, block of 32) inside the tiled scales: tiles of 128 rows x 4 blocks, 512 bytes each, `tile_cols` tiles per
// row of tiles (an even number, so that two tiles = 256 elements of K are one aligned kilobyte).
DFB_DEVICE long long mx_scale_at(long long row, int block, int tile_cols) {
  return ((row >> 7) * tile_cols + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}
__host__ __device__ inline int mx_tile_cols(int K) { return 2 * ((K + 255) / 256); }

// Scale byte of a block from its largest magnitude: X = 2^(byte - 127) = 2^max(floor(log2 amax) - 2, -127), so that amax / X is
// in [4, 8) and saturates at e2m1's 6; 255 (NaN) when the block holds an infinity or a NaN.
DFB_DEVICE uint32_t mx_scale_byte(float amax) {
  const uint32_t e = (__float_as_uint(amax) >> 23) & 255u;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
DFB_DEVICE float mx_scale_inv(uint32_t byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }
DFB_DEVICE float mx_scale_value(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
}
// largest magnitude of eight values; NaN if one is (its exponent is that of an infinity)
DFB_DEVICE float mx_amax8(const float* f) {
  float a = fabsf(f[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) a = max_nan(a, fabsf(f[i]));
  return a;
}
// over the four (eight elements a lane) or two (sixteen) neighbouring lanes that hold a block
template <int LANES>
DFB_DEVICE float mx_amax_lanes(float a) {
  if constexpr (LANES == 4) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 2));
  return max_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));
}
// f *= 2^k in pairs, then the codes
DFB_DEVICE uint32_t mx_pack8(const float* f);
DFB_DEVICE uint32_t mx_scale_pack8(const float* f, float inv) {
  float g[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = mul2(make_float2(f[2 * i], f[2 * i + 1]), both(inv));
    g[2 * i] = v.x;
    g[2 * i + 1] = v.y;
  }
  return mx_pack8(g);
}

// eight e2m1 codes, element 0 in the lowest nibble; round to nearest even, saturating
DFB_DEVICE uint32_t mx_pack8(const float* f) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r) : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}
// the values of eight codes
DFB_DEVICE void mx_unpack8(uint32_t c, float* f) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(c));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

// Scale bytes of four neighbouring blocks, LANES lanes to a block, as the tile's word.
template <int LANES>
DFB_DEVICE uint32_t mx_scale_word(uint32_t byte) {
  uint32_t w = byte << (8 * ((threadIdx.x / LANES) & 3));
  w |= __shfl_xor_sync(0xffffffffu, w, LANES);
  return w | __shfl_xor_sync(0xffffffffu, w, 2 * LANES);
}

// 32 bytes in one access (aligned to them)
DFB_DEVICE void load32(const void* p, uint32_t* u) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]) : "l"(p) : "memory");
}
DFB_DEVICE void store32(void* p, const uint32_t* u) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               :: "l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]) : "memory");
}

// two e4m3 codes: a in the low byte
DFB_DEVICE uint32_t e4m3_pack2(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }
DFB_DEVICE float2 e4m3_unpack2(uint32_t p) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(p), __NV_E4M3);
  return __half22float2(__half2(h));
}

}  // namespace dfb
