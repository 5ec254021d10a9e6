// One AdamW step over many tensors in one launch, moments in fp32 or in 8 bits.
//
//   m' = b1 m + (1 - b1) g      v' = b2 v + (1 - b2) g^2      w -= lr (m' / bc1 / (sqrt(v' / bc2) + eps) + wd w)
//
// 8-bit moments hold m and r = sqrt(v) as e4m3 codes with one fp32 scale per 128 elements (amax / 448); the root halves the
// exponent range that v needs.  Rounding is stochastic: with b2 = 0.95 the root decays by 2.5 % per step at most, less than half
// of e4m3's 6 to 12 % spacing, so rounding to nearest would never let it fall again.  The random bits are a hash of (element
// index, seed).  A positive r keeps at least the smallest code.  The update itself uses the unrounded moments.
//
// The kernel moves 10 bytes per element with 8-bit moments (28 with fp32 moments and a master) and is bound by memory: a block
// takes 4096 consecutive elements of one tensor, a thread eight at a time, sixteen lanes share one scale.  Tensors travel as a
// table in the kernel's parameters (no copy, no device-side table that a captured graph would share); a block finds its tensor
// by bisection.
#include "lowbit.h"
#include "lowbit_common.cuh"

namespace dfb {
namespace {

constexpr int kChunk = 4096, kThreads = 256;

struct Entry {
  AdamTensor t;
  int first_block;
};
template <int NT>
struct Args {
  Entry e[NT];
  int count;
  AdamHyper h;
};

// 32-bit integer mixer: two rounds of xor-shift and multiply
DFB_DEVICE uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}

// e4m3-representable neighbour of y (|y| <= 448) below or above it in magnitude, with the odds of the distance: 16 random bits
// are added below the kept mantissa and the rest is cut off; adding 2^-6 first puts subnormal codes on one binade's grid.
// The result may exceed 448 by nothing (448's kept bits are its own, and the conversion saturates); the minimum keeps a NaN's
// bits from carrying into the sign.
template <bool SIGNED>
DFB_DEVICE float dither_e4m3(float y, uint32_t rnd16) {
  const float a = SIGNED ? fabsf(y) : y;
  const float base = a < 0x1p-6f ? 0x1p-6f : 0.f;
  const float t = __uint_as_float((min(__float_as_uint(a + base), 0x7ff00000u) + (rnd16 << 4)) & 0xfff00000u) - base;
  return SIGNED ? copysignf(t, y) : t;
}

template <typename T>
DFB_DEVICE void load8(const T* p, long long i, long long n, bool vec, float* f) {
  if (vec && i + 8 <= n) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p + i), b = *reinterpret_cast<const float4*>(p + i + 4);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
      unpack8(ld8(reinterpret_cast<const bf16*>(p) + i), f);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f[k] = 0.f;
      if (i + k < n) {
        if constexpr (sizeof(T) == 4) f[k] = p[i + k];
        else f[k] = bf2f(p[i + k]);
      }
    }
  }
}
template <typename T>
DFB_DEVICE void store8(T* p, long long i, long long n, bool vec, const float* f) {
  if (vec && i + 8 <= n) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p + i) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(p + i + 4) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      st8(reinterpret_cast<bf16*>(p) + i, pack8(f));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) {
        if constexpr (sizeof(T) == 4) p[i + k] = f[k];
        else p[i + k] = f2bf(f[k]);
      }
  }
}
DFB_DEVICE void load_codes(const uint8_t* p, long long i, long long n, bool vec, float scale, float* f) {
  uint2 q = make_uint2(0, 0);
  if (vec && i + 8 <= n) {
    q = *reinterpret_cast<const uint2*>(p + i);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) (k < 4 ? q.x : q.y) |= static_cast<uint32_t>(p[i + k]) << (8 * (k & 3));
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 v = e4m3_unpack2(((k < 2 ? q.x : q.y) >> (16 * (k & 1))) & 0xffffu);
    f[2 * k] = __fmul_rn(v.x, scale);
    f[2 * k + 1] = __fmul_rn(v.y, scale);
  }
}
DFB_DEVICE void store_codes(uint8_t* p, long long i, long long n, bool vec, const float* f) {
  uint2 q;
  q.x = e4m3_pack2(f[0], f[1]) | e4m3_pack2(f[2], f[3]) << 16;
  q.y = e4m3_pack2(f[4], f[5]) | e4m3_pack2(f[6], f[7]) << 16;
  if (vec && i + 8 <= n) {
    *reinterpret_cast<uint2*>(p + i) = q;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) p[i + k] = static_cast<uint8_t>((k < 4 ? q.x : q.y) >> (8 * (k & 3)));
  }
}
DFB_DEVICE float max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The products and sums in front of the stochastic rounding are kept unfused (__fmul_rn, __fadd_rn): a state then has the same
// code on every machine and in the plain-torch lane.
template <int WK, typename G, bool BITS8, int NT>
__global__ void __launch_bounds__(kThreads) adamw_multi_kernel(const __grid_constant__ Args<NT> a) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.e[mid].first_block <= static_cast<int>(blockIdx.x)) lo = mid;
    else hi = mid - 1;
  }
  const AdamTensor& t = a.e[lo].t;
  const AdamHyper& h = a.h;
  const long long n = t.n, base = static_cast<long long>(blockIdx.x - a.e[lo].first_block) * kChunk;
  const bool vec = ((reinterpret_cast<uintptr_t>(t.w) | reinterpret_cast<uintptr_t>(t.g) | reinterpret_cast<uintptr_t>(t.extra)) & 15) == 0 &&
                   ((reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) & (BITS8 ? 7 : 15)) == 0;
#pragma unroll 1
  for (int it = 0; it < kChunk / (kThreads * 8); ++it) {
    const long long i = base + (it * kThreads + threadIdx.x) * 8LL;
    if (base + it * kThreads * 8LL >= n) break;                    // uniform over the block: the shuffles below stay whole
    float g[8], m[8], r[8], w[8];
    load8(reinterpret_cast<const G*>(t.g), i, n, vec, g);
    if constexpr (WK == kAdamF32) load8(reinterpret_cast<const float*>(t.w), i, n, vec, w);
    else if constexpr (WK == kAdamMaster) load8(reinterpret_cast<const float*>(t.extra), i, n, vec, w);
    else load8(reinterpret_cast<const bf16*>(t.w), i, n, vec, w);
    if constexpr (WK == kAdamSplit) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < n) w[k] = __uint_as_float(__float_as_uint(w[k]) + static_cast<int32_t>(reinterpret_cast<const int16_t*>(t.extra)[i + k]));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) g[k] = __fmul_rn(g[k], h.gscale);
    if constexpr (BITS8) {
      const bool live = i < n;
      load_codes(reinterpret_cast<const uint8_t*>(t.m), i, n, vec, live ? t.m_scale[i >> 7] : 0.f, m);
      load_codes(reinterpret_cast<const uint8_t*>(t.v), i, n, vec, live ? t.v_scale[i >> 7] : 0.f, r);
      __syncwarp();                                                 // every lane has read its old scale
      float am = 0.f, ar = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m[k] = __fadd_rn(__fmul_rn(m[k], h.b1), __fmul_rn(g[k], h.c1));
        r[k] = __fsqrt_rn(__fadd_rn(__fmul_rn(__fmul_rn(r[k], r[k]), h.b2), __fmul_rn(__fmul_rn(g[k], g[k]), h.c2)));
        am = fmaxf(am, fabsf(m[k]));
        ar = fmaxf(ar, r[k]);
      }
      const float sm = fmaxf(__fmul_rn(max16(am), 1.f / kE4M3Top), kMinScale), sr = fmaxf(__fmul_rn(max16(ar), 1.f / kE4M3Top), kMinScale);
      if (live && (threadIdx.x & 15) == 0) {
        t.m_scale[i >> 7] = sm;
        t.v_scale[i >> 7] = sr;
      }
      const float im = __frcp_rn(sm), ir = __frcp_rn(sr);
      float qm[8], qr[8];
      const uint32_t salt = h.seed * 0x85ebca6bu + static_cast<uint32_t>(i >> 32) * 0xc2b2ae35u;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t rnd = mix32((static_cast<uint32_t>(i) + k) * 0x9e3779b9u + salt);
        qm[k] = dither_e4m3<true>(__fmul_rn(m[k], im), rnd & 0xffffu);
        const float y = __fmul_rn(r[k], ir);
        qr[k] = dither_e4m3<false>(y, rnd >> 16);
        if (y > 0.f) qr[k] = fmaxf(qr[k], 0x1p-9f);
      }
      store_codes(reinterpret_cast<uint8_t*>(t.m), i, n, vec, qm);
      store_codes(reinterpret_cast<uint8_t*>(t.v), i, n, vec, qr);
    } else {
      load8(reinterpret_cast<const float*>(t.m), i, n, vec, m);
      load8(reinterpret_cast<const float*>(t.v), i, n, vec, r);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m[k] = m[k] * h.b1 + g[k] * h.c1;
        r[k] = r[k] * h.b2 + g[k] * g[k] * h.c2;
      }
      store8(reinterpret_cast<float*>(t.m), i, n, vec, m);
      store8(reinterpret_cast<float*>(t.v), i, n, vec, r);
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = sqrtf(r[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] -= h.lr * (__fdividef(m[k] * h.inv_bc1, r[k] * h.inv_sqrt_bc2 + h.eps) + t.wd * w[k]);
    if constexpr (WK == kAdamF32) {
      store8(reinterpret_cast<float*>(t.w), i, n, vec, w);
    } else if constexpr (WK == kAdamSplit) {
      // the working weight is the master rounded half away from zero, which makes the cut an exact inverse of the join
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < n) {
          const uint32_t b = __float_as_uint(w[k]);
          reinterpret_cast<uint16_t*>(t.w)[i + k] = static_cast<uint16_t>((b + 0x8000u) >> 16);
          reinterpret_cast<uint16_t*>(t.extra)[i + k] = static_cast<uint16_t>(b);
        }
    } else {
      if constexpr (WK == kAdamMaster) store8(reinterpret_cast<float*>(t.extra), i, n, vec, w);
      store8(reinterpret_cast<bf16*>(t.w), i, n, vec, w);
    }
  }
}

template <int NT>
int launch(const AdamTensor* t, int count, int weights, bool g_f32, bool bits8, const AdamHyper& h, cudaStream_t s) {
  Args<NT> a;
  long long blocks = 0;
  for (int i = 0; i < count; ++i) {
    a.e[i].t = t[i];
    a.e[i].first_block = static_cast<int>(blocks);
    blocks += (t[i].n + kChunk - 1) / kChunk;
  }
  if (blocks > 0x7fffffffLL) return -3;
  a.count = count;
  a.h = h;
  auto go = [&](auto kernel) { kernel<<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(a); };
  auto by_bits = [&](auto wk, auto gt) {
    constexpr int WK = decltype(wk)::value;
    using G = decltype(gt);
    if (bits8) go(adamw_multi_kernel<WK, G, true, NT>);
    else go(adamw_multi_kernel<WK, G, false, NT>);
  };
  auto by_grad = [&](auto wk) {
    if (g_f32) by_bits(wk, float{});
    else by_bits(wk, bf16{});
  };
  switch (weights) {
    case kAdamBf16: by_grad(std::integral_constant<int, kAdamBf16>{}); break;
    case kAdamF32: by_grad(std::integral_constant<int, kAdamF32>{}); break;
    case kAdamMaster: by_grad(std::integral_constant<int, kAdamMaster>{}); break;
    case kAdamSplit: by_grad(std::integral_constant<int, kAdamSplit>{}); break;
    default: return -2;
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // namespace

// ``t`` holds no empty tensor.  A list longer than the table goes out in several launches.
int adamw_multi(const AdamTensor* t, int count, int weights, bool g_f32, bool bits8, const AdamHyper& h, cudaStream_t s) {
  constexpr int kMany = 256;
  for (int at = 0; at < count; at += kMany) {
    const int rc = launch<kMany>(t + at, count - at < kMany ? count - at : kMany, weights, g_f32, bits8, h, s);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace dfb
