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
// within 2^-23 of the root and the reciprocal; numbers below 2^-126 count as zero
DFB_DEVICE float root(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
DFB_DEVICE float recip(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
DFB_DEVICE float min_nan(float a, float b) {      // the smaller one, or NaN if either is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// e4m3-representable neighbour of y (|y| <= 448) below or above it in magnitude, with the odds of the distance: 16 random bits
// are added below the kept mantissa and the rest is cut off.  448 cannot be left upwards (its kept bits are its own).
// This form is for 2^-6 <= |y|, where the codes are normal numbers; the sign bit rides along.
DFB_DEVICE float dither_normal(float y, uint32_t rnd16) { return __uint_as_float((__float_as_uint(y) + (rnd16 << 4)) & 0xfff00000u); }
// Any y: adding 2^-6 first puts subnormal codes on one binade's grid; the minimum keeps a NaN's bits from carrying.
DFB_DEVICE float dither_any(float y, uint32_t rnd16) {
  const float a = fabsf(y);
  const float base = a < 0x1p-6f ? 0x1p-6f : 0.f;
  const float t = __uint_as_float((min(__float_as_uint(a + base), 0x7ff00000u) + (rnd16 << 4)) & 0xfff00000u) - base;
  return copysignf(t, y);
}

// Eight elements as they lie in memory; a load that may not be whole (FULL false) goes element by element, zeros past n.  The two
// forms are chosen once per block, so that a thread's loads stand one behind the other without a branch between.
template <int BYTES>
struct alignas(BYTES >= 2 ? 16 : 8) Raw { uint32_t u[2 * BYTES]; };      // 8 elements of BYTES bytes
template <int BYTES, bool FULL>
DFB_DEVICE Raw<BYTES> load(const void* p, long long i, long long n) {
  Raw<BYTES> r;
  if constexpr (FULL) {
    r = *reinterpret_cast<const Raw<BYTES>*>(static_cast<const char*>(p) + i * BYTES);
  } else {
#pragma unroll
    for (int k = 0; k < 2 * BYTES; ++k) r.u[k] = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) {
        if constexpr (BYTES == 4) r.u[k] = static_cast<const uint32_t*>(p)[i + k];
        else if constexpr (BYTES == 2) r.u[k >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i + k]) << (16 * (k & 1));
        else r.u[k >> 2] |= static_cast<uint32_t>(static_cast<const uint8_t*>(p)[i + k]) << (8 * (k & 3));
      }
  }
  return r;
}
template <int BYTES, bool FULL>
DFB_DEVICE void store(void* p, long long i, long long n, const Raw<BYTES>& r) {
  if constexpr (FULL) {
    *reinterpret_cast<Raw<BYTES>*>(static_cast<char*>(p) + i * BYTES) = r;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) {
        if constexpr (BYTES == 4) static_cast<uint32_t*>(p)[i + k] = r.u[k];
        else if constexpr (BYTES == 2) static_cast<uint16_t*>(p)[i + k] = static_cast<uint16_t>(r.u[k >> 1] >> (16 * (k & 1)));
        else static_cast<uint8_t*>(p)[i + k] = static_cast<uint8_t>(r.u[k >> 2] >> (8 * (k & 3)));
      }
  }
}
DFB_DEVICE float2 pair(const Raw<4>& r, int j) { return make_float2(__uint_as_float(r.u[2 * j]), __uint_as_float(r.u[2 * j + 1])); }
DFB_DEVICE float2 pair(const Raw<2>& r, int j) { return make_float2(__uint_as_float(r.u[j] << 16), __uint_as_float(r.u[j] & 0xffff0000u)); }
DFB_DEVICE float2 pair(const Raw<1>& r, int j) { return e4m3_unpack2((r.u[j >> 1] >> (16 * (j & 1))) & 0xffffu); }
DFB_DEVICE void set_pair(Raw<4>& r, int j, float2 v) { r.u[2 * j] = __float_as_uint(v.x); r.u[2 * j + 1] = __float_as_uint(v.y); }
DFB_DEVICE void set_pair(Raw<2>& r, int j, float2 v) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
  r.u[j] = *reinterpret_cast<const uint32_t*>(&b);
}
DFB_DEVICE float max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <int WK, int GB, bool BITS8>
struct Loaded {
  Raw<WK == kAdamF32 || WK == kAdamMaster ? 4 : 2> w;
  Raw<2> lo;                               // split master only
  Raw<GB> g;
  Raw<BITS8 ? 1 : 4> m, v;
  float sm, sv;
};

// Eight elements of one thread.
template <int WK, int GB, bool BITS8, bool FULL>
DFB_DEVICE void step8(const AdamTensor& t, const AdamHyper& h, Loaded<WK, GB, BITS8>& in, long long i) {
  const long long n = t.n;
  float2 w[4], m[4], r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w[j] = pair(in.w, j);
    if constexpr (WK == kAdamSplit) {
      w[j].x = __uint_as_float(__float_as_uint(w[j].x) + static_cast<int32_t>(static_cast<int16_t>(in.lo.u[j] & 0xffffu)));
      w[j].y = __uint_as_float(__float_as_uint(w[j].y) + static_cast<int32_t>(static_cast<int16_t>(in.lo.u[j] >> 16)));
    }
  }
  const float2 b1 = both(h.b1), c1 = both(h.c1), b2 = both(h.b2), c2 = both(h.c2), gs = both(h.gscale);
  if constexpr (BITS8) {
    float am = 0.f, ar = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 g = mul2(pair(in.g, j), gs), r0 = mul2(pair(in.v, j), both(in.sv));
      m[j] = fma2(mul2(pair(in.m, j), both(in.sm)), b1, mul2(g, c1));
      const float2 v = fma2(mul2(r0, r0), b2, mul2(mul2(g, g), c2));
      r[j] = make_float2(root(v.x), root(v.y));
      am = fmaxf(am, fmaxf(fabsf(m[j].x), fabsf(m[j].y)));
      ar = fmaxf(ar, fmaxf(r[j].x, r[j].y));
    }
    const float sm = fmaxf(__fmul_rn(max16(am), 1.f / kE4M3Top), kMinScale), sr = fmaxf(__fmul_rn(max16(ar), 1.f / kE4M3Top), kMinScale);
    if ((FULL || i < n) && (threadIdx.x & 15) == 0) {
      t.m_scale[i >> 7] = sm;
      t.v_scale[i >> 7] = sr;
    }
    const float2 im = both(__frcp_rn(sm)), ir = both(__frcp_rn(sr));
    float2 y[4], z[4];
    float low = 0x1p-6f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      y[j] = mul2(m[j], im);
      z[j] = mul2(r[j], ir);
      low = min_nan(min_nan(low, min_nan(fabsf(y[j].x), fabsf(y[j].y))), min_nan(z[j].x, z[j].y));
    }
    uint32_t x = static_cast<uint32_t>(i) * 0x9e3779b9u + h.seed * 0x85ebca6bu + static_cast<uint32_t>(i >> 32) * 0xc2b2ae35u;
    // every value of the warp a normal code: almost always, where no moment is zero
    if (__all_sync(0xffffffffu, low == 0x1p-6f)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t ra = mix32(x), rb = mix32(x + 0x9e3779b9u);
        x += 2 * 0x9e3779b9u;
        y[j] = make_float2(dither_normal(y[j].x, ra & 0xffffu), dither_normal(y[j].y, rb & 0xffffu));
        z[j] = make_float2(dither_normal(z[j].x, ra >> 16), dither_normal(z[j].y, rb >> 16));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t ra = mix32(x), rb = mix32(x + 0x9e3779b9u);
        x += 2 * 0x9e3779b9u;
        y[j] = make_float2(dither_any(y[j].x, ra & 0xffffu), dither_any(y[j].y, rb & 0xffffu));
        const float2 q = make_float2(dither_any(z[j].x, ra >> 16), dither_any(z[j].y, rb >> 16));
        // a root above zero keeps at least the smallest code
        z[j] = make_float2(z[j].x > 0.f ? fmaxf(q.x, 0x1p-9f) : q.x, z[j].y > 0.f ? fmaxf(q.y, 0x1p-9f) : q.y);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      in.m.u[k] = e4m3_pack2(y[2 * k].x, y[2 * k].y) | e4m3_pack2(y[2 * k + 1].x, y[2 * k + 1].y) << 16;
      in.v.u[k] = e4m3_pack2(z[2 * k].x, z[2 * k].y) | e4m3_pack2(z[2 * k + 1].x, z[2 * k + 1].y) << 16;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 g = mul2(pair(in.g, j), gs);
      m[j] = fma2(pair(in.m, j), b1, mul2(g, c1));
      r[j] = fma2(pair(in.v, j), b2, mul2(mul2(g, g), c2));
      set_pair(in.m, j, m[j]);
      set_pair(in.v, j, r[j]);
      r[j] = make_float2(sqrtf(r[j].x), sqrtf(r[j].y));
    }
  }
  store<BITS8 ? 1 : 4, FULL>(t.m, i, n, in.m);
  store<BITS8 ? 1 : 4, FULL>(t.v, i, n, in.v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 den = fma2(r[j], both(h.inv_sqrt_bc2), both(h.eps));
    const float2 up = mul2(mul2(m[j], both(h.inv_bc1)), make_float2(recip(den.x), recip(den.y)));
    w[j] = fma2(both(-h.lr), fma2(both(t.wd), w[j], up), w[j]);
  }
  if constexpr (WK == kAdamSplit) {
    // the working weight is the master rounded half away from zero, which makes the cut an exact inverse of the join
    Raw<2> hi;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = __float_as_uint(w[j].x), b = __float_as_uint(w[j].y);
      hi.u[j] = ((a + 0x8000u) >> 16) | ((b + 0x8000u) & 0xffff0000u);
      in.lo.u[j] = (a & 0xffffu) | (b << 16);
    }
    store<2, FULL>(t.w, i, n, hi);
    store<2, FULL>(t.extra, i, n, in.lo);
  } else if constexpr (WK == kAdamF32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) set_pair(in.w, j, w[j]);
    store<4, FULL>(t.w, i, n, in.w);
  } else {
    Raw<2> out;
#pragma unroll
    for (int j = 0; j < 4; ++j) set_pair(out, j, w[j]);
    store<2, FULL>(t.w, i, n, out);
    if constexpr (WK == kAdamMaster) {
#pragma unroll
      for (int j = 0; j < 4; ++j) set_pair(in.w, j, w[j]);
      store<4, FULL>(t.extra, i, n, in.w);
    }
  }
}

// A chunk of one tensor.  With 8-bit moments the loads of both of a thread's groups are issued before the first is computed on.
template <int WK, int GB, bool BITS8, bool FULL>
DFB_DEVICE void chunk(const AdamTensor& t, const AdamHyper& h, long long base) {
  constexpr int kGroups = kChunk / (kThreads * 8), kAhead = BITS8 && FULL ? kGroups : 1;
  constexpr int WB = WK == kAdamF32 || WK == kAdamMaster ? 4 : 2, SB = BITS8 ? 1 : 4;
  const long long n = t.n;
#pragma unroll 1
  for (int it = 0; it < kGroups; it += kAhead) {
    Loaded<WK, GB, BITS8> in[kAhead];
    const long long i0 = base + (it * kThreads + threadIdx.x) * 8LL;
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const long long i = i0 + a * kThreads * 8LL;
      in[a].w = load<WB, FULL>(WK == kAdamMaster ? t.extra : t.w, i, n);
      if constexpr (WK == kAdamSplit) in[a].lo = load<2, FULL>(t.extra, i, n);
      in[a].g = load<GB, FULL>(t.g, i, n);
      in[a].m = load<SB, FULL>(t.m, i, n);
      in[a].v = load<SB, FULL>(t.v, i, n);
      if constexpr (BITS8) {
        in[a].sm = FULL || i < n ? t.m_scale[i >> 7] : 0.f;
        in[a].sv = FULL || i < n ? t.v_scale[i >> 7] : 0.f;
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      // uniform over the block: the shuffles stay whole.  The scales of a block of 128 are read and written by one half warp, in
      // that order (the shuffles stand between).
      if (!FULL && base + (it + a) * kThreads * 8LL >= n) return;
      step8<WK, GB, BITS8, FULL>(t, h, in[a], i0 + a * kThreads * 8LL);
    }
  }
}

template <int WK, int GB, bool BITS8, int NT>
__global__ void __launch_bounds__(kThreads, BITS8 ? 3 : 4) adamw_multi_kernel(const __grid_constant__ Args<NT> a) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.e[mid].first_block <= static_cast<int>(blockIdx.x)) lo = mid;
    else hi = mid - 1;
  }
  const AdamTensor& t = a.e[lo].t;
  const long long base = static_cast<long long>(blockIdx.x - a.e[lo].first_block) * kChunk;
  const bool vec = ((reinterpret_cast<uintptr_t>(t.w) | reinterpret_cast<uintptr_t>(t.g) | reinterpret_cast<uintptr_t>(t.extra)) & 15) == 0 &&
                   ((reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) & (BITS8 ? 7 : 15)) == 0;
  if (vec && base + kChunk <= t.n) chunk<WK, GB, BITS8, true>(t, a.h, base);
  else chunk<WK, GB, BITS8, false>(t, a.h, base);
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
  auto by_grad = [&](auto wk) {
    constexpr int WK = decltype(wk)::value;
    if (g_f32) bits8 ? go(adamw_multi_kernel<WK, 4, true, NT>) : go(adamw_multi_kernel<WK, 4, false, NT>);
    else bits8 ? go(adamw_multi_kernel<WK, 2, true, NT>) : go(adamw_multi_kernel<WK, 2, false, NT>);
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
  // a table of 256 is 20 KB of kernel parameters, one of 24 is 2 KB: a layer's fields fit the small one
  constexpr int kFew = 24, kMany = 256;
  if (count <= kFew) return launch<kFew>(t, count, weights, g_f32, bits8, h, s);
  for (int at = 0; at < count; at += kMany) {
    const int rc = launch<kMany>(t + at, count - at < kMany ? count - at : kMany, weights, g_f32, bits8, h, s);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace dfb
