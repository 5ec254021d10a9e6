// One AdamW step over many tensors in one launch, moments in fp32 or in 8 bits.
//
//   m' = b1 m + (1 - b1) g      v' = b2 v + (1 - b2) g^2      w -= lr (m' / bc1 / (sqrt(v' / bc2) + eps) + wd w)
//
// 8-bit moments hold m and r = sqrt(v) as e4m3 codes with one fp32 scale per 128 elements (amax / 448); the root halves the
// exponent range that v needs.  Rounding is stochastic: with b2 = 0.95 the root decays by 2.5 % per step at most, less than half
// of e4m3's 6 to 12 % spacing, so rounding to nearest would never let it fall again.  The random bits are a hash of (element
// index, seed).  A positive r keeps at least the smallest code.  The update itself uses the unrounded moments.
//
// The kernel moves 10 bytes per element with 8-bit moments (28 with fp32 moments and a master) and is bound by memory: 8 bits 378 us
// at 218M parameters, 0.89 of the copy rate with the arithmetic close behind (47 instructions an element, issue slots 73 % busy; 6 us of
// it for roots that are right at every size); 32 bits 175 us at 42M, the copy rate.  A block takes consecutive elements of one tensor, a
// thread eight or (8-bit moments) sixteen of them, so that eight lanes share a scale.  Tensors travel as a table in the kernel's
// parameters (no copy, no device-side table that a captured graph would share); a block finds its tensor by bisection.
#include "lowbit.h"
#include "lowbit_common.cuh"

namespace dfb {
namespace {

// Elements of a block with 8-bit moments, for lists of at least twice what stays resident (39M); below, and with fp32 moments,
// a block takes one group of its threads (512 and 2048 elements).  8 bits, 8192 / 512 elements: 1M 15 / 4 us, 21M 52 / 47 us,
// 42M 86 / 90 us; fp32, 4096 / 2048: 1M 5.0 / 4.7 us, 42M 138 / 135 us.
constexpr int kChunk = 8192;
// Threads of a block, and blocks per SM.  The 8-bit form at 176M parameters, sixteen elements a thread, the next group on its way:
// one warp a block, 16 blocks 304 us (copy rate: 272), 18 blocks 363; 64 threads, 8 blocks 303 to 309 us; without the loads ahead 330
// at best; eight elements a thread 379.
template <bool BITS8>
constexpr int kThreads = BITS8 ? 32 : 256;
template <bool BITS8>
constexpr int kBlocks = BITS8 ? 16 : 4;

struct Entry {
  AdamTensor t;
  int first_block;
};
template <int NT>
struct Args {
  Entry e[NT];
  int count, chunk;
  AdamHyper h;
};

// 32-bit integer mixer: two rounds of xor-shift and multiply; shifts and factors from C. Wellons, "Prospecting for Hash Functions"
// (2018), found there by a search for the least bias between input and output bits
DFB_DEVICE uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}

// Square roots, rounded to nearest: Heron's step on an approximate reciprocal root with the residual from a fused product
// (Markstein 1990, "Computation of elementary functions on the IBM RISC System/6000 processor").  For 2^-90 <= x < infinity, where
// the residual x - s^2 is exact (its last bit is worth x 2^-48 or more).  Below, down to the smallest normal number, a last place may be
// off, but the result is below 2^-45; of zero, a subnormal number, infinity and NaN the result is NaN.
DFB_DEVICE float2 root2(float2 x) {
  float2 y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(x.x));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(x.y));
  const float2 s = mul2(x, y);
  const float2 e = fma2(make_float2(-s.x, -s.y), s, x);
  return fma2(e, mul2(y, both(0.5f)), s);
}
// within 2^-23 of the reciprocal
DFB_DEVICE float recip(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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

// A thread's elements as they lie in memory.  How they are fetched is chosen once per block, so that the loads stand one behind
// the other without a branch between: 32 bytes at a time with 8-bit moments where every operand of the tensor starts on 32
// (176M parameters 304 us; by 16 bytes 309 to 319; with fp32 moments both at the copy rate), 16 bytes where on 16, else element by
// element with zeros past n.
enum Fetch { kElements, k16Bytes, k32Bytes };
template <int BYTES, int E>
struct alignas(BYTES * E >= 16 ? 16 : 8) Raw { uint32_t u[BYTES * E / 4]; };      // E elements of BYTES bytes
template <int BYTES, int E, int HOW>
DFB_DEVICE Raw<BYTES, E> load(const void* p, long long i, long long n) {
  Raw<BYTES, E> r;
  if constexpr (HOW == k32Bytes && BYTES * E % 32 == 0) {
#pragma unroll
    for (int k = 0; k < BYTES * E / 32; ++k) load32(static_cast<const char*>(p) + i * BYTES + k * 32, r.u + k * 8);
  } else if constexpr (HOW != kElements) {
    r = *reinterpret_cast<const Raw<BYTES, E>*>(static_cast<const char*>(p) + i * BYTES);
  } else {
#pragma unroll
    for (int k = 0; k < BYTES * E / 4; ++k) r.u[k] = 0;
#pragma unroll
    for (int k = 0; k < E; ++k)
      if (i + k < n) {
        if constexpr (BYTES == 4) r.u[k] = static_cast<const uint32_t*>(p)[i + k];
        else if constexpr (BYTES == 2) r.u[k >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i + k]) << (16 * (k & 1));
        else r.u[k >> 2] |= static_cast<uint32_t>(static_cast<const uint8_t*>(p)[i + k]) << (8 * (k & 3));
      }
  }
  return r;
}
template <int BYTES, int E, int HOW>
DFB_DEVICE void store(void* p, long long i, long long n, const Raw<BYTES, E>& r) {
  if constexpr (HOW == k32Bytes && BYTES * E % 32 == 0) {
#pragma unroll
    for (int k = 0; k < BYTES * E / 32; ++k) store32(static_cast<char*>(p) + i * BYTES + k * 32, r.u + k * 8);
  } else if constexpr (HOW != kElements) {
    *reinterpret_cast<Raw<BYTES, E>*>(static_cast<char*>(p) + i * BYTES) = r;
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k)
      if (i + k < n) {
        if constexpr (BYTES == 4) static_cast<uint32_t*>(p)[i + k] = r.u[k];
        else if constexpr (BYTES == 2) static_cast<uint16_t*>(p)[i + k] = static_cast<uint16_t>(r.u[k >> 1] >> (16 * (k & 1)));
        else static_cast<uint8_t*>(p)[i + k] = static_cast<uint8_t>(r.u[k >> 2] >> (8 * (k & 3)));
      }
  }
}
template <int E>
DFB_DEVICE float2 pair(const Raw<4, E>& r, int j) { return make_float2(__uint_as_float(r.u[2 * j]), __uint_as_float(r.u[2 * j + 1])); }
template <int E>
DFB_DEVICE float2 pair(const Raw<2, E>& r, int j) { return make_float2(__uint_as_float(r.u[j] << 16), __uint_as_float(r.u[j] & 0xffff0000u)); }
template <int E>
DFB_DEVICE float2 pair(const Raw<1, E>& r, int j) { return e4m3_unpack2((r.u[j >> 1] >> (16 * (j & 1))) & 0xffffu); }
template <int E>
DFB_DEVICE void set_pair(Raw<4, E>& r, int j, float2 v) { r.u[2 * j] = __float_as_uint(v.x); r.u[2 * j + 1] = __float_as_uint(v.y); }
template <int E>
DFB_DEVICE void set_pair(Raw<2, E>& r, int j, float2 v) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
  r.u[j] = *reinterpret_cast<const uint32_t*>(&b);
}
// over the lanes that share a scale: 128 elements
template <int LANES>
DFB_DEVICE float max_lanes(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// elements per thread: sixteen with 8-bit moments (one 16-byte load of codes, half the shuffles per element), else eight
template <bool BITS8>
constexpr int kPer = BITS8 ? 16 : 8;

template <int WK, int GB, bool BITS8>
struct Loaded {
  static constexpr int E = kPer<BITS8>;
  Raw<WK == kAdamF32 || WK == kAdamMaster ? 4 : 2, E> w;
  Raw<2, E> lo;                            // split master only
  Raw<GB, E> g;
  Raw<BITS8 ? 1 : 4, E> m, v;
  float sm, sv;
};

// The elements of one thread.  Products and sums in front of the 8-bit rounding are rounded one by one (a sum is a fused product
// with a factor of one that the compiler does not know), so a state has the same codes here and in the plain-torch lane.
template <int WK, int GB, bool BITS8, int HOW>
DFB_DEVICE void step(const AdamTensor& t, const AdamHyper& h, Loaded<WK, GB, BITS8>& in, long long i) {
  constexpr int E = kPer<BITS8>, P = E / 2;
  const long long n = t.n;
  float2 w[P], m[P], r[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    w[j] = pair(in.w, j);
    if constexpr (WK == kAdamSplit) {
      w[j].x = __uint_as_float(__float_as_uint(w[j].x) + static_cast<int32_t>(static_cast<int16_t>(in.lo.u[j] & 0xffffu)));
      w[j].y = __uint_as_float(__float_as_uint(w[j].y) + static_cast<int32_t>(static_cast<int16_t>(in.lo.u[j] >> 16)));
    }
  }
  const float2 one = both(h.one);
  const float2 b1 = both(h.b1), c1 = both(h.c1), b2 = both(h.b2), c2 = both(h.c2), gs = both(h.gscale);
  if constexpr (BITS8) {
    float am = 0.f, ar = 0.f, least = INFINITY;
    auto square = [&](float2 g, int j) {
      const float2 r0 = mul2(pair(in.v, j), both(in.sv));
      return fma2(mul2(mul2(r0, r0), b2), one, mul2(mul2(g, g), c2));
    };
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const float2 g = mul2(pair(in.g, j), gs);
      m[j] = fma2(mul2(mul2(pair(in.m, j), both(in.sm)), b1), one, mul2(g, c1));
      r[j] = root2(square(g, j));
      am = fmaxf(am, fmaxf(fabsf(m[j].x), fabsf(m[j].y)));
      ar = fmaxf(ar, fmaxf(r[j].x, r[j].y));
      least = min_nan(least, r[j].x, r[j].y);
    }
    if (!(least >= 0x1p-45f) && (HOW != kElements || i < n)) {      // some square is none that root2 takes: this thread's roots again
      ar = 0.f;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float2 x = square(mul2(pair(in.g, j), gs), j);
        r[j] = make_float2(sqrtf(x.x), sqrtf(x.y));
        ar = fmaxf(ar, fmaxf(r[j].x, r[j].y));
      }
    }
    const float sm = fmaxf(__fmul_rn(max_lanes<128 / E>(am), 1.f / kE4M3Top), kMinScale);
    const float sr = fmaxf(__fmul_rn(max_lanes<128 / E>(ar), 1.f / kE4M3Top), kMinScale);
    if ((HOW != kElements || i < n) && (threadIdx.x & (128 / E - 1)) == 0) {
      t.m_scale[i >> 7] = sm;
      t.v_scale[i >> 7] = sr;
    }
    const float2 im = both(__frcp_rn(sm)), ir = both(__frcp_rn(sr));
    float2 y[P], z[P];
    float low = 0x1p-6f;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      y[j] = mul2(m[j], im);
      z[j] = mul2(r[j], ir);
      low = min_nan(min_nan(low, fabsf(y[j].x), fabsf(y[j].y)), z[j].x, z[j].y);
    }
    uint32_t x = static_cast<uint32_t>(i) * 0x9e3779b9u + t.seed * 0x85ebca6bu + static_cast<uint32_t>(i >> 32) * 0xc2b2ae35u;
    // every value of the warp a normal code: almost always, where no moment is zero
    if (__all_sync(0xffffffffu, low == 0x1p-6f)) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const uint32_t ra = mix32(x), rb = mix32(x + 0x9e3779b9u);
        x += 2 * 0x9e3779b9u;
        y[j] = make_float2(dither_normal(y[j].x, ra & 0xffffu), dither_normal(y[j].y, rb & 0xffffu));
        z[j] = make_float2(dither_normal(z[j].x, ra >> 16), dither_normal(z[j].y, rb >> 16));
      }
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const uint32_t ra = mix32(x), rb = mix32(x + 0x9e3779b9u);
        x += 2 * 0x9e3779b9u;
        y[j] = make_float2(dither_any(y[j].x, ra & 0xffffu), dither_any(y[j].y, rb & 0xffffu));
        const float2 q = make_float2(dither_any(z[j].x, ra >> 16), dither_any(z[j].y, rb >> 16));
        // a root above zero keeps at least the smallest code
        z[j] = make_float2(z[j].x > 0.f ? fmaxf(q.x, 0x1p-9f) : q.x, z[j].y > 0.f ? fmaxf(q.y, 0x1p-9f) : q.y);
      }
    }
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      in.m.u[k] = e4m3_pack2(y[2 * k].x, y[2 * k].y) | e4m3_pack2(y[2 * k + 1].x, y[2 * k + 1].y) << 16;
      in.v.u[k] = e4m3_pack2(z[2 * k].x, z[2 * k].y) | e4m3_pack2(z[2 * k + 1].x, z[2 * k + 1].y) << 16;
    }
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const float2 g = mul2(pair(in.g, j), gs);
      m[j] = fma2(pair(in.m, j), b1, mul2(g, c1));
      r[j] = fma2(pair(in.v, j), b2, mul2(mul2(g, g), c2));
      set_pair(in.m, j, m[j]);
      set_pair(in.v, j, r[j]);
      r[j] = make_float2(sqrtf(r[j].x), sqrtf(r[j].y));
    }
  }
  store<BITS8 ? 1 : 4, E, HOW>(t.m, i, n, in.m);
  store<BITS8 ? 1 : 4, E, HOW>(t.v, i, n, in.v);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const float2 den = fma2(r[j], both(h.inv_sqrt_bc2), both(h.eps));
    const float2 up = mul2(mul2(m[j], both(h.inv_bc1)), make_float2(recip(den.x), recip(den.y)));
    w[j] = fma2(both(-h.lr), fma2(both(t.wd), w[j], up), w[j]);
  }
  if constexpr (WK == kAdamSplit) {
    // the working weight is the master rounded half away from zero, which makes the cut an exact inverse of the join
    Raw<2, E> hi;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const uint32_t a = __float_as_uint(w[j].x), b = __float_as_uint(w[j].y);
      hi.u[j] = ((a + 0x8000u) >> 16) | ((b + 0x8000u) & 0xffff0000u);
      in.lo.u[j] = (a & 0xffffu) | (b << 16);
    }
    store<2, E, HOW>(t.w, i, n, hi);
    store<2, E, HOW>(t.extra, i, n, in.lo);
  } else if constexpr (WK == kAdamF32) {
#pragma unroll
    for (int j = 0; j < P; ++j) set_pair(in.w, j, w[j]);
    store<4, E, HOW>(t.w, i, n, in.w);
  } else {
    Raw<2, E> out;
#pragma unroll
    for (int j = 0; j < P; ++j) set_pair(out, j, w[j]);
    store<2, E, HOW>(t.w, i, n, out);
    if constexpr (WK == kAdamMaster) {
#pragma unroll
      for (int j = 0; j < P; ++j) set_pair(in.w, j, w[j]);
      store<4, E, HOW>(t.extra, i, n, in.w);
    }
  }
}

template <int WK, int GB, bool BITS8, int HOW>
DFB_DEVICE Loaded<WK, GB, BITS8> fetch(const AdamTensor& t, long long i) {
  constexpr int E = kPer<BITS8>, WB = WK == kAdamF32 || WK == kAdamMaster ? 4 : 2, SB = BITS8 ? 1 : 4;
  Loaded<WK, GB, BITS8> in;
  in.w = load<WB, E, HOW>(WK == kAdamMaster ? t.extra : t.w, i, t.n);
  if constexpr (WK == kAdamSplit) in.lo = load<2, E, HOW>(t.extra, i, t.n);
  in.g = load<GB, E, HOW>(t.g, i, t.n);
  in.m = load<SB, E, HOW>(t.m, i, t.n);
  in.v = load<SB, E, HOW>(t.v, i, t.n);
  if constexpr (BITS8) {                     // read here, written behind the shuffles of the lanes that share it
    in.sm = HOW != kElements || i < t.n ? t.m_scale[i >> 7] : 0.f;
    in.sv = HOW != kElements || i < t.n ? t.v_scale[i >> 7] : 0.f;
  }
  return in;
}

// A chunk of one tensor.  With 8-bit moments a thread's next group is on its way while it computes on this one; with fp32 moments
// the registers for that cost more than it gains (42M parameters with a master: 249 us with, 176 us without).
template <int WK, int GB, bool BITS8, int HOW>
DFB_DEVICE void chunk(const AdamTensor& t, const AdamHyper& h, long long base, int elems) {
  constexpr int kGroup = kThreads<BITS8> * kPer<BITS8>;
  long long i = base + threadIdx.x * kPer<BITS8>;
  if constexpr (HOW != kElements && BITS8) {
    Loaded<WK, GB, BITS8> in = fetch<WK, GB, BITS8, HOW>(t, i);
#pragma unroll 1
    for (int left = elems - kGroup; left > 0; left -= kGroup) {
      const Loaded<WK, GB, BITS8> next = fetch<WK, GB, BITS8, HOW>(t, i + kGroup);
      step<WK, GB, BITS8, HOW>(t, h, in, i);
      in = next;
      i += kGroup;
    }
    step<WK, GB, BITS8, HOW>(t, h, in, i);
  } else {
#pragma unroll 1
    for (int at = 0; at < elems && (HOW != kElements || base + at < t.n); at += kGroup, i += kGroup) {      // uniform over the block
      Loaded<WK, GB, BITS8> in = fetch<WK, GB, BITS8, HOW>(t, i);
      step<WK, GB, BITS8, HOW>(t, h, in, i);
    }
  }
}

template <int WK, int GB, bool BITS8, int NT>
__global__ void __launch_bounds__(kThreads<BITS8>, kBlocks<BITS8>) adamw_multi_kernel(const __grid_constant__ Args<NT> a) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.e[mid].first_block <= static_cast<int>(blockIdx.x)) lo = mid;
    else hi = mid - 1;
  }
  const AdamTensor& t = a.e[lo].t;
  const long long base = static_cast<long long>(blockIdx.x - a.e[lo].first_block) * a.chunk;
  // the codes of 8-bit moments are 16 bytes a thread at most
  const uintptr_t wide = reinterpret_cast<uintptr_t>(t.w) | reinterpret_cast<uintptr_t>(t.g) | reinterpret_cast<uintptr_t>(t.extra);
  const uintptr_t state = reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v);
  const bool whole = base + a.chunk <= t.n && (state & 15) == 0;
  if constexpr (BITS8) {
    if (whole && (wide & 31) == 0) {
      chunk<WK, GB, BITS8, k32Bytes>(t, a.h, base, a.chunk);
      return;
    }
  }
  if (whole && (wide & 15) == 0) chunk<WK, GB, BITS8, k16Bytes>(t, a.h, base, a.chunk);
  else chunk<WK, GB, BITS8, kElements>(t, a.h, base, a.chunk);
}

template <int NT>
int launch(const AdamTensor* t, int count, int weights, bool g_f32, bool bits8, const AdamHyper& h, int num_sms, cudaStream_t s) {
  Args<NT> a;
  long long total = 0, blocks = 0;
  for (int i = 0; i < count; ++i) total += t[i].n;
  const int group = bits8 ? kThreads<true> * kPer<true> : kThreads<false> * kPer<false>;
  a.chunk = bits8 && total >= 2LL * num_sms * kBlocks<true> * kChunk ? kChunk : group;
  for (int i = 0; i < count; ++i) {
    a.e[i].t = t[i];
    a.e[i].first_block = static_cast<int>(blocks);
    blocks += (t[i].n + a.chunk - 1) / a.chunk;
  }
  if (blocks > 0x7fffffffLL) return -3;
  a.count = count;
  a.h = h;
  auto go = [&](auto kernel) { kernel<<<static_cast<unsigned>(blocks), bits8 ? kThreads<true> : kThreads<false>, 0, s>>>(a); };
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
int adamw_multi(const AdamTensor* t, int count, int weights, bool g_f32, bool bits8, const AdamHyper& h, int num_sms, cudaStream_t s) {
  // A table of 256 is 20 KB of kernel parameters, one of 24 is 2 KB, and a layer's fields fit it: 4.0 us to issue instead of 6.8.
  constexpr int kFew = 24, kMany = 256;
  if (count <= kFew) return launch<kFew>(t, count, weights, g_f32, bits8, h, num_sms, s);
  for (int at = 0; at < count; at += kMany) {
    const int rc = launch<kMany>(t + at, count - at < kMany ? count - at : kMany, weights, g_f32, bits8, h, num_sms, s);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace dfb
