// RMS norm with the residual's addition whose output leaves in a narrow format.
//
//   h = bf16(x + residual)      rstd = (mean h^2 + eps)^(-1/2)      y = h rstd w  (fp32)
//   fp8:    s = max(amax |y| / 448, 2^-120) per row (1 for a row of zeros), q = e4m3(y (1 / s))
//   mxfp4:  blocks of 32 columns, X = 2^(floor(log2 amax) - 2), q = e2m1(y / X)
//
// The statistics are those of the rounded h, the tensor that the backward pass reads again.  Bound by memory: a row is read once
// into registers (up to 16384 columns) and stays there through both reductions.  16384 x 4096 to fp8 with the residual: 71 us for
// 470 MB, the copy rate; 8191 x 2048 to 4 bits 13 us, of which about four are the launch's ramp.
#include "lowbit.h"
#include "lowbit_common.cuh"

namespace dfb {
namespace {

// max / sum over the T threads of a row; every thread gets the result.  `part` holds one value per warp of the row and is not
// written again before every thread has read it, so a single barrier is enough.
template <int T, bool MAX>
DFB_DEVICE float row_reduce(float v, float* part) {
  v = MAX ? warp_max(v) : warp_sum(v);
  if constexpr (T > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < T / 32; ++i) v = MAX ? fmaxf(v, part[i]) : v + part[i];
  }
  return v;
}

// scale words past the rows and past the blocks are zero; emit writes the `words` words that hold a row's own blocks
DFB_DEVICE void zero_scale_tail(uint8_t* tile, int words, int tile_cols, int tid, int threads) {
  for (int t = words + tid; t < tile_cols; t += threads) *reinterpret_cast<uint32_t*>(tile + t * 512) = 0;
}

// E columns of a bf16 row as they lie in memory: 32 bytes in one access where every row starts on 32, else 16.
template <int E>
struct Cols { uint32_t u[E / 2]; };
template <int E>
DFB_DEVICE Cols<E> load_cols(const bf16* p) {
  Cols<E> r;
  if constexpr (E == 16) load32(p, r.u);
  else *reinterpret_cast<uint4*>(r.u) = *reinterpret_cast<const uint4*>(p);
  return r;
}
template <int E>
DFB_DEVICE void store_cols(bf16* p, const Cols<E>& r) {
  if constexpr (E == 16) store32(p, r.u);
  else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.u);
}
// h = bf16(x + residual): the exact sum rounded once (the sum in 32 bits, rounded again, is the same number)
template <int E>
DFB_DEVICE void add_round(Cols<E>& a, const Cols<E>& b) {
#pragma unroll
  for (int i = 0; i < E / 2; ++i) asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(a.u[i]) : "r"(b.u[i]));
}
DFB_DEVICE float2 wide2(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
template <int E>
DFB_DEVICE float sum_squares(const Cols<E>& h) {
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const float2 f = wide2(h.u[i]);
    s = fma2(f, f, s);
  }
  return s.x + s.y;
}
template <int E>
DFB_DEVICE void scaled(const Cols<E>& h, const Cols<E>& w, float r, float* f) {
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const float2 v = mul2(mul2(wide2(h.u[i]), both(r)), wide2(w.u[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
// E columns of y into the output format; `on` = these columns exist, v = their index in E's, q / tile = where the row's codes and
// its first scale word lie.  mxfp4: 32 / E neighbouring lanes hold a block, four times as many a word of scales; 512 bytes to the
// next word.
template <bool MX, int E>
DFB_DEVICE void emit(const float* f, float inv, bool on, uint8_t* q, uint8_t* tile, int v) {
  if constexpr (MX) {
    constexpr int kLanes = kMxBlock / E;
    float amax = mx_amax8(f);
    if constexpr (E == 16) amax = max_nan(amax, mx_amax8(f + 8));
    amax = mx_amax_lanes<kLanes>(amax);
    const uint32_t sb = on ? mx_scale_byte(amax) : 0u;        // a block lies inside the row or behind it; there y is NaN where rstd is
    const uint32_t word = mx_scale_word<kLanes>(sb);
    if (on) {
      const float x = mx_scale_inv(sb);
      if constexpr (E == 16) *reinterpret_cast<uint2*>(q + v * 8) = make_uint2(mx_scale_pack8(f, x), mx_scale_pack8(f + 8, x));
      else *reinterpret_cast<uint32_t*>(q + v * 4) = mx_scale_pack8(f, x);
      if (v % (4 * kLanes) == 0) *reinterpret_cast<uint32_t*>(tile + v / (4 * kLanes) * 512) = word;
    }
  } else if (on) {
    uint32_t c[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const float2 y = mul2(make_float2(f[4 * i], f[4 * i + 1]), both(inv)), z = mul2(make_float2(f[4 * i + 2], f[4 * i + 3]), both(inv));
      c[i] = e4m3_pack2(y.x, y.y) | e4m3_pack2(z.x, z.y) << 16;
    }
    if constexpr (E == 16) *reinterpret_cast<uint4*>(q + v * 16) = *reinterpret_cast<const uint4*>(c);
    else *reinterpret_cast<uint2*>(q + v * 8) = make_uint2(c[0], c[1]);
  }
}

struct NormArgs {
  const bf16* x;
  const bf16* res;
  const bf16* w;
  const float* rstd_in;
  bf16* h;
  uint8_t* q;
  float* scale;
  uint8_t* tiles;
  float* rstd_out;
  long long ldx, ldr, ldh, rows;
  int cols;
  float eps, inv_cols;
};

// T threads hold a row in registers, VPT vectors of E columns each, and walk over rows with the next row's loads in flight
// (one row per block left a gap between a row's loads and the last block's stores); the gain stays in registers.  A block takes
// max(1, 128 / T) rows at a time.
template <bool MX, bool RES, int E, int T, int VPT>
__global__ void __launch_bounds__(T < 128 ? 128 : T, VPT * E <= 16 ? 1024 / (T < 128 ? 128 : T) : 1)
rmsnorm_quant_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float part[2][2][T / 32];             // [sum | max][parity of the row]: the next row's writes never meet this row's reads
  static_assert(T == 32 || T >= 128, "a row is one warp (no barrier) or a whole block");
  constexpr int kRows = T < 128 ? 128 / T : 1;
  const int tid = threadIdx.x % T, nvec = a.cols / E, tile_cols = mx_tile_cols(a.cols);
  const long long step = static_cast<long long>(gridDim.x) * kRows, rows_pad = MX ? (a.rows + 127) / 128 * 128 : a.rows;
  long long row = blockIdx.x * static_cast<long long>(kRows) + threadIdx.x / T;
  Cols<E> w[VPT], x[VPT], res[VPT];
  // where this thread's part of the row being fetched lies; advanced row by row
  const bf16 *xp = a.x + row * a.ldx + tid * E, *rp = a.res + (RES ? row * a.ldr + tid * E : 0);
  auto fetch = [&]() {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const bool on = j * T + tid < nvec;
      x[j] = Cols<E>{};
      if (on) x[j] = load_cols<E>(xp + j * (T * E));
      if (RES) {
        res[j] = Cols<E>{};
        if (on) res[j] = load_cols<E>(rp + j * (T * E));
      }
    }
    xp += step * a.ldx;
    if (RES) rp += step * a.ldr;
  };
  const int words = (a.cols + 127) >> 7;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int v = j * T + tid;
    w[j] = Cols<E>{};
    if (v < nvec) w[j] = load_cols<E>(a.w + v * E);
  }
  if (row < a.rows) fetch();
  for (int it = 0; row < rows_pad; row += step, it ^= 1) {
    uint8_t* tile = MX ? a.tiles + mx_scale_at(row, 0, tile_cols) : nullptr;
    uint8_t* q = a.q + row * (MX ? a.cols >> 1 : a.cols);
    if (MX && (words < tile_cols || row >= a.rows)) zero_scale_tail(tile, row < a.rows ? words : 0, tile_cols, tid, T);
    if (row >= a.rows) continue;                   // whole warps, and whole blocks where a row needs a barrier
    Cols<E> h[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      h[j] = x[j];
      if (RES) {
        add_round(h[j], res[j]);
        if (j * T + tid < nvec) store_cols(a.h + row * a.ldh + (j * T + tid) * E, h[j]);
      }
    }
    if (row + step < a.rows) fetch();
    float r;
    if (a.rstd_in) {
      r = a.rstd_in[row];
    } else {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < VPT; ++j) ss += sum_squares(h[j]);
      r = rsqrtf(row_reduce<T, false>(ss, part[0][it]) * a.inv_cols + a.eps);
      if (tid == 0) a.rstd_out[row] = r;
    }
    float inv = 1.f, y[VPT][E];
#pragma unroll
    for (int j = 0; j < VPT; ++j) scaled(h[j], w[j], r, y[j]);
    if (!MX) {
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < E; ++i) amax = fmaxf(amax, fabsf(y[j][i]));
      amax = row_reduce<T, true>(amax, part[1][it]);
      const float s = amax > 0.f ? fmaxf(__fmul_rn(amax, 1.f / kE4M3Top), kMinScale) : 1.f;
      inv = __frcp_rn(s);
      if (tid == 0) a.scale[row] = s;
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) emit<MX, E>(y[j], inv, j * T + tid < nvec, q, tile, j * T + tid);
  }
}

// Rows too wide for registers: the sum (or x) is read again from cache.
template <bool MX, bool RES>
__global__ void __launch_bounds__(512) rmsnorm_quant_wide_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float part[2][16];
  const long long row = blockIdx.x;
  const int nvec = a.cols >> 3, tile_cols = mx_tile_cols(a.cols);
  uint8_t* tile = MX ? a.tiles + mx_scale_at(row, 0, tile_cols) : nullptr;
  uint8_t* q = a.q + row * (MX ? a.cols >> 1 : a.cols);
  if (MX) zero_scale_tail(tile, row < a.rows ? (a.cols + 127) >> 7 : 0, tile_cols, threadIdx.x, 512);
  if (row >= a.rows) return;
  const bf16* hr = RES ? a.h + row * a.ldh : a.x + row * a.ldx;
  float ss = 0.f;
  if (RES || !a.rstd_in) {
    for (int v = threadIdx.x; v < nvec; v += 512) {
      Cols<8> h = load_cols<8>(a.x + row * a.ldx + v * 8);
      if (RES) {
        add_round(h, load_cols<8>(a.res + row * a.ldr + v * 8));
        store_cols(a.h + row * a.ldh + v * 8, h);
      }
      ss += sum_squares(h);
    }
  }
  float r;
  if (a.rstd_in) {
    r = a.rstd_in[row];
  } else {
    r = rsqrtf(row_reduce<512, false>(ss, part[0]) * a.inv_cols + a.eps);
    if (threadIdx.x == 0) a.rstd_out[row] = r;
  }
  float inv = 1.f;
  if (!MX) {
    float amax = 0.f;
    for (int v = threadIdx.x; v < nvec; v += 512) {
      float f[8];
      scaled(load_cols<8>(hr + v * 8), load_cols<8>(a.w + v * 8), r, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[i]));
    }
    amax = row_reduce<512, true>(amax, part[1]);
    const float s = amax > 0.f ? fmaxf(__fmul_rn(amax, 1.f / kE4M3Top), kMinScale) : 1.f;
    inv = __frcp_rn(s);
    if (threadIdx.x == 0) a.scale[row] = s;
  }
  for (int v0 = 0; v0 < nvec; v0 += 512) {
    const int v = v0 + threadIdx.x;
    float f[8] = {};
    if (v < nvec) scaled(load_cols<8>(hr + v * 8), load_cols<8>(a.w + v * 8), r, f);
    emit<MX, 8>(f, inv, v < nvec, q, tile, v);
  }
}

template <bool MX, bool RES>
int launch(const NormArgs& a, int num_sms, cudaStream_t s) {
  if (!a.rows) return 0;
  const long long rows = MX ? (a.rows + 127) / 128 * 128 : a.rows;      // with the padding of the scale tiles
  if (rows > 0x7fffffffLL) return -3;
  const int nvec = a.cols >> 3;
  // Blocks for 1024 threads per SM: all resident where a thread holds at most 16 columns; with more (108 to 149 registers) an SM holds
  // 256 to 512 threads at a time and the other blocks follow, each walking its own rows.
  auto go = [&](auto kernel, int threads, int rows_per_block) {
    const long long need = (rows + rows_per_block - 1) / rows_per_block, fit = static_cast<long long>(num_sms) * (1024 / threads);
    kernel<<<static_cast<unsigned>(need < fit ? need : fit), threads, 0, s>>>(a);
  };
  // 32-byte accesses (16 columns a lane) where every row of every operand starts on 32 bytes, 16-byte ones (8 columns) elsewhere.
  // us with the residual into 8 bits, 16 / 8 columns a lane, 16384 rows of 256: 7.2 / 5.4, 512: 12.3 / 12.1, 1024: 20.7 / 22.2,
  // 2048: 38.0 / 37.9, 4096: 71.7 / 72.9 (470 MB at the copy rate: 71.7); 8192 rows of 8192: 74.4 / 80.3.
  auto starts_on_32 = [](const void* p, long long ld) { return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(2 * ld)) & 31) == 0; };
  const bool e16 = a.cols % 16 == 0 && starts_on_32(a.x, a.ldx) && starts_on_32(a.res, a.ldr) && starts_on_32(a.h, a.ldh) && starts_on_32(a.w, 0);
  // Threads of a row, by the same measure: 1024 columns a warp 20.7, 128 threads 25; 2048: 128 threads 38.0, a warp 38.9; 4096: 128
  // of two vectors 71.7, 256 of one 72.0; 8192: 256 of two 74.4, 512 of one 76.5; 4096 rows of 16384: 512 of two 84.6, 1024 of one
  // 92.8, not held in registers 131.
  if (nvec <= 32) go(rmsnorm_quant_kernel<MX, RES, 8, 32, 1>, 128, 4);
  else if (e16 && nvec <= 64) go(rmsnorm_quant_kernel<MX, RES, 16, 32, 1>, 128, 4);
  else if (e16 && nvec <= 128) go(rmsnorm_quant_kernel<MX, RES, 16, 32, 2>, 128, 4);
  else if (e16 && nvec <= 256) go(rmsnorm_quant_kernel<MX, RES, 16, 128, 1>, 128, 1);
  else if (e16 && nvec <= 512) go(rmsnorm_quant_kernel<MX, RES, 16, 128, 2>, 128, 1);
  else if (e16 && nvec <= 1024) go(rmsnorm_quant_kernel<MX, RES, 16, 256, 2>, 256, 1);
  else if (e16 && nvec <= 2048) go(rmsnorm_quant_kernel<MX, RES, 16, 512, 2>, 512, 1);
  else if (nvec <= 64) go(rmsnorm_quant_kernel<MX, RES, 8, 32, 2>, 128, 4);
  else if (nvec <= 128) go(rmsnorm_quant_kernel<MX, RES, 8, 32, 4>, 128, 4);
  else if (nvec <= 256) go(rmsnorm_quant_kernel<MX, RES, 8, 128, 2>, 128, 1);
  else if (nvec <= 512) go(rmsnorm_quant_kernel<MX, RES, 8, 256, 2>, 256, 1);
  else if (nvec <= 1024) go(rmsnorm_quant_kernel<MX, RES, 8, 512, 2>, 512, 1);
  else if (nvec <= 2048) go(rmsnorm_quant_kernel<MX, RES, 8, 512, 4>, 512, 1);
  else rmsnorm_quant_wide_kernel<MX, RES><<<static_cast<unsigned>(rows), 512, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // namespace

int rmsnorm_fp8(const void* x, long long ldx, const void* res, long long ldr, const void* w, const float* rstd_in, float eps, void* h,
                long long ldh, void* q, float* scale, float* rstd, long long rows, int cols, int num_sms, cudaStream_t s) {
  const NormArgs a{(const bf16*)x, (const bf16*)res, (const bf16*)w, rstd_in, (bf16*)h, (uint8_t*)q, scale, nullptr, rstd,
                   ldx, ldr, ldh, rows, cols, eps, 1.f / cols};
  return res ? launch<false, true>(a, num_sms, s) : launch<false, false>(a, num_sms, s);
}
int rmsnorm_mxfp4(const void* x, long long ldx, const void* res, long long ldr, const void* w, const float* rstd_in, float eps, void* h,
                  long long ldh, void* q, void* tiles, float* rstd, long long rows, int cols, int num_sms, cudaStream_t s) {
  const NormArgs a{(const bf16*)x, (const bf16*)res, (const bf16*)w, rstd_in, (bf16*)h, (uint8_t*)q, nullptr, (uint8_t*)tiles, rstd,
                   ldx, ldr, ldh, rows, cols, eps, 1.f / cols};
  return res ? launch<true, true>(a, num_sms, s) : launch<true, false>(a, num_sms, s);
}

}  // namespace dfb
