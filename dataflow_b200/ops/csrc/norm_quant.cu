// RMS norm with the residual's addition whose output leaves in a narrow format.
//
//   h = bf16(x + residual)      rstd = (mean h^2 + eps)^(-1/2)      y = h rstd w  (fp32)
//   fp8:    s = max(amax |y| / 448, 2^-120) per row (1 for a row of zeros), q = e4m3(y (1 / s))
//   mxfp4:  blocks of 32 columns, X = 2^(floor(log2 amax) - 2), q = e2m1(y / X)
//
// The statistics are those of the rounded h, the tensor that the backward pass reads again.  One block per row.
#include "lowbit.h"
#include "lowbit_common.cuh"

namespace dfb {
namespace {

template <bool MX, bool RES>
__global__ void __launch_bounds__(256) rmsnorm_quant_kernel(const bf16* x, long long ldx, const bf16* res, long long ldr,
                                                             const bf16* __restrict__ w, const float* __restrict__ rstd_in, float eps, bf16* h,
                                                             long long ldh, uint8_t* __restrict__ q, float* __restrict__ scale,
                                                             uint8_t* __restrict__ tiles, float* __restrict__ rstd_out, long long rows, int cols) {
  __shared__ float scratch[33];
  const long long row = blockIdx.x;
  const int nvec = cols >> 3;
  const int tile_cols = mx_tile_cols(cols);
  if (MX) {
    // scale bytes past the rows and blocks are zero
    for (int b = threadIdx.x; b < tile_cols * 4; b += blockDim.x)
      if (row >= rows || b >= cols / kMxBlock) tiles[mx_scale_at(row, b, tile_cols)] = 0;
    if (row >= rows) return;
  }
  const bf16* xr = x + row * ldx;
  const bf16* hr = RES ? h + row * ldh : xr;
  float ss = 0.f;
  if (RES || !rstd_in) {
    for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
      float f[8];
      unpack8(ld8(xr + v * 8), f);
      if (RES) {
        float g[8];
        unpack8(ld8(res + row * ldr + v * 8), g);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += g[i];
        const bf16x8 p = pack8(f);
        st8(h + row * ldh + v * 8, p);
        unpack8(p, f);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += f[i] * f[i];
    }
  }
  float r;
  if (rstd_in) r = rstd_in[row];
  else r = rsqrtf(block_sum(ss, scratch) / cols + eps);
  if (threadIdx.x == 0 && rstd_out) rstd_out[row] = r;
  float s = 1.f, inv = 1.f;
  if (!MX) {
    float amax = 0.f;
    for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
      float f[8], g[8];
      unpack8(ld8(hr + v * 8), f);
      unpack8(ld8(w + v * 8), g);
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[i] * r * g[i]));
    }
    amax = block_max(amax, scratch);
    if (amax > 0.f) s = fmaxf(__fmul_rn(amax, 1.f / kE4M3Top), kMinScale);
    inv = __frcp_rn(s);
    if (threadIdx.x == 0) scale[row] = s;
  }
  for (int v0 = 0; v0 < nvec; v0 += blockDim.x) {
    const int v = v0 + threadIdx.x;
    const bool on = v < nvec;
    float f[8] = {}, g[8];
    if (on) {
      unpack8(ld8(hr + v * 8), f);
      unpack8(ld8(w + v * 8), g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * r * g[i];
    }
    if (MX) {
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, mx_abs(f[i]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const uint32_t sb = mx_scale_byte(amax);
      const float iv = mx_scale_inv(sb);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= iv;
      if (on) {
        *reinterpret_cast<uint32_t*>(q + row * (cols >> 1) + v * 4) = mx_pack8(f);
        if ((v & 3) == 0) tiles[mx_scale_at(row, v >> 2, tile_cols)] = static_cast<uint8_t>(sb);
      }
    } else if (on) {
      uint2 p;
      p.x = e4m3_pack2(f[0] * inv, f[1] * inv) | e4m3_pack2(f[2] * inv, f[3] * inv) << 16;
      p.y = e4m3_pack2(f[4] * inv, f[5] * inv) | e4m3_pack2(f[6] * inv, f[7] * inv) << 16;
      *reinterpret_cast<uint2*>(q + row * cols + v * 8) = p;
    }
  }
}

template <bool MX>
int launch(const void* x, long long ldx, const void* res, long long ldr, const void* w, const float* rstd_in, float eps, void* h,
           long long ldh, void* q, float* scale, void* tiles, float* rstd, long long rows, int cols, cudaStream_t s) {
  if (!rows) return 0;
  const long long blocks = MX ? (rows + 127) / 128 * 128 : rows;
  if (blocks > 0x7fffffffLL) return -3;
  auto go = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(blocks), 256, 0, s>>>((const bf16*)x, ldx, (const bf16*)res, ldr, (const bf16*)w, rstd_in, eps, (bf16*)h, ldh,
                                                         (uint8_t*)q, scale, (uint8_t*)tiles, rstd, rows, cols);
  };
  if (res) go(rmsnorm_quant_kernel<MX, true>);
  else go(rmsnorm_quant_kernel<MX, false>);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

}  // namespace

int rmsnorm_fp8(const void* x, long long ldx, const void* res, long long ldr, const void* w, const float* rstd_in, float eps, void* h,
                long long ldh, void* q, float* scale, float* rstd, long long rows, int cols, cudaStream_t s) {
  return launch<false>(x, ldx, res, ldr, w, rstd_in, eps, h, ldh, q, scale, nullptr, rstd, rows, cols, s);
}
int rmsnorm_mxfp4(const void* x, long long ldx, const void* res, long long ldr, const void* w, const float* rstd_in, float eps, void* h,
                  long long ldh, void* q, void* tiles, float* rstd, long long rows, int cols, cudaStream_t s) {
  return launch<true>(x, ldx, res, ldr, w, rstd_in, eps, h, ldh, q, nullptr, tiles, rstd, rows, cols, s);
}

}  // namespace dfb
