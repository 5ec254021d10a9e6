// Launch API of the narrow-format operators (adamw_multi.cu, norm_quant.cu, mxfp4.cu, gemm_mxfp4.cu).  Every function
// enqueues on ``s`` of the current device and returns 0, or a negative code when it refuses or the launch failed.
#pragma once
#include <cuda_runtime_api.h>
#include <stdint.h>

namespace dfb {

// one tensor of an AdamW step over many; null pointers for what the call's types do not have
struct AdamTensor {
  void* w;
  const void* g;
  void* m;
  void* v;
  void* extra;            // fp32 master, or the int16 low halves of a split master
  float* m_scale;
  float* v_scale;
  long long n;
  float wd;
  uint32_t seed;          // of the 8-bit rounding
};
enum AdamWeights { kAdamBf16 = 0, kAdamF32 = 1, kAdamMaster = 2, kAdamSplit = 3 };
struct AdamHyper {
  float lr, b1, c1, b2, c2, eps, inv_bc1, inv_sqrt_bc2, gscale;
  float one = 1.f;
};
int adamw_multi(const AdamTensor* t, int count, int weights, bool g_f32, bool bits8, const AdamHyper& h, int num_sms, cudaStream_t s);

// h = bf16(x + residual) (h == null: x is taken as it is), y = h * rstd * w.  rstd_in: statistics to apply (null: computed).
int rmsnorm_fp8(const void* x, long long ldx, const void* res, long long ldr, const void* w, const float* rstd_in, float eps, void* h,
                long long ldh, void* q, float* scale, float* rstd, long long rows, int cols, int num_sms, cudaStream_t s);
int rmsnorm_mxfp4(const void* x, long long ldx, const void* res, long long ldr, const void* w, const float* rstd_in, float eps, void* h,
                  long long ldh, void* q, void* tiles, float* rstd, long long rows, int cols, int num_sms, cudaStream_t s);

// x (rows, K), row pitch ldx elements (transposed: x (K, rows), pitch of a K row); q (rows, K / 2), tiles as in lowbit_common.cuh
int quant_mxfp4(const void* x, long long ldx, int x_f32, int transposed, void* q, void* tiles, long long rows, int K, cudaStream_t s);
int dequant_mxfp4(const void* q, const void* tiles, void* y, int y_f32, long long rows, int K, cudaStream_t s);

int gemm_mxfp4(const void* A, const void* sa, const void* B, const void* sb, void* D, long long ldd, int d_f32, const void* add,
               long long ld_add, const void* bias, long long M, long long N, int K, int num_sms, cudaStream_t s);
int gemm_mxfp4_last_error();

}  // namespace dfb
