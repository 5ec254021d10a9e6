// Product of two operands in the microscaled 4-bit format on CTA pairs: D (M, N) = A (M, K) x B (N, K)^T (+ bias) (+ addend).
//
//   D[m, n] = sum over blocks b of 32:  2^(sa[m, b] + sb[n, b] - 254) * sum_i a[m, 32 b + i] b[n, 32 b + i]
//
// tcgen05.mma kind::mxf4 with one e8m0 scale per 32 elements: the tensor core multiplies the scales in itself, reading them from
// tensor memory.  256 x 256 outputs per pair of SMs, 256 elements of K (128 bytes per row, 128-byte swizzle) per stage.
// Per CTA:
//   warp 0      TMA producer: own 128 rows of A, own half of B's rows, own rows' A scales, and ALL 256 rows' B scales (each SM
//               of the pair multiplies its 128 rows by the whole tile's columns)
//   warp 1      leader only: copies the stage's scales from shared to tensor memory (tcgen05.cp, both CTAs) and issues the four
//               MMAs of the stage; both run in issue order, so the copy needs no wait
//   warps 2-5   epilogue of the CTA's own 128 accumulator lanes
// Tensor memory: scales need 24 columns per stage (two stages in turn), which two whole 256-column accumulators would not leave.
// The accumulators overlap by 64 columns instead: [0, 256) and [192, 448).  The epilogue drains the shared columns first and
// then lets the next tile's MMAs begin, so all but that quarter of the epilogue stays hidden behind the main loop.
// Rows and blocks past the operands read as zero codes with zero scale bytes.  Every wait is bounded.
//
// 8192 x 28672 x 4096: 356 us alone (5.4 PFLOP/s), 409 us back to back (4.7: the power cap); 8192 x 8192 x 16384 6.35 PFLOP/s, 0.96
// of four times the library's bf16 rate.  A stage takes about 700 cycles instead of the MMA's 512: 35 KB arrive in shared memory and
// 32 KB are read from it, which its port bounds, in this kind as in bf16 and fp8.  The epilogue's pass through shared memory costs
// 15 % of a K of 4096 alone and nothing under the cap; halves of 128 columns on three accumulators hid it no better.
#include <cuda.h>

#include <atomic>
#include <mutex>

#include "lowbit.h"
#include "lowbit_common.cuh"
#include "ops.h"
#include "ptx.cuh"

namespace dfb {
namespace {
namespace mx {

constexpr int BM = 256, HALF_M = 128, BN = 256, HALF_N = 128, BK = 256;      // BK in elements: 128 bytes per row
constexpr int STAGES = 5;                                                    // 3 / 4 / 5 stages: 133 / 117 / 113 us at 8192 x 8192 x 4096
constexpr int A_BYTES = HALF_M * BK / 2, B_BYTES = HALF_N * BK / 2;          // 16 KiB each
constexpr int SF_TILE = 512;                                                 // scales of 128 rows x 128 elements
constexpr int SFA_BYTES = 2 * SF_TILE, SFB_BYTES = 4 * SF_TILE;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 4096;                        // 3 KiB of scales, kept 1024-byte aligned
constexpr int LOAD_BYTES = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
constexpr int TMEM_COLS = 512, ACC1 = 192, OVERLAP = 64, SF_COL = 448, SF_STRIDE = 32;
constexpr int THREADS = 192;
constexpr int EPI_BOX_BYTES = 32 * 128;
constexpr int EPI_BYTES = 4 * 2 * EPI_BOX_BYTES;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + 1024 + 256;

struct Params {
  int M, N, K;
  void* D;
  const void* addend;
  const void* bias;
  long long ldd, ld_add;
  int d_is_f32;
  int group_m;
  int tma_epi;
};

struct Barriers {
  uint64_t full[STAGES];       // used in the leader: both CTAs' bytes land here
  uint64_t empty[STAGES];      // per CTA
  uint64_t tmem_full[2];       // per CTA
  uint64_t drained;            // used in the leader: both CTAs' epilogues have read the shared columns of the tile before
  uint64_t add_full[4][2];     // per epilogue warp and box
  uint32_t tmem_base;
  int abort;
};

__device__ int g_error;

// block-scaled instruction descriptor: A and B e2m1 (1), scales e8m0, fp32 accumulators, which pair of the four scale bytes of
// a tensor-memory word the instruction takes ([4,6) for B, [29,31) for A)
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N, int pair) {
  return (static_cast<uint32_t>(2 * pair) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(M >> 7) << 27) | (static_cast<uint32_t>(2 * pair) << 29);
}
DFB_PTX void umma_mxf4_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      : : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// 512 bytes of scales (32 rows of 16 bytes, unswizzled) -> four columns, repeated in the four lane quarters, in both CTAs
DFB_PTX void scales_to_tmem_pair(uint32_t taddr, uint32_t smem_addr) {
  const uint64_t desc = static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | ptx::kDescVersion;
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" : : "r"(taddr), "l"(desc) : "memory");
}

DFB_DEVICE void tile_coords(int tile, int m_blocks, int n_blocks, int group_m, int& mb, int& nb) {
  const int per_group = group_m * n_blocks, g = tile / per_group, first = g * group_m;
  const int gm = min(m_blocks - first, group_m), r = tile - g * per_group;
  mb = first + r % gm;
  nb = r / gm;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                  const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb,
                  const __grid_constant__ CUtensorMap tmap_d, const __grid_constant__ CUtensorMap tmap_add, Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_smem = smem + STAGES * STAGE_BYTES;
  Barriers* sb = reinterpret_cast<Barriers*>(epi_smem + EPI_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = ptx::cluster_ctarank();
  const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
  const int m_blocks = (p.M + BM - 1) / BM, n_blocks = (p.N + BN - 1) / BN, num_tiles = m_blocks * n_blocks;
  const int k_blocks = (p.K + BK - 1) / BK;
  volatile int* abort_flag = &sb->abort;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { ptx::mbar_init(&sb->full[s], 1); ptx::mbar_init(&sb->empty[s], 1); }
    for (int a = 0; a < 2; ++a) ptx::mbar_init(&sb->tmem_full[a], 1);
    ptx::mbar_init(&sb->drained, 8);
    for (int w = 0; w < 4; ++w) { ptx::mbar_init(&sb->add_full[w][0], 1); ptx::mbar_init(&sb->add_full[w][1], 1); }
    sb->abort = 0;
    ptx::mbar_fence_init();
    ptx::prefetch_tmap(&tmap_a);
    ptx::prefetch_tmap(&tmap_b);
    ptx::prefetch_tmap(&tmap_sa);
    ptx::prefetch_tmap(&tmap_sb);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(&sb->tmem_base, TMEM_COLS);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  const uint32_t tmem_base = sb->tmem_base;

  if (warp == 0) {
    if (ptx::elect_one()) {
      uint32_t it = 0;
      for (int tile = cluster_id; tile < num_tiles && !*abort_flag; tile += num_clusters) {
        int mb, nb;
        tile_coords(tile, m_blocks, n_blocks, p.group_m, mb, nb);
        const int m0 = mb * BM + static_cast<int>(cta) * HALF_M, n0 = nb * BN + static_cast<int>(cta) * HALF_N;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % STAGES;
          if (!ptx::mbar_wait(&sb->empty[s], ((it / STAGES) & 1) ^ 1, abort_flag)) { sb->abort = 1; atomicExch(&g_error, 11); break; }
          uint8_t* st = smem + s * STAGE_BYTES;
          if (cta == 0) ptx::mbar_expect_tx(&sb->full[s], 2 * LOAD_BYTES);
          ptx::tma_load_2d_pair(st, &tmap_a, &sb->full[s], kb * (BK / 2), m0);
          ptx::tma_load_2d_pair(st + A_BYTES, &tmap_b, &sb->full[s], kb * (BK / 2), n0);
          // one row of a scale map = the two tiles of 128 rows x 256 elements; rows past the operand read as zero
          uint8_t* sf = st + A_BYTES + B_BYTES;
          ptx::tma_load_2d_pair(sf, &tmap_sa, &sb->full[s], 0, (m0 >> 7) * k_blocks + kb);
          ptx::tma_load_2d_pair(sf + SFA_BYTES, &tmap_sb, &sb->full[s], 0, nb * 2 * k_blocks + kb);
          ptx::tma_load_2d_pair(sf + SFA_BYTES + 2 * SF_TILE, &tmap_sb, &sb->full[s], 0, (nb * 2 + 1) * k_blocks + kb);
        }
      }
    }
  } else if (warp == 1) {
    if (cta == 0 && ptx::elect_one()) {
      uint32_t it = 0, tcount = 0;
      for (int tile = cluster_id; tile < num_tiles && !*abort_flag; tile += num_clusters, ++tcount) {
        const int acc = tcount & 1;
        if (tcount && !ptx::mbar_wait(&sb->drained, (tcount - 1) & 1, abort_flag)) { sb->abort = 1; atomicExch(&g_error, 12); break; }
        ptx::tc_fence_after();
        const uint32_t tmem_d = tmem_base + acc * ACC1;
        bool failed = false;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % STAGES;
          if (!ptx::mbar_wait(&sb->full[s], (it / STAGES) & 1, abort_flag)) { sb->abort = 1; atomicExch(&g_error, 13); failed = true; break; }
          ptx::tc_fence_after();
          const uint32_t a_addr = ptx::smem_u32(smem + s * STAGE_BYTES), sf = a_addr + A_BYTES + B_BYTES;
          const uint32_t sfa = tmem_base + SF_COL + (it & 1) * SF_STRIDE, sfb = sfa + 8;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            scales_to_tmem_pair(sfa + c * 4, sf + c * SF_TILE);
            scales_to_tmem_pair(sfb + c * 8, sf + SFA_BYTES + c * SF_TILE);
            scales_to_tmem_pair(sfb + c * 8 + 4, sf + SFA_BYTES + (2 + c) * SF_TILE);
          }
          const uint64_t adesc = ptx::desc_kmajor_sw128(a_addr), bdesc = ptx::desc_kmajor_sw128(a_addr + A_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k)         // 64 elements = 32 bytes of K per instruction
            umma_mxf4_pair(tmem_d, adesc + k * 2, bdesc + k * 2, idesc_mxf4(BM, BN, k & 1), sfa + (k >> 1) * 4, sfb + (k >> 1) * 8, (kb | k) != 0);
          ptx::umma_commit_pair(&sb->empty[s], 0x3);
        }
        if (failed) break;
        ptx::umma_commit_pair(&sb->tmem_full[acc], 0x3);
      }
    }
  } else {
    const int q = warp & 3;
    const int box_cols = p.d_is_f32 ? 32 : 64, chunks = BN / box_cols, shared_chunks = OVERLAP / box_cols;
    const int row_in_cta = static_cast<int>(cta) * HALF_M + q * 32;
    uint8_t* my_smem = epi_smem + q * 2 * EPI_BOX_BYTES;
    uint64_t* my_bar = sb->add_full[q];
    const bool tma = p.tma_epi != 0, tma_add = tma && p.addend != nullptr;
    // the i-th box of a tile: the columns that the accumulators share come first (the last of acc 0, the first of acc 1)
    auto box_of = [&](uint32_t tc, int i) { return (tc & 1) ? i : (i + chunks - shared_chunks) % chunks; };
    uint32_t tcount = 0, cc = 0;
    if (tma_add && lane == 0 && cluster_id < num_tiles) {
      int mb, nb;
      tile_coords(cluster_id, m_blocks, n_blocks, p.group_m, mb, nb);
      ptx::mbar_expect_tx(&my_bar[0], EPI_BOX_BYTES);
      ptx::tma_load_2d(my_smem, &tmap_add, &my_bar[0], nb * BN + box_of(0, 0) * box_cols, mb * BM + row_in_cta);
    }
    for (int tile = cluster_id; tile < num_tiles && !*abort_flag; tile += num_clusters, ++tcount) {
      int mb, nb;
      tile_coords(tile, m_blocks, n_blocks, p.group_m, mb, nb);
      const int acc = tcount & 1;
      if (!ptx::mbar_wait(&sb->tmem_full[acc], (tcount >> 1) & 1, abort_flag)) { sb->abort = 1; atomicExch(&g_error, 14); break; }
      ptx::tc_fence_after();
      const int row0 = mb * BM + row_in_cta;
      const uint32_t taddr = tmem_base + acc * ACC1 + (static_cast<uint32_t>(q * 32) << 16);
      bool failed = false;
#pragma unroll 1
      for (int i = 0; i < chunks; ++i, ++cc) {
        const int c = box_of(tcount, i), b = cc & 1;
        uint8_t* buf = my_smem + b * EPI_BOX_BYTES;
        uint8_t* my_row = buf + lane * 128;
        const int col0 = nb * BN + c * box_cols;
        float f[64];
        {
          uint32_t r[32];
          ptx::tmem_ld_32x32(taddr + c * box_cols, r);
          if (!p.d_is_f32) {
            uint32_t r2[32];
            ptx::tmem_ld_32x32(taddr + c * box_cols + 32, r2);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) f[32 + k] = __uint_as_float(r2[k]);
          } else {
            ptx::tmem_ld_wait();
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) f[k] = __uint_as_float(r[k]);
        }
        if (i == shared_chunks - 1) {        // the next tile may write the columns both accumulators use
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cluster(&sb->drained, 0);
        }
        if (p.bias) {
          const bf16* bp = reinterpret_cast<const bf16*>(p.bias) + col0;
#pragma unroll
          for (int k = 0; k < 64; ++k)
            if (k < box_cols && col0 + k < p.N) f[k] += bf2f(bp[k]);
        }
        if (!tma) {
          // rows that no TMA box can start on: element by element
          const int row = row0 + lane;
          if (row < p.M) {
#pragma unroll
            for (int k = 0; k < 64; ++k)
              if (k < box_cols && col0 + k < p.N) {
                const long long at = row * p.ldd + col0 + k, from = row * p.ld_add + col0 + k;
                if (p.d_is_f32) {
                  if (p.addend) f[k] += reinterpret_cast<const float*>(p.addend)[from];
                  reinterpret_cast<float*>(p.D)[at] = f[k];
                } else {
                  if (p.addend) f[k] += bf2f(reinterpret_cast<const bf16*>(p.addend)[from]);
                  reinterpret_cast<bf16*>(p.D)[at] = f2bf(f[k]);
                }
              }
          }
          continue;
        }
        if (tma_add) {
          if (!ptx::mbar_wait(&my_bar[b], (cc >> 1) & 1, abort_flag)) { sb->abort = 1; atomicExch(&g_error, 15); failed = true; break; }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint4 v = *reinterpret_cast<const uint4*>(my_row + ((j ^ (lane & 7)) << 4));
            if (p.d_is_f32) {
              f[j * 4] += __uint_as_float(v.x); f[j * 4 + 1] += __uint_as_float(v.y);
              f[j * 4 + 2] += __uint_as_float(v.z); f[j * 4 + 3] += __uint_as_float(v.w);
            } else {
              float t[8];
              unpack8(*reinterpret_cast<const bf16x8*>(&v), t);
#pragma unroll
              for (int k = 0; k < 8; ++k) f[j * 8 + k] += t[k];
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint4 v;
          if (p.d_is_f32) {
            v = make_uint4(__float_as_uint(f[j * 4]), __float_as_uint(f[j * 4 + 1]), __float_as_uint(f[j * 4 + 2]), __float_as_uint(f[j * 4 + 3]));
          } else {
            const bf16x8 pk = pack8(f + j * 8);
            v = *reinterpret_cast<const uint4*>(&pk);
          }
          *reinterpret_cast<uint4*>(my_row + ((j ^ (lane & 7)) << 4)) = v;
        }
        ptx::fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          if (col0 < p.N && row0 < p.M) ptx::tma_store_2d(&tmap_d, buf, col0, row0);
          ptx::tma_store_commit();
          ptx::tma_store_wait_read<1>();           // the other box's store has left shared memory
          if (tma_add) {
            int nt = tile, ni = i + 1;
            uint32_t ntc = tcount;
            if (ni == chunks) { nt = tile + num_clusters; ni = 0; ++ntc; }
            if (nt < num_tiles) {
              int nmb, nnb;
              tile_coords(nt, m_blocks, n_blocks, p.group_m, nmb, nnb);
              ptx::mbar_expect_tx(&my_bar[b ^ 1], EPI_BOX_BYTES);
              ptx::tma_load_2d(my_smem + (b ^ 1) * EPI_BOX_BYTES, &tmap_add, &my_bar[b ^ 1], nnb * BN + box_of(ntc, ni) * box_cols,
                               nmb * BM + row_in_cta);
            }
          }
        }
        __syncwarp();
      }
      if (failed) break;
    }
    if (tma && lane == 0) ptx::tma_store_wait<0>();
    __syncwarp();
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);      // let copies still in flight land
  }
  ptx::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess) fn = reinterpret_cast<EncodeFn>(p);
  });
  return fn;
}
bool make_map(CUtensorMap* m, CUtensorMapDataType type, const void* base, uint64_t inner, uint64_t outer, uint64_t pitch_bytes, uint32_t box_inner,
              uint32_t box_outer, bool swizzle) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {inner, outer}, strides[1] = {pitch_bytes};
  cuuint32_t box[2] = {box_inner, box_outer}, estr[2] = {1, 1};
  return fn(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}


// ---------------------------------------------------------------------------------------------------------------------------
// Few tiles: rows of B (the weight) are the 128 rows of a CTA's MMA, up to 128 rows of A its columns, and the CTAs of a cluster
// split K.  Each leaves its partial sums in its own shared memory; then every CTA of the cluster adds a share of them up, in rank
// order (the result does not depend on who came first), and writes it.  A weight of 4096 x 4096 for a few tokens is spread over
// 128 SMs instead of 32.
namespace skinny {
constexpr int TM = 128, TN = 128;                                            // weight rows, tokens
constexpr int STAGES = 6;
constexpr int W_BYTES = TM * BK / 2, X_BYTES = TN * BK / 2, SF_BYTES = 2 * SF_TILE;
constexpr int STAGE_BYTES = W_BYTES + X_BYTES + 2 * SF_BYTES;
constexpr int SF_COL = 128, SF_STRIDE = 16, TMEM_COLS = 256;
constexpr int THREADS = 128;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256;
static_assert(STAGES * STAGE_BYTES >= TM * TN * 4, "the partial sums take the stages' place");

struct Barriers {
  uint64_t full[STAGES], empty[STAGES], done;
  uint32_t tmem_base;
  int abort;
};

DFB_PTX void umma_mxf4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      : : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
DFB_PTX void scales_to_tmem(uint32_t taddr, uint32_t smem_addr) {
  const uint64_t desc = static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | ptx::kDescVersion;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" : : "r"(taddr), "l"(desc) : "memory");
}
DFB_PTX float4 load_remote(uint32_t smem_addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [ra];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem_addr), "r"(rank) : "memory");
  return v;
}

// grid (SPLITS * tiles of N, tiles of M), clusters of SPLITS along x
template <int SPLITS>
__global__ void __launch_bounds__(THREADS, 1)
gemm_mxfp4_skinny_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                         const __grid_constant__ CUtensorMap tmap_sw, const __grid_constant__ CUtensorMap tmap_sx, Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Barriers* sb = reinterpret_cast<Barriers*>(smem + STAGES * STAGE_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int n0 = (blockIdx.x / SPLITS) * TM, m0 = blockIdx.y * TN;
  const int tokens = min(TN, p.M - m0), mma_n = (tokens + 15) & ~15;
  const int k_blocks = (p.K + BK - 1) / BK, per = (k_blocks + SPLITS - 1) / SPLITS;
  const int k_lo = min(rank * per, k_blocks), k_hi = min(k_lo + per, k_blocks);
  volatile int* abort_flag = &sb->abort;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { ptx::mbar_init(&sb->full[s], 1); ptx::mbar_init(&sb->empty[s], 1); }
    ptx::mbar_init(&sb->done, 1);
    sb->abort = 0;
    ptx::mbar_fence_init();
    ptx::prefetch_tmap(&tmap_w);
    ptx::prefetch_tmap(&tmap_x);
    ptx::prefetch_tmap(&tmap_sw);
    ptx::prefetch_tmap(&tmap_sx);
  }
  if (warp == 1) {
    ptx::tmem_alloc(&sb->tmem_base, TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = sb->tmem_base;
  if (warp == 0) {
    if (ptx::elect_one()) {
      for (int kb = k_lo, it = 0; kb < k_hi; ++kb, ++it) {
        const int s = it % STAGES;
        if (!ptx::mbar_wait(&sb->empty[s], ((it / STAGES) & 1) ^ 1, abort_flag)) { sb->abort = 1; atomicExch(&g_error, 21); break; }
        uint8_t* st = smem + s * STAGE_BYTES;
        ptx::mbar_expect_tx(&sb->full[s], STAGE_BYTES);
        ptx::tma_load_2d(st, &tmap_w, &sb->full[s], kb * (BK / 2), n0);
        ptx::tma_load_2d(st + W_BYTES, &tmap_x, &sb->full[s], kb * (BK / 2), m0);
        ptx::tma_load_2d(st + W_BYTES + X_BYTES, &tmap_sw, &sb->full[s], 0, (n0 >> 7) * k_blocks + kb);
        ptx::tma_load_2d(st + W_BYTES + X_BYTES + SF_BYTES, &tmap_sx, &sb->full[s], 0, (m0 >> 7) * k_blocks + kb);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (ptx::elect_one()) {
      bool failed = false;
      for (int kb = k_lo, it = 0; kb < k_hi; ++kb, ++it) {
        const int s = it % STAGES;
        if (!ptx::mbar_wait(&sb->full[s], (it / STAGES) & 1, abort_flag)) { sb->abort = 1; atomicExch(&g_error, 22); failed = true; break; }
        ptx::tc_fence_after();
        const uint32_t w_addr = ptx::smem_u32(smem + s * STAGE_BYTES), sf = w_addr + W_BYTES + X_BYTES;
        const uint32_t sfw = tmem_base + SF_COL + (it & 1) * SF_STRIDE, sfx = sfw + 8;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          scales_to_tmem(sfw + c * 4, sf + c * SF_TILE);
          scales_to_tmem(sfx + c * 4, sf + SF_BYTES + c * SF_TILE);
        }
        const uint64_t wdesc = ptx::desc_kmajor_sw128(w_addr), xdesc = ptx::desc_kmajor_sw128(w_addr + W_BYTES);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_mxf4(tmem_base, wdesc + k * 2, xdesc + k * 2, idesc_mxf4(TM, mma_n, k & 1), sfw + (k >> 1) * 4, sfx + (k >> 1) * 4, it != 0 || k != 0);
        ptx::umma_commit(&sb->empty[s]);
      }
      if (!failed) ptx::umma_commit(&sb->done);
    }
    __syncwarp();
  }
  // partial sums to shared memory, one token's 128 values in a row: every copy into the stages has been read by then
  float* part = reinterpret_cast<float*>(smem);
  if (!ptx::mbar_wait(&sb->done, 0, abort_flag)) { sb->abort = 1; atomicExch(&g_error, 23); }
  ptx::tc_fence_after();
  const uint32_t taddr = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
  for (int c = 0; c < tokens; c += 32) {
    uint32_t r[32];
    ptx::tmem_ld_32x32(taddr + c, r);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (c + i < tokens) part[(c + i) * TM + warp * 32 + lane] = k_lo < k_hi ? __uint_as_float(r[i]) : 0.f;
  }
  ptx::tc_fence_before();
  ptx::cluster_sync();
  // this CTA's share of the tokens: one warp takes a token, a lane four neighbouring outputs
  const int n = n0 + lane * 4;
  for (int t = rank * 4 + warp; t < tokens; t += SPLITS * 4) {
    const uint32_t at = ptx::smem_u32(part + t * TM + lane * 4);
    const long long row = m0 + t;
    float4 v[SPLITS];                        // all of them on their way at once
#pragma unroll
    for (int r = 0; r < SPLITS; ++r) v[r] = load_remote(at, r);
    float more[4] = {0.f, 0.f, 0.f, 0.f};    // bias and addend
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) {
        if (p.bias) more[i] = bf2f(reinterpret_cast<const bf16*>(p.bias)[n + i]);
        if (p.addend)
          more[i] += p.d_is_f32 ? reinterpret_cast<const float*>(p.addend)[row * p.ld_add + n + i]
                                : bf2f(reinterpret_cast<const bf16*>(p.addend)[row * p.ld_add + n + i]);
      }
    float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < SPLITS; ++r) {
      f[0] += v[r].x; f[1] += v[r].y; f[2] += v[r].z; f[3] += v[r].w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) {
        if (p.d_is_f32) reinterpret_cast<float*>(p.D)[row * p.ldd + n + i] = f[i] + more[i];
        else reinterpret_cast<bf16*>(p.D)[row * p.ldd + n + i] = f2bf(f[i] + more[i]);
      }
  }
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);      // let copies still in flight land
  }
  ptx::cluster_sync();                     // nobody leaves while its sums may still be read
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}
}  // namespace skinny

// cudaFuncSetAttribute once per kernel and device
template <typename Kernel>
bool configure(Kernel kernel, int smem_bytes, std::atomic<bool>* done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return false;
  if (done[dev].load()) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes) != cudaSuccess) return false;
  done[dev].store(true);
  return true;
}

}  // namespace mx
}  // namespace

int gemm_mxfp4(const void* A, const void* sa, const void* B, const void* sb, void* D, long long ldd, int d_f32, const void* add,
               long long ld_add, const void* bias, long long M, long long N, int K, int num_sms, cudaStream_t stream) {
  using namespace mx;
  if (!M || !N) return 0;
  const long long m_blocks = (M + BM - 1) / BM, n_blocks = (N + BN - 1) / BN, tiles = m_blocks * n_blocks, k_blocks = (K + BK - 1) / BK;
  if (tiles > 0x7fffffffLL || 2 * (m_blocks > n_blocks ? m_blocks : n_blocks) * k_blocks > 0x7fffffffLL) return -3;
  ensure_context();
  const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8, u32 = CU_TENSOR_MAP_DATA_TYPE_UINT32;
  CUtensorMap ta, tb, tsa, tsb, td, tadd;
  bool ok = make_map(&ta, u8, A, K / 2, M, K / 2, BK / 2, HALF_M, true) && make_map(&tb, u8, B, K / 2, N, K / 2, BK / 2, HALF_N, true) &&
            make_map(&tsa, u32, sa, 256, (M + 127) / 128 * k_blocks, 1024, 256, 1, false) &&
            make_map(&tsb, u32, sb, 256, (N + 127) / 128 * k_blocks, 1024, 256, 1, false);
  // TMA boxes need rows that start on 16 bytes
  const int per16 = d_f32 ? 4 : 8;
  const bool tma_epi = ((reinterpret_cast<uintptr_t>(D) | reinterpret_cast<uintptr_t>(add)) & 15) == 0 && ldd % per16 == 0 && ld_add % per16 == 0;
  if (tma_epi) {
    const auto dt = d_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int es = d_f32 ? 4 : 2, bc = d_f32 ? 32 : 64;
    ok = ok && make_map(&td, dt, D, N, M, ldd * es, bc, 32, true) && make_map(&tadd, dt, add ? add : D, N, M, (add ? ld_add : ldd) * es, bc, 32, true);
  } else {
    td = ta;
    tadd = ta;
  }
  if (!ok) return -4;
  Params p;
  p.M = (int)M; p.N = (int)N; p.K = K;
  p.D = D; p.addend = add; p.bias = bias;
  p.ldd = ldd; p.ld_add = ld_add; p.d_is_f32 = d_f32;
  p.group_m = 16;
  p.tma_epi = tma_epi;
  // Stages that a CTA goes through one after the other: `pair` in the pair kernel, `few` in the skinny one, whose stages take as
  // long for a quarter of the outputs, and whose sums pass through shared memory.  It is taken where it halves the stages of a call
  // with at most 256 tokens, or, with at most 64, where it shortens them or is one wave.  us of the pair / skinny kernel, tokens x N
  // x K: 17 x 4096 x 4096 10.5 / 6.2, 128: 10.8 / 8.1, 256: 11.1 / 10.4, 512: 11.3 / 12.6; 64 x 4096 x 256 6.5 / 6.1; 17 x 14336 x
  // 4096 13.9 / 12.7, x 28672 22.0 / 22.3, x 131072 75 / 87; 128 x 14336 x 4096 13.4 / 14.1; 300 x 14336 x 4096 18.7 / 30.1;
  // 1024 x 1024 x 1024 7.4 / 8.5.
  const int clusters = num_sms / 2;
  const long long ctas = (N + skinny::TM - 1) / skinny::TM * ((M + skinny::TN - 1) / skinny::TN);
  int splits = 1;
  while (splits < 8 && ctas * splits * 2 <= num_sms && splits * 2 <= k_blocks) splits *= 2;
  const long long pair = (tiles + clusters - 1) / clusters * k_blocks;
  const long long few = (ctas * splits + num_sms - 1) / num_sms * ((k_blocks + splits - 1) / splits);
  const bool one_wave = ctas * splits <= num_sms;
  if (M <= 64 ? few < pair || (few == pair && one_wave) : M <= 256 && 2 * few <= pair) {
    static std::atomic<bool> ready[4][64];
    const int which = splits == 1 ? 0 : splits == 2 ? 1 : splits == 4 ? 2 : 3;
    auto kernel = which == 0 ? skinny::gemm_mxfp4_skinny_kernel<1> : which == 1 ? skinny::gemm_mxfp4_skinny_kernel<2>
                : which == 2 ? skinny::gemm_mxfp4_skinny_kernel<4> : skinny::gemm_mxfp4_skinny_kernel<8>;
    if (!configure(kernel, skinny::SMEM_BYTES, ready[which])) return -1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((N + skinny::TM - 1) / skinny::TM) * splits, static_cast<unsigned>((M + skinny::TN - 1) / skinny::TN));
    cfg.blockDim = dim3(skinny::THREADS);
    cfg.dynamicSmemBytes = skinny::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, tb, ta, tsb, tsa, p) == cudaSuccess ? 0 : -1;
  }
  static std::atomic<bool> ready[64];
  if (!configure(gemm_mxfp4_kernel, SMEM_BYTES, ready)) return -1;
  gemm_mxfp4_kernel<<<2 * static_cast<int>(tiles < clusters ? tiles : clusters), THREADS, SMEM_BYTES, stream>>>(ta, tb, tsa, tsb, td, tadd, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -1;
}

// The kernel's error word on the current device: 0, or which bounded wait ran out (11 producer, 12 / 13 MMA, 14 / 15 epilogue; 21 to 23 the same of
// the kernel for few tiles)
int gemm_mxfp4_last_error() {
  int v = 0;
  return cudaMemcpyFromSymbol(&v, mx::g_error, sizeof(int)) == cudaSuccess ? v : -1;
}

}  // namespace dfb
