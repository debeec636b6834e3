// Products of rows with weights, act(A B^T + bias): block-scaled e4m3, and rows in ragged groups that each have a matrix
// of their own (occamy_matmul_e4m3, occamy_matmul_grouped).
//
//   out[m][n] = act( sum over blocks j of 128 along K:  sA[m][j] * sB[n / 128][j] * sum over k in j: a[m][k] b[n][k]   + bias[n] )
//
// The weights are the M side of the tensor core's tile (128 of them to the TMEM lanes) and the rows its N side (the
// columns): N may be any multiple of 16, so that a group of a few rows takes a narrow tile and the last tile of a
// group no more than it has, where 128 rows on the M side would be multiplied whatever there are.
//
// The tensor core adds the products of one k-step (128 bytes of K) into a TMEM buffer; eight epilogue warps take each
// finished buffer, multiply it by its scales and add it to sums they hold in registers, fp32.  16-bit operands have no
// scales, but go the same way every few k-steps: the tensor core truncates when it adds to its accumulator, an error
// that grows with the number of additions (fp16, K = 1160: see PT_PER).  A thread's values are those of mma fragments
// (16x256b loads: two rows of weights, pairs of columns), so one scale serves four of its sums and its 16-bit results
// leave through a transposing stmatrix as rows of 64 bytes.
//
// With few tiles the CTAs of a cluster share a tile's K and add up their sums in rank order through each other's
// shared memory: no workspace, and the same bits every time.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>
#include <mutex>

#include "conv_tc_dev.cuh"
#include "expert_ops.h"
#include "runtime.h"

namespace occ {
namespace {

constexpr int PT_THREADS = 384;        // loads, MMAs, two warps of scales; eight epilogue warps
constexpr int PT_EPI_WARPS = 8;
constexpr int PT_ROWS = 128;           // weights of a tile
constexpr int PT_BOX = 32;             // rows of one copy
constexpr int PT_RASTER = 16;          // row tiles that go through all weights together
constexpr int PT_PER = 4;              // k-steps of 16-bit operands that the tensor core adds up by itself

struct alignas(64) PtParams {
  CUtensorMap ta, tb;
  const int32_t *index, *offsets;
  const float *scale_a, *scale_b, *bias;
  void *out;
  int64_t ldo;
  int a_rows, rows, groups, N, act, out_type, gated;
  int kblocks;                         // k-steps: blocks of 128 bytes along K
  int blocks_n;                        // scale blocks of a matrix along N
  int tiles_n, stages, splits, bufs;
  uint32_t idesc;
  int vec_out;                         // 16-byte stores of the result are possible
  int *err;
};

template <bool SCALED>
__device__ __forceinline__ void pt_mma(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                       uint32_t idesc, uint32_t accumulate) {
  if constexpr (SCALED)
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 da, db;\n"
        "elect.sync _|q, 0xffffffff;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "mov.b64 da, {%1, %2};\n"
        "mov.b64 db, {%3, %4};\n"
        "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n}" ::"r"(d_tmem),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    mma_warp(d_tmem, a_lo, a_hi, b_lo, b_hi, idesc, accumulate);
}
__device__ __forceinline__ void load_2d_warp(uint32_t dst, const CUtensorMap *m, uint32_t bar, int c0, int c1) {
  asm volatile(
      "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n}" ::"r"(dst),
      "l"(m), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void load_5d_warp(uint32_t dst, const CUtensorMap *m, uint32_t bar, int c0, int c3, int c4) {
  asm volatile(
      "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
      "@q cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %6, %6, %4, %5}], [%2];\n}" ::"r"(dst),
      "l"(m), "r"(bar), "r"(c0), "r"(c3), "r"(c4), "r"(0)
      : "memory");
}
// Four rows, by the executing lane.
__device__ __forceinline__ void gather_4_rows(uint32_t dst, const CUtensorMap *m, uint32_t bar, int c0, int4 r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(m), "r"(bar), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w)
      : "memory");
}
// 16 lanes x 32 columns: r[4 g + 0, 1] lane t / 4, columns 8 g + 2 (t % 4) + 0, 1; r[4 g + 2, 3] the same of lane t / 4 + 8.
__device__ __forceinline__ void ld_16x32(uint32_t taddr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void ld_16x16(uint32_t taddr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ void stmatrix_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case ACT_SIGMOID: return 1.0f / (1.0f + expf(-v));
    case ACT_RELU: return v < 0.0f ? 0.0f : v;
    case ACT_TANH: return tanhf(v);
    case ACT_CLIP: return fminf(fmaxf(v, 0.0f), 6.0f);
    case ACT_SILU:
    case ACT_GATED_SILU: return v / (1.0f + expf(-v));
    default: return v;
  }
}
__device__ __forceinline__ uint32_t pack16(float a, float b, int type) {
  return type == ELEM_F16 ? f2_to_bf16x2<true>(f2_pack(a, b)) : f2_to_bf16x2<false>(f2_pack(a, b));
}
__device__ __forceinline__ void store_one(const PtParams &p, int64_t at, float v) {
  if (p.out_type == ELEM_F32) ((float *)p.out)[at] = v;
  else if (p.out_type == ELEM_BF16) ((__nv_bfloat16 *)p.out)[at] = __float2bfloat16_rn(v);
  else ((__half *)p.out)[at] = __float2half_rn(v);
}

struct PtTile {
  int g, m0, rows, n0;   // group, first row, rows in the tile, first weight (of a gated pair)
};

// A thread's sums: acc[h][g][0, 1] of weight 16 h + t / 4 and columns 8 g + 2 (t % 4) + 0, 1 of its warp's share, [2, 3] the
// same of weight 16 h + t / 4 + 8.
template <int BN, bool SCALED, bool GATED>
__global__ void __launch_bounds__(PT_THREADS, BN <= 64 ? 2 : 1) block_product_kernel(const __grid_constant__ PtParams p) {
  constexpr int CW = BN / 2;             // columns of an epilogue warp
  constexpr int NG = CW / 8;             // groups of eight of them
  constexpr int SETS = GATED ? 2 : 1;    // scales of a column: first and second matrix
  constexpr int TILE_N = GATED ? PT_ROWS / 2 : PT_ROWS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if ((smem_u32(smem_raw) & 1023u) != 0u) {
    if (threadIdx.x == 0) atomicExch(p.err, 1007);
    return;
  }
  const int stages = p.stages, bufs = p.bufs;
  constexpr uint32_t W_BYTES = PT_ROWS * 128, R_BYTES = BN * 128;
  const uint32_t sW = smem_u32(smem_raw), sR = sW + stages * W_BYTES;
  uint8_t *misc = smem_raw + stages * (W_BYTES + R_BYTES);
  uint8_t *stage_out = misc;                                                      // 1 KB for each epilogue warp
  float *scales = reinterpret_cast<float *>(misc + PT_EPI_WARPS * 1024);          // [bufs][SETS][BN]
  uint64_t *bars = reinterpret_cast<uint64_t *>(scales + (SCALED ? bufs * SETS * BN : 0));
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (stages + s); };
  auto tfull_bar = [&](int b) { return bar0 + 8u * (2 * stages + b); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * stages + bufs + b); };
  auto sfull_bar = [&](int b) { return bar0 + 8u * (2 * stages + 2 * bufs + b); };
  int32_t *words = reinterpret_cast<int32_t *>(bars + 2 * stages + 3 * bufs);
  volatile uint32_t *tmem_holder = reinterpret_cast<volatile uint32_t *>(words);
  volatile int *abort_flag = words + 1;
  int32_t *first = words + 4, *last = first + p.groups, *before = last + p.groups;   // rows of a group; row tiles before it

  const int warp = warp_index(), lane = threadIdx.x & 31;
  constexpr uint32_t COLS = BN == 256 ? 512 : (BN == 128 ? 512 : BN * 4);
  if (threadIdx.x == 0) {
    tma_prefetch_map(&p.ta);
    tma_prefetch_map(&p.tb);
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < bufs; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), PT_EPI_WARPS);
      mbar_init(sfull_bar(b), 2);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32((const void *)tmem_holder)),
                 "r"(COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_launch_dependents();
  pdl_wait();
  // the groups' rows, cut off at [0, rows], and how many row tiles come before each
  for (int g = threadIdx.x; g < p.groups; g += PT_THREADS) {
    const int lo = p.offsets ? min(max(p.offsets[g], 0), p.rows) : 0;
    first[g] = lo;
    last[g] = p.offsets ? min(max(p.offsets[g + 1], lo), p.rows) : p.rows;
  }
  __syncthreads();
  if (warp == 0) {
    int sum = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
      const int g = g0 + lane, n = g < p.groups ? (last[g] - first[g] + BN - 1) / BN : 0;
      int upto = n;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
      }
      if (g < p.groups) before[g] = sum + upto - n;
      sum += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) before[p.groups] = sum;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int splits = p.splits, rank = splits > 1 ? (int)cluster_ctarank() : 0;
  const int total = (int)min((int64_t)before[p.groups] * p.tiles_n, (int64_t)0x7fffffff);
  const int tile0 = (int)blockIdx.x / splits, tstep = (int)gridDim.x / splits;
  const int k0 = (int)((int64_t)p.kblocks * rank / splits), k1 = (int)((int64_t)p.kblocks * (rank + 1) / splits);
  constexpr int PER = SCALED ? 1 : PT_PER;
  int err_code = 0;

  auto decode = [&](int tile) {
    const int t = tile / p.tiles_n;
    int lo = 0, hi = p.groups - 1;          // last group with before[g] <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (before[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    const int local = tile - before[lo] * p.tiles_n, all = before[lo + 1] - before[lo];
    const int band = local / (PT_RASTER * p.tiles_n), in_band = local - band * PT_RASTER * p.tiles_n;
    const int height = min(PT_RASTER, all - band * PT_RASTER), n = in_band / height;
    const int m = band * PT_RASTER + in_band - n * height;
    PtTile tl;
    tl.g = lo;
    tl.m0 = first[lo] + m * BN;
    tl.rows = min(BN, last[lo] - tl.m0);
    tl.n0 = n * TILE_N;
    return tl;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    int stage = 0;
    uint32_t phase = 0;
    for (int tile = tile0; tile < total && !err_code; tile += tstep) {
      const PtTile tl = decode(tile);
      int4 rows4[BN > 128 ? 2 : 1];
      const int n4 = (tl.rows + 3) / 4;
      if (p.index) {
#pragma unroll
        for (int i = 0; i < (BN > 128 ? 2 : 1); ++i) {
          int r[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {   // a row that there is not, or none, reads as zeros
            const int m = (lane + 32 * i) * 4 + j;
            r[j] = m < tl.rows ? p.index[tl.m0 + m] : -1;
            if (r[j] < 0 || r[j] >= p.a_rows) r[j] = p.a_rows;
          }
          rows4[i] = make_int4(r[0], r[1], r[2], r[3]);
        }
      }
      const int boxes = (tl.rows + PT_BOX - 1) / PT_BOX;
      const uint32_t bytes = W_BYTES + (p.index ? (uint32_t)n4 * 512u : (uint32_t)boxes * (PT_BOX * 128u));
      for (int kb = k0; kb < k1; ++kb) {
        if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag)) {
          err_code = 1;
          break;
        }
        const int k = kb * (SCALED ? 128 : 64);
        expect_tx_warp(full_bar(stage), bytes);
        if constexpr (GATED) load_5d_warp(sW + stage * W_BYTES, &p.tb, full_bar(stage), k, tl.n0 / 8, tl.g);
        else load_2d_warp(sW + stage * W_BYTES, &p.tb, full_bar(stage), k, tl.g * p.N + tl.n0);
        const uint32_t dst = sR + stage * R_BYTES;
        if (p.index) {
#pragma unroll
          for (int i = 0; i < (BN > 128 ? 2 : 1); ++i)
            if (lane + 32 * i < n4)
              gather_4_rows(dst + (lane + 32 * i) * 512u, &p.ta, full_bar(stage), k, rows4[i]);
          __syncwarp();
        } else {
          for (int b = 0; b < boxes; ++b)
            load_2d_warp(dst + b * (PT_BOX * 128u), &p.ta, full_bar(stage), k, tl.m0 + b * PT_BOX);
        }
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // Nothing may be under way to this CTA's memory when it ends: no arrivals of the last MMAs, and after an error no copies
    // (the flag that ends other waits is set by then; these have their own).
    int unset = 0;
    for (int s = 0; s < stages; ++s) {
      const uint32_t last_use = s < stage ? phase : phase ^ 1u;
      mbar_wait_warp(err_code ? full_bar(s) : empty_bar(s), last_use, err_code ? &unset : abort_flag);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMAs
    int stage = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0;
    const uint64_t w0 = make_smem_desc(sW, 64), r0 = make_smem_desc(sR, 64);
    const uint32_t hi = (uint32_t)(w0 >> 32), w_lo = (uint32_t)w0, r_lo = (uint32_t)r0;
    for (int tile = tile0; tile < total && !err_code; tile += tstep) {
      const PtTile tl = decode(tile);
      const uint32_t idesc = p.idesc | ((uint32_t)((tl.rows + 15) / 16 * 2) << 17);
      int in_chunk = 0;
      for (int kb = k0; kb < k1; ++kb) {
        if (in_chunk == 0 && !mbar_wait_warp(tempty_bar(buf), buf_phase ^ 1u, abort_flag)) {
          err_code = 2;
          break;
        }
        if (!mbar_wait_warp(full_bar(stage), phase, abort_flag)) {
          err_code = 3;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf * BN);
        const uint32_t a = w_lo + (uint32_t)stage * (W_BYTES >> 4), b = r_lo + (uint32_t)stage * (R_BYTES >> 4);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          pt_mma<SCALED>(d, a + 2u * kk, hi, b + 2u * kk, hi, idesc, kk ? 1u : (uint32_t)(in_chunk != 0));
        commit_warp(empty_bar(stage));
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
        if (++in_chunk == PER || kb + 1 == k1) {
          commit_warp(tfull_bar(buf));
          in_chunk = 0;
          if (++buf == bufs) {
            buf = 0;
            buf_phase ^= 1u;
          }
        }
      }
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------ scales
    // sA * sB of every column, one k-step after another, in the order in which a thread wants them: four together for the
    // two columns each of two neighbouring groups.
    if constexpr (SCALED) {
      constexpr int MINE = (BN + 63) / 64;
      const int t = threadIdx.x - 64;
      int buf = 0;
      uint32_t buf_phase = 0;
      for (int tile = tile0; tile < total && !err_code; tile += tstep) {
        const PtTile tl = decode(tile);
        const float *sa[MINE];
        int at[MINE];
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          const int c = t + 64 * i;
          int row = c < tl.rows ? (p.index ? p.index[tl.m0 + c] : tl.m0 + c) : -1;
          sa[i] = row >= 0 && row < p.a_rows ? p.scale_a + (int64_t)row * p.kblocks : nullptr;
          at[i] = (c >> 4) * 16 + ((c >> 1) & 3) * 4 + ((c >> 3) & 1) * 2 + (c & 1);
        }
        const float *sb = p.scale_b + ((int64_t)tl.g * SETS * p.blocks_n + tl.n0 / SCALE_BLOCK) * p.kblocks;
        const int64_t second = (int64_t)p.blocks_n * p.kblocks;
        for (int kq = k0; kq < k1; kq += 4) {
          float va[MINE][4], vb[SETS][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int i = 0; i < MINE; ++i) va[i][j] = sa[i] && kq + j < k1 ? __ldg(sa[i] + kq + j) : 0.0f;
#pragma unroll
            for (int h = 0; h < SETS; ++h) vb[h][j] = kq + j < k1 ? __ldg(sb + h * second + kq + j) : 0.0f;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (kq + j >= k1 || err_code) continue;
            if (!mbar_wait_warp(tempty_bar(buf), buf_phase ^ 1u, abort_flag)) {
              err_code = 4;
              continue;
            }
            float *dst = scales + buf * (SETS * BN);
#pragma unroll
            for (int i = 0; i < MINE; ++i)
#pragma unroll
              for (int h = 0; h < SETS; ++h)
                if (BN >= 64 || t + 64 * i < BN) dst[h * BN + at[i]] = va[i][j] * vb[h][j];
            __syncwarp();
            if (lane == 0) mbar_arrive(sfull_bar(buf));
            if (++buf == bufs) {
              buf = 0;
              buf_phase ^= 1u;
            }
          }
          if (err_code) break;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ sums and results
    const int ew = warp - 4, quad = ew & 3, c0 = (ew >> 2) * CW;   // a warp reads the TMEM lanes of its own quadrant
    const int r8 = lane >> 2, q = lane & 3;
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int tile = tile0; tile < total && !err_code; tile += tstep) {
      const PtTile tl = decode(tile);
      uint64_t acc[2][NG][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < NG; ++g) acc[h][g][0] = acc[h][g][1] = 0;
      for (int kb = k0; kb < k1; kb += PER) {
        if (SCALED && !mbar_wait_warp(sfull_bar(buf), buf_phase, abort_flag)) {
          err_code = 5;
          break;
        }
        if (!mbar_wait_warp(tfull_bar(buf), buf_phase, abort_flag)) {
          err_code = 5;
          break;
        }
        tc_fence_after();
        constexpr int SG = CW >= 32 ? 4 : 2;     // groups of one step
        const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN + c0);
        const float *sc = scales + buf * (SETS * BN) + c0 + q * 4;
#pragma unroll
        for (int s = 0; s < NG; s += SG) {
          uint32_t v[2][SG * 4];
          uint4 f[SETS][SG / 2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if constexpr (SG == 4) ld_16x32(from + ((uint32_t)(h * 16) << 16) + (uint32_t)(s * 8), v[h]);
            else ld_16x16(from + ((uint32_t)(h * 16) << 16) + (uint32_t)(s * 8), v[h]);
          if constexpr (SCALED) {
#pragma unroll
            for (int m = 0; m < SETS; ++m)
#pragma unroll
              for (int i = 0; i < SG / 2; ++i)
                f[m][i] = *reinterpret_cast<const uint4 *>(sc + m * BN + (s / 2 + i) * 16);
          }
          tc_ld_wait();
          if (s + SG == NG) {   // the last of this buffer has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar(buf));
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int g = 0; g < SG; ++g)
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                const uint64_t x = pair_of(v[h][4 * g + 2 * m], v[h][4 * g + 2 * m + 1]);
                uint64_t &y = acc[h][s + g][m];
                if constexpr (SCALED) {
                  const uint4 w = f[GATED ? m : 0][g / 2];
                  y = f2_fma(x, g & 1 ? pair_of(w.z, w.w) : pair_of(w.x, w.y), y);
                } else {
                  y = f2_add(x, y);
                }
              }
        }
        if (++buf == bufs) {
          buf = 0;
          buf_phase ^= 1u;
        }
      }
      if (splits > 1 || err_code) break;
      // ---- results of a whole tile
      const int n_tile = min(TILE_N, p.N - tl.n0);
      float bias[2][2] = {};
      if (p.bias) {
        const float *bp = p.bias + (int64_t)tl.g * SETS * p.N + tl.n0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const int n = GATED ? quad * 16 + h * 8 + r8 : quad * 32 + h * 16 + m * 8 + r8;
            if (n < n_tile) bias[h][m] = bp[(GATED ? (int64_t)m * p.N : 0) + n];
          }
      }
      const uint32_t so = smem_u32(stage_out) + ew * 1024;
#pragma unroll
      for (int g = 0; g < NG; g += 2) {      // sixteen rows at a time
        if (c0 + g * 8 >= tl.rows) break;
        float r[2][2][2][2];                 // [group][h][m][column]
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x[2][2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              f2_unpack(acc[h][g + i][m], x[m][0], x[m][1]);
              x[m][0] += bias[h][m];
              x[m][1] += bias[h][m];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              r[i][h][0][c] = GATED ? activate(x[0][c], ACT_GATED_SILU) * x[1][c] : activate(x[0][c], p.act);
              r[i][h][1][c] = GATED ? 0.0f : activate(x[1][c], p.act);
            }
          }
        if (p.vec_out) {
          // 16-bit, through shared memory: [row][8 weights of 16 bytes], four (gated: two) such pieces a row
          __syncwarp();
          if constexpr (GATED) {
            const int row = (lane & 7) + ((lane >> 4) & 1) * 8, piece = (lane >> 3) & 1;
            stmatrix_trans(so + row * 32 + (piece ^ ((row >> 2) & 1)) * 16, pack16(r[0][0][0][0], r[0][0][0][1], p.out_type),
                           pack16(r[0][1][0][0], r[0][1][0][1], p.out_type), pack16(r[1][0][0][0], r[1][0][0][1], p.out_type),
                           pack16(r[1][1][0][0], r[1][1][0][1], p.out_type));
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int row = (lane & 7) + i * 8, piece = lane >> 3;
              stmatrix_trans(so + row * 64 + (piece ^ ((row >> 1) & 3)) * 16, pack16(r[i][0][0][0], r[i][0][0][1], p.out_type),
                             pack16(r[i][0][1][0], r[i][0][1][1], p.out_type), pack16(r[i][1][0][0], r[i][1][0][1], p.out_type),
                             pack16(r[i][1][1][0], r[i][1][1][1], p.out_type));
            }
          }
          __syncwarp();
          constexpr int PIECES = GATED ? 2 : 4;
#pragma unroll
          for (int i = 0; i < 16 * PIECES / 32; ++i) {
            const int row = (lane + 32 * i) / PIECES, piece = lane % PIECES;
            const int m = c0 + g * 8 + row, n = quad * (PIECES * 8) + piece * 8;
            if (m >= tl.rows || n >= n_tile) continue;
            const uint4 v = *reinterpret_cast<const uint4 *>(
                stage_out + ew * 1024 + row * (PIECES * 16) +
                (GATED ? (piece ^ ((row >> 2) & 1)) : (piece ^ ((row >> 1) & 3))) * 16);
            uint16_t *dst = (uint16_t *)p.out + (int64_t)(tl.m0 + m) * p.ldo + tl.n0 + n;
            if (n + 8 <= n_tile) {
              *reinterpret_cast<uint4 *>(dst) = v;
            } else {
              const uint16_t *e = reinterpret_cast<const uint16_t *>(&v);
              for (int j = 0; n + j < n_tile; ++j) dst[j] = e[j];
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int m = 0; m < (GATED ? 1 : 2); ++m)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const int row = c0 + (g + i) * 8 + q * 2 + c;
                  const int n = GATED ? quad * 16 + h * 8 + r8 : quad * 32 + h * 16 + m * 8 + r8;
                  if (row < tl.rows && n < n_tile) store_one(p, (int64_t)(tl.m0 + row) * p.ldo + tl.n0 + n, r[i][h][m][c]);
                }
        }
      }
    }
  }
  if (err_code) {
    *abort_flag = 1;
    if (lane == 0) atomicExch(p.err, 1000 + err_code);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
  }
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

bool encode(CUtensorMap *m, int type, const void *ptr, int rank, const cuuint64_t *dims, const cuuint64_t *strides,
            const cuuint32_t *box) {
  static EncodeFn fn = [] {
    void *sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess) cudaGetLastError();
    return (EncodeFn)sym;
  }();
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType t = type == ELEM_E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  count(CNT_TMAP_ENCODES);
  return fn && fn(m, t, (cuuint32_t)rank, const_cast<void *>(ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
                   CUDA_SUCCESS;
}

template <int BN, bool SCALED, bool GATED>
cudaError_t launch_tiles(PtParams &p, int64_t most_tiles, int num_sms, cudaStream_t s) {
  constexpr size_t LIMIT = BN <= 64 ? TC_SMEM_DUO : TC_SMEM_LIMIT;
  p.bufs = BN == 256 ? 2 : 4;
  const size_t misc = PT_EPI_WARPS * 1024 + (SCALED ? p.bufs * (GATED ? 2 : 1) * BN * 4 : 0) + 8 * 3 * 4 + 16 +
                      (3 * (size_t)p.groups + 1) * 4;
  const size_t stage = (PT_ROWS + BN) * 128 + 16;
  p.stages = (int)std::min<size_t>((LIMIT - misc) / stage, 16);
  const size_t smem = p.stages * stage + misc;
  // the attribute is the device's: set for each once
  static std::once_flag once[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::call_once(once[dev & 63], [] {
    cudaFuncSetAttribute(block_product_kernel<BN, SCALED, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)LIMIT);
  });
  p.splits = 1;
  const int64_t resident = (int64_t)num_sms * (BN <= 64 ? 2 : 1);
  const int64_t grid = std::min<int64_t>(most_tiles, resident);
  return launch_after(block_product_kernel<BN, SCALED, GATED>, dim3((unsigned)grid), dim3(PT_THREADS), smem, s, p);
}

template <int BN>
cudaError_t launch_width(PtParams &p, bool scaled, int64_t most_tiles, int num_sms, cudaStream_t s) {
  if (scaled)
    return p.gated ? launch_tiles<BN, true, true>(p, most_tiles, num_sms, s)
                   : launch_tiles<BN, true, false>(p, most_tiles, num_sms, s);
  return p.gated ? launch_tiles<BN, false, true>(p, most_tiles, num_sms, s)
                 : launch_tiles<BN, false, false>(p, most_tiles, num_sms, s);
}

}  // namespace

cudaError_t launch_product(const ProductArgs &a, int num_sms, cudaStream_t s) {
  PtParams p;
  memset(&p, 0, sizeof(p));
  const bool scaled = a.type == ELEM_E4M3;
  const int es = elem_size(a.type), bk = 128 / es;
  p.gated = a.act == ACT_GATED_SILU;
  {
    const cuuint64_t dims[2] = {(cuuint64_t)a.K, (cuuint64_t)a.a_rows}, strides[1] = {(cuuint64_t)a.lda * es};
    const cuuint32_t box[2] = {(cuuint32_t)bk, a.index ? 1u : (cuuint32_t)PT_BOX};
    if (!encode(&p.ta, a.type, a.a, 2, dims, strides, box)) return cudaErrorInvalidValue;
  }
  if (p.gated) {
    // eight rows of the first matrix, the same eight of the second, and so on: both halves of a result meet in a thread
    const cuuint64_t ld = (cuuint64_t)a.ldb * es;
    const cuuint64_t dims[5] = {(cuuint64_t)a.K, 8, 2, (cuuint64_t)a.N / 8, (cuuint64_t)a.groups};
    const cuuint64_t strides[4] = {ld, ld * a.N, ld * 8, ld * a.N * 2};
    const cuuint32_t box[5] = {(cuuint32_t)bk, 8, 2, 8, 1};
    if (!encode(&p.tb, a.type, a.b, 5, dims, strides, box)) return cudaErrorInvalidValue;
  } else {
    const cuuint64_t dims[2] = {(cuuint64_t)a.K, (cuuint64_t)(a.N * a.groups)}, strides[1] = {(cuuint64_t)a.ldb * es};
    const cuuint32_t box[2] = {(cuuint32_t)bk, PT_ROWS};
    if (!encode(&p.tb, a.type, a.b, 2, dims, strides, box)) return cudaErrorInvalidValue;
  }
  p.index = a.index;
  p.offsets = a.offsets;
  p.scale_a = a.scale_a;
  p.scale_b = a.scale_b;
  p.bias = a.bias;
  p.out = a.out;
  p.ldo = a.ldo;
  p.a_rows = (int)a.a_rows;
  p.rows = (int)a.rows;
  p.groups = (int)a.groups;
  p.N = (int)a.N;
  p.act = a.act;
  p.out_type = a.out_type;
  p.kblocks = (int)((a.K + bk - 1) / bk);
  p.blocks_n = (int)scale_blocks(a.N);
  const int tile_n = p.gated ? PT_ROWS / 2 : PT_ROWS;
  p.tiles_n = (int)((a.N + tile_n - 1) / tile_n);
  // F32 accumulator; the type of A and B (f16 0, bf16 1, e4m3 0); M = 128
  const uint32_t fmt = a.type == ELEM_BF16 ? 1u : 0u;
  p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(PT_ROWS >> 4) << 24);
  p.vec_out = a.out_type != ELEM_F32 && (uintptr_t)a.out % 16 == 0 && a.ldo % 8 == 0;
  p.err = a.err;
  const int64_t each = (a.rows + a.groups - 1) / a.groups;
  const int BN = each <= 32 ? 32 : (each <= 64 ? 64 : (each <= 128 ? 128 : 256));
  const int64_t most_tiles = std::min<int64_t>((std::min(a.groups, a.rows) + a.rows / BN) * p.tiles_n, 1 << 30);
  switch (BN) {
    case 32: return launch_width<32>(p, scaled, most_tiles, num_sms, s);
    case 64: return launch_width<64>(p, scaled, most_tiles, num_sms, s);
    case 128: return launch_width<128>(p, scaled, most_tiles, num_sms, s);
    default: return launch_width<256>(p, scaled, most_tiles, num_sms, s);
  }
}

}  // namespace occ
