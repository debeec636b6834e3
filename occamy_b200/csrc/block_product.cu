// Products of rows with weights, act(A B^T + bias): block-scaled e4m3, and rows in ragged groups that each have a matrix
// of their own (occamy_matmul_e4m3, occamy_matmul_grouped).
//
//   out[m][n] = act( sum over blocks j of 128 along K:  sA[m][j] * sB[n / 128][j] * sum over k in j: a[m][k] b[n][k]   + bias[n] )
//
// In this form the weights are the M side of the tensor core's tile (128 of them, to the TMEM lanes) and the rows its
// N side (the columns): N may be any multiple of 16, so that a group of a few rows takes a narrow tile and the last tile of a
// group no more than it has, where 128 rows on the M side would be multiplied whatever there are.
//
// The tensor core adds the products of one k-step (128 bytes of K) into a TMEM buffer; epilogue warps take each
// finished buffer, multiply it by its scales and add it to sums they hold in registers, fp32.  A column's scale comes from
// shared memory, which is as much as these tiles' k-steps of memory time have room for; many rows of e4m3 take the other
// form (block_product_wide.cu).  16-bit operands have no scales, but go the same way every few k-steps: the tensor core
// truncates when it adds to its accumulator, an error that grows with the number of additions.
//
// With few tiles the CTAs of a cluster share a tile's K and add up their sums in rank order through each other's
// shared memory: no workspace, and the same bits every time.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>

#include "block_product_dev.cuh"
#include "runtime.h"

namespace occ {
namespace {

constexpr int PT_ROWS = 128;           // weights of a tile
constexpr int PT_PER = 4;              // k-steps of 16-bit operands that the tensor core adds up by itself

__device__ __forceinline__ float2 ld_cluster_f32x2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

template <int BN, bool SCALED, bool GATED>
__global__ void __launch_bounds__(PT_THREADS, BN <= 64 ? 2 : 1) block_product_kernel(const __grid_constant__ PtParams p) {
  constexpr int EW = PT_EPI_WARPS;
  constexpr int CW = BN / (EW / 4);      // columns of an epilogue warp
  constexpr int NG = CW / 8;             // groups of eight of them
  // Columns of one TMEM load.  (Of 64 columns 16: with 32 the code around the sums decided whether 256 x 4096 x 25088 took 50 or 58 us.)
  constexpr int LD = CW < 32 || BN == 128 ? 16 : 32;
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
  float *scales = reinterpret_cast<float *>(misc + EW * 1024);                    // [bufs][SETS][BN]
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
  const PtGroups groups = {words + 4, words + 4 + p.groups, words + 4 + 2 * p.groups};
  // of each buffer, for factors out of range: the powers that go with them ([SETS][BN]), whether a scale warp wants them applied, and a
  // barrier for the answer
  float *powers = reinterpret_cast<float *>(smem_raw + ((reinterpret_cast<uint8_t *>(words + 5 + 3 * p.groups) - smem_raw + 15) & ~15));
  volatile int *wanted = reinterpret_cast<volatile int *>(powers + bufs * SETS * BN);
  const uint32_t applied0 = smem_u32(powers + bufs * SETS * BN + 2 * bufs);
  auto applied_bar = [&](int b, int w) { return applied0 + 8u * (2 * b + w); };

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const bool indexed = BN < 256 && p.index;   // (choose_rows)
  constexpr uint32_t COLS = BN >= 128 ? 512 : BN * 4;
  if (threadIdx.x == 0) {
    if (!indexed) tma_prefetch_map(&p.ta);
    tma_prefetch_map(&p.tb);
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), indexed ? 1 + 32 * PT_GATHERERS : 1);   // loads, lanes that copy rows chosen by an index
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < bufs; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), EW);
      mbar_init(sfull_bar(b), 2);
      if constexpr (SCALED)
        for (int w = 0; w < 2; ++w) {
          mbar_init(applied_bar(b, w), EW);
          wanted[2 * b + w] = 0;
        }
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
    // (not before: a CTA of the next kernel that took the columns first would keep them until this one ends)
    pdl_launch_dependents();
  }
  // (without offsets nothing here was written by the kernel before: this much of the start goes on beside its end)
  if (p.offsets) pdl_wait();
  pt_read_groups<PT_THREADS>(p, groups);
  __syncthreads();
  if (warp == 0) pt_count_tiles<BN>(p, groups, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (!p.offsets) pdl_wait();
  const uint32_t tmem = *tmem_holder;
  const int splits = p.splits, rank = splits > 1 ? (int)cluster_ctarank() : 0;
  const int total = pt_total(p, groups);
  // CTAs that share a tile's K do one tile (and there are enough of them for all)
  const int tile0 = (int)blockIdx.x / splits, tstep = splits > 1 ? 0x40000000 : (int)gridDim.x;
  const int k0 = (int)((int64_t)p.kblocks * rank / splits), k1 = (int)((int64_t)p.kblocks * (rank + 1) / splits);
  constexpr int PER = SCALED ? 1 : PT_PER;
  int err_code = 0;
  auto decode = [&](int tile) { return pt_decode<BN, TILE_N>(p, groups, tile); };
  // By all warps.  CTAs of a cluster do it before they wait for each other: one that waited with its columns for a CTA that waits for
  // columns could do so for good, if what holds those waits in the same way (another kernel's cluster, on another stream).
  auto free_tmem = [&] {
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
    }
  };

  // An epilogue warp's place.
  const int ew = warp - PT_EPI_WARP, quad = warp & 3, c0 = (ew >> 2) * CW;

  // Eight rows of results (columns c0 + 8 g ...) through 1 KB of shared memory, [row][32 weights].  There is one copy of the
  // code behind it: with the activations of all sums unrolled, fetching instructions took 30 us a tile.
  const int row = lane >> 2, piece = lane & 3;
  constexpr int W = GATED ? 4 : 8;                       // results of a lane
  const int n_lane = quad * (W * 4) + piece * W;
  float *buf_out = reinterpret_cast<float *>(stage_out + (ew & (EW - 1)) * 1024);
  auto finish = [&](const PtTile &tl, int g, auto &&sum_of) {
    const int n_tile = min(TILE_N, p.N - tl.n0);
    __syncwarp();
    sum_of(g, [&](int j, float a, float b) {   // columns 2 j, 2 j + 1 of the eight
      buf_out[(2 * j) * 32 + lane] = a;
      buf_out[(2 * j + 1) * 32 + lane] = b;
    });
    __syncwarp();
    const int m = c0 + g * 8 + row;
    if (m >= tl.rows || n_lane >= n_tile) return;
    const float *src = buf_out + row * 32;
    const float *bias = p.bias ? p.bias + (int64_t)tl.g * SETS * p.N + tl.n0 + n_lane : nullptr;
    float r[W];
    if constexpr (GATED) {
      // lanes 0-7, 16-23: first matrix; 8-15, 24-31: the same eight of the second
      const float4 a = *reinterpret_cast<const float4 *>(src + (piece >> 1) * 16 + (piece & 1) * 4);
      const float4 b = *reinterpret_cast<const float4 *>(src + (piece >> 1) * 16 + (piece & 1) * 4 + 8);
      const float x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool has = bias && n_lane + j < n_tile;
        r[j] = silu(x[j] + (has ? bias[j] : 0.0f)) * (y[j] + (has ? bias[p.N + j] : 0.0f));
      }
    } else {
      const float4 a = *reinterpret_cast<const float4 *>(src + piece * 8);
      const float4 b = *reinterpret_cast<const float4 *>(src + piece * 8 + 4);
      const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = x[j] + (bias && n_lane + j < n_tile ? bias[j] : 0.0f);
      if (p.act == ACT_RELU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = r[j] < 0.0f ? 0.0f : r[j];
      } else if (p.act != ACT_IDENTITY) {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = activate(r[j], p.act);
      }
    }
    store_row<W>(p, (uint8_t *)p.out + ((int64_t)(tl.m0 + m) * p.ldo + tl.n0 + n_lane) * (p.out_type == ELEM_F32 ? 4 : 2), r,
                 n_tile - n_lane);
  };

  // The sums' warps take the registers that the others do without: (256 x 48 + 256 x 208) = 512 x 128 (256 rows: 56 and 200, with
  // which nothing is spilled), of two CTAs (256 x 40 + 256 x 88) = 512 x 64.  (Each at the head of its roles: behind a point where both
  // come together the compiler keeps to the smaller number.)
  if (warp < PT_EPI_WARP) {
    if constexpr (BN <= 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    else if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 0) {
      // ------------------------------------------------------------ loads
      TCT_DECL
      int stage = 0;
      uint32_t phase = 0;
      for (int tile = tile0; tile < total && !err_code; tile += tstep) {
        const PtTile tl = decode(tile);
        const int boxes = indexed ? 0 : (tl.rows + PT_BOX - 1) / PT_BOX;
        const uint32_t bytes = W_BYTES + (uint32_t)boxes * (PT_BOX * 128u);
        for (int kb = k0; kb < k1; ++kb) {
          if (!TCT_WAIT(0, mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag))) {
            err_code = 1;
            break;
          }
          const int k = kb * (SCALED ? 128 : 64);
          expect_tx_warp(full_bar(stage), bytes);
          if constexpr (GATED) load_5d_warp(sW + stage * W_BYTES, &p.tb, full_bar(stage), k, tl.n0 / 8, tl.g);
          else load_2d_warp(sW + stage * W_BYTES, &p.tb, full_bar(stage), k, tl.g * p.N + tl.n0);
          const uint32_t dst = sR + stage * R_BYTES;
          for (int b = 0; b < boxes; ++b)
            load_2d_warp(dst + b * (PT_BOX * 128u), &p.ta, full_bar(stage), k, tl.m0 + b * PT_BOX);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      TCT_FLUSH(0)
      // Nothing may be under way to this CTA's memory when it ends: no arrivals of the last MMAs, and after an error no copies
      // (the flag that ends other waits is set by then; these have their own).
      int unset = 0;
      for (int s = 0; s < stages; ++s) {
        const uint32_t last_use = s < stage ? phase : phase ^ 1u;
        mbar_wait_warp(err_code ? full_bar(s) : empty_bar(s), last_use, err_code ? &unset : abort_flag);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMAs
      TCT_DECL
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      const uint64_t w0 = make_smem_desc(sW, 64), r0 = make_smem_desc(sR, 64);
      const uint32_t hi = (uint32_t)(w0 >> 32), w_lo = (uint32_t)w0, r_lo = (uint32_t)r0;
      for (int tile = tile0; tile < total && !err_code; tile += tstep) {
        const PtTile tl = decode(tile);
        const uint32_t idesc = p.idesc | ((uint32_t)((tl.rows + 15) / 16 * 2) << 17);
        int in_chunk = 0;
        for (int kb = k0; kb < k1; ++kb) {
          if (in_chunk == 0 && !TCT_WAIT(0, mbar_wait_warp(tempty_bar(buf), buf_phase ^ 1u, abort_flag))) {
            err_code = 2;
            break;
          }
          if (!TCT_WAIT(1, mbar_wait_warp(full_bar(stage), phase, abort_flag))) {
            err_code = 3;
            break;
          }
          if (indexed) fence_async_smem();
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
      TCT_FLUSH(1)
    } else if (warp >= PT_GATHER_WARP) {
      // ------------------------------------------------------------ rows chosen by an index
      if constexpr (BN < 256) {
        if (p.index)
          err_code = pt_gather_role<BN, PT_GATHERERS>(p, tile0, total, tstep, k0, k1, sR, stages, warp - PT_GATHER_WARP, lane, abort_flag,
                                                      decode, full_bar, empty_bar);
      }
    } else {
      // ------------------------------------------------------------ scales
      // sA * sB of every column, one k-step after another.
      if constexpr (SCALED) {
        TCT_DECL
        constexpr int MINE = BN <= 64 ? 1 : BN / 64;
        const int t = threadIdx.x - 64;
        int buf = 0;
        uint32_t buf_phase = 0, applied = 0;   // (a phase for each buffer)
        for (int tile = tile0; tile < total && !err_code; tile += tstep) {
          const PtTile tl = decode(tile);
          const float *sa[MINE];
#pragma unroll
          for (int i = 0; i < MINE; ++i) {
            const int c = t + 64 * i;
            const int r = c < tl.rows ? (p.index ? p.index[tl.m0 + c] : tl.m0 + c) : -1;
            sa[i] = r >= 0 && r < p.a_rows ? p.scale_a + (int64_t)r * p.kblocks : nullptr;
          }
          const float *sb = p.scale_b + ((int64_t)tl.g * SETS * p.blocks_n + tl.n0 / SCALE_BLOCK) * p.kblocks;
          const int64_t second = (int64_t)p.blocks_n * p.kblocks;
          float va[MINE][4], vb[SETS][4];
          auto fetch = [&](int kq) {   // 1 where there is none (the numbers of a row that an index does not give are zeros)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
              for (int i = 0; i < MINE; ++i) va[i][j] = sa[i] && kq + j < k1 ? __ldg(sa[i] + kq + j) : 1.0f;
#pragma unroll
              for (int h = 0; h < SETS; ++h) vb[h][j] = kq + j < k1 ? __ldg(sb + h * second + kq + j) : 1.0f;
            }
          };
          fetch(k0);
          for (int kq = k0; kq < k1 && !err_code; kq += 4) {
            uint32_t range = 0;   // of these four
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int i = 0; i < MINE; ++i)
#pragma unroll
                for (int h = 0; h < SETS; ++h) range = max(range, pt_range(va[i][j], vb[h][j]));
            const bool look = __any_sync(0xffffffffu, range > PT_RANGE);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (kq + j >= k1 || err_code) continue;
              if (!TCT_WAIT(0, mbar_wait_warp(tempty_bar(buf), buf_phase ^ 1u, abort_flag))) {
                err_code = 4;
                continue;
              }
              float *dst = scales + buf * (SETS * BN) + t;
#pragma unroll
              for (int i = 0; i < MINE; ++i)
#pragma unroll
                for (int h = 0; h < SETS; ++h)
                  if (BN >= 64 || t < BN) dst[h * BN + 64 * i] = va[i][j] * vb[h][j];
              if (look) {
                bool met = false;
                float *pow = powers + buf * (SETS * BN) + t;
#pragma unroll
                for (int i = 0; i < MINE; ++i)
#pragma unroll
                  for (int h = 0; h < SETS; ++h) {
                    float f;
                    const float power = pt_factor(va[i][j], vb[h][j], f);
                    met = met || power != 1.0f;
                    if (BN >= 64 || t < BN) dst[h * BN + 64 * i] = f, pow[h * BN + 64 * i] = power;
                  }
                if (__any_sync(0xffffffffu, met)) {
                  // The sums' warps find this while they wait for the scales, which do not arrive before it is done; their loop does not look
                  // for it.  (A word read in every k-step took 256 x 4096 x 25088 from 50 us to 52 at best, 60 at worst.)
                  __threadfence_block();
                  __syncwarp();
                  if (lane == 0) wanted[2 * buf + warp - 2] = 1;
                  if (!mbar_wait_warp(applied_bar(buf, warp - 2), applied >> buf & 1u, abort_flag)) {
                    err_code = 6;
                    continue;
                  }
                  applied ^= 1u << buf;
                  if (lane == 0) wanted[2 * buf + warp - 2] = 0;
                }
              }
              __syncwarp();
              if (lane == 0) mbar_arrive(sfull_bar(buf));
              if (++buf == bufs) {
                buf = 0;
                buf_phase ^= 1u;
              }
            }
            if (kq + 4 < k1) fetch(kq + 4);
          }
        }
        if (warp == 2) { TCT_FLUSH(2) }
      }
    }
    if (splits > 1) {   // where the sums' warps meet, the CTAs of the cluster among them
      __syncwarp();
      free_tmem();
      cluster_sync_all();
    }
  } else {
    // ------------------------------------------------------------ sums and results
    if constexpr (BN <= 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
    else if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    TCT_DECL
    // For a buffer's scales; applies the powers that a scale warp wants before they arrive, to its 32 columns of every 64.
    auto wait_scales = [&](const PtTile &tl, int buf, uint32_t phase) {
      if (__all_sync(0xffffffffu, mbar_try(sfull_bar(buf), phase))) return true;
      const long long t0 = clock64();
      int done = 0;
      for (int it = 1; !__all_sync(0xffffffffu, mbar_try(sfull_bar(buf), phase)); ++it) {
        for (int w = 0; w < 2; ++w) {
          if (done >> w & 1 || !__shfl_sync(0xffffffffu, wanted[2 * buf + w], 0)) continue;
          __threadfence_block();
          if (!mbar_wait_warp(tfull_bar(buf), phase, abort_flag)) return false;
          tc_fence_after();
          if (c0 < tl.rows) {
            const int at = buf * (SETS * BN) + (GATED ? ((lane >> 3) & 1) * BN : 0) + c0;
#pragma unroll 1
            for (int s = 0; s < CW; s += 16)
              if (((c0 + s) / 32 & 1) == w) pt_rescale(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN + c0 + s), powers + at + s);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          }
          done |= 1 << w;
          __syncwarp();
          if (lane == 0) mbar_arrive(applied_bar(buf, w));
        }
        if ((it & 15) == 0) {
          const bool late = clock64() - t0 > 4000000000LL;
          if (__any_sync(0xffffffffu, *abort_flag != 0 || late)) {
            if (late) *abort_flag = 1;
            return false;
          }
        }
      }
      return true;
    };
    uint64_t acc[CW / 2];                  // sums of weight `lane` of the quadrant and columns c0 + 2 i, 2 i + 1
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int tile = tile0; tile < total && !err_code; tile += tstep) {
      const PtTile tl = decode(tile);
      if (splits > 1 && p.bias && n_lane < p.N - tl.n0)   // there when the sums are
        asm volatile("prefetch.global.L1 [%0];" ::"l"(p.bias + (int64_t)tl.g * SETS * p.N + tl.n0 + n_lane));
#pragma unroll
      for (int i = 0; i < CW / 2; ++i) acc[i] = 0;
      for (int kb = k0; kb < k1; kb += PER) {
        if (SCALED && !TCT_WAIT(0, wait_scales(tl, buf, buf_phase))) {
          err_code = 5;
          break;
        }
        if (!TCT_WAIT(1, mbar_wait_warp(tfull_bar(buf), buf_phase, abort_flag))) {
          err_code = 5;
          break;
        }
        tc_fence_after();
        const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN + c0);
        const float *sc = scales + buf * (SETS * BN) + (GATED ? ((lane >> 3) & 1) * BN : 0) + c0;
        // columns behind the tile's rows are not looked at
        if (c0 < tl.rows) {
#pragma unroll
          for (int s = 0; s < CW; s += LD) {
            uint32_t v[LD];
            tc_ld<LD>(from + s, v);
            if constexpr (SCALED) {
              uint4 f[LD / 4];
#pragma unroll
              for (int i = 0; i < LD / 4; ++i) f[i] = *reinterpret_cast<const uint4 *>(sc + s + 4 * i);
              tc_ld_wait();
#pragma unroll
              for (int i = 0; i < LD / 4; ++i) {
                uint64_t *y = acc + (s + 4 * i) / 2;
                y[0] = f2_fma(pair_of(v[4 * i], v[4 * i + 1]), pair_of(f[i].x, f[i].y), y[0]);
                y[1] = f2_fma(pair_of(v[4 * i + 2], v[4 * i + 3]), pair_of(f[i].z, f[i].w), y[1]);
              }
            } else {
              tc_ld_wait();
#pragma unroll
              for (int i = 0; i < LD / 2; ++i) acc[s / 2 + i] = f2_add(pair_of(v[2 * i], v[2 * i + 1]), acc[s / 2 + i]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(buf));
        if (++buf == bufs) {
          buf = 0;
          buf_phase ^= 1u;
        }
      }
      if (splits > 1 || err_code) break;
      if (p.vec_out && (GATED || p.act == ACT_IDENTITY || p.act == ACT_RELU) && (tl.n0 + TILE_N <= p.N || p.N % 8 == 0)) {
        // straight through all sums: a loop over them, as below, waits for one group's stores after another's loads
        uint8_t *out = (uint8_t *)p.out + ((int64_t)(tl.m0 + c0 + row) * p.ldo + tl.n0 + n_lane) * (p.out_type == ELEM_F32 ? 4 : 2);
        const int64_t step = p.ldo * (p.out_type == ELEM_F32 ? 32 : 16);
        const bool here = tl.n0 + n_lane < p.N;
        const float floor = !GATED && p.act == ACT_RELU ? 0.0f : -INFINITY;
        float bias[8] = {};                // of this lane's weights
        if (p.bias && here) {
          const float *from = p.bias + (int64_t)tl.g * SETS * p.N + tl.n0 + n_lane;
#pragma unroll
          for (int j = 0; j < 8; ++j) bias[j] = __ldg(from + (GATED && j >= 4 ? p.N + j - 4 : j));
        }
#pragma unroll
        for (int g = 0; g < NG; ++g, out += step) {
          if (c0 + g * 8 >= tl.rows) break;
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float a, b;
            f2_unpack(acc[g * 4 + j], a, b);
            buf_out[(2 * j) * 32 + lane] = a;
            buf_out[(2 * j + 1) * 32 + lane] = b;
          }
          __syncwarp();
          const float *src = buf_out + row * 32 + (GATED ? (piece >> 1) * 16 + (piece & 1) * 4 : piece * 8);
          const float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + (GATED ? 8 : 4));
          if (c0 + g * 8 + row < tl.rows && here) {
            float r[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] += bias[j];
            if constexpr (GATED) {
#pragma unroll
              for (int j = 0; j < 4; ++j) r[j] = silu(r[j]) * r[4 + j];
              store_row<4, true>(p, out, r, 4);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) asm("max.NaN.f32 %0, %0, %1;" : "+f"(r[j]) : "f"(floor));
              store_row<8, true>(p, out, r, 8);
            }
          }
        }
        continue;
      }
#pragma unroll 1
      for (int g = 0; g < NG && c0 + g * 8 < tl.rows; ++g)
        finish(tl, g, [&](int g, auto &&put) {
#pragma unroll
          for (int i = 0; i < NG; ++i)
            if (i == g)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float a, b;
                f2_unpack(acc[i * 4 + j], a, b);
                put(j, a, b);
              }
        });
    }
    if (ew == 0 || ew == EW - 1) { TCT_FLUSH(ew ? 4 : 3) }
    if (splits > 1) {
      // Every copy has landed and every MMA of the tile is complete: the ring holds the sums now, [column pair][thread].
      const bool mine = tile0 < total && !err_code;
      if (mine) {
        uint64_t *sums = reinterpret_cast<uint64_t *>(smem_raw);
#pragma unroll
        for (int i = 0; i < CW / 2; ++i) sums[i * (EW * 32) + threadIdx.x - 32 * PT_EPI_WARP] = acc[i];
      }
      __syncwarp();
      free_tmem();
      cluster_sync_all();
      if (mine) {
        const PtTile tl = decode(tile0);
#pragma unroll 1
        for (int g = 0; g < NG && c0 + g * 8 < tl.rows; ++g) {
          if ((ew * NG + g) % splits != rank) continue;
          // (all CTAs' sums on their way together: one after another took 2 us)
          float t[8] = {};
          const uint32_t from = sW + (uint32_t)(g * 4 * EW * 32 + (int)threadIdx.x - 32 * PT_EPI_WARP) * 8u;
          float2 x[8][4];
#pragma unroll
          for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              x[r][j] = r < splits ? ld_cluster_f32x2(cluster_map(from, (uint32_t)r) + j * (EW * 32 * 8)) : make_float2(0.0f, 0.0f);
#pragma unroll
          for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) t[2 * j] += x[r][j].x, t[2 * j + 1] += x[r][j].y;
          finish(tl, g, [&](int, auto &&put) {
#pragma unroll
            for (int j = 0; j < 4; ++j) put(j, t[2 * j], t[2 * j + 1]);
          });
        }
      }
      __syncwarp();
    }
  }
  if (err_code) {
    *abort_flag = 1;
    if (lane == 0) atomicExch(p.err, 1000 + err_code);
  }
  if (splits > 1) cluster_sync_all();   // nobody leaves while its sums are still to be read
  else free_tmem();
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

// CTAs that share a tile's K: as many as there is room for, eight k-steps for each.
int shares_of_k(int64_t tiles, int64_t resident, int kblocks) {
  int s = 1;
  while (s < 8 && tiles * s * 2 <= resident && kblocks >= s * 8) s *= 2;
  return s;
}

// Rows of a tile in the form of 256 rows: fewer where that comes to less time, for a group's last tile is cut off and a round of tiles
// may be nearly empty.  A tile takes as long as what it loads, 128 weights and its rows.  How many tiles several groups have is an
// estimate: fewer rows are taken when they are better by more than a few percent with two standard deviations more of tiles (of the
// groups' last ones, each anything between none and all of a tile).  (us with 256 rows and this way: 5003 rows in 8 groups, N = 1000,
// K = 1160 36.6 28.8; 16384 in 32, 1024, 2048 87 78; 1500 in one, 2048, 4096 29.0 27.4.)
int tile_height(const ProductArgs &a, int tiles_n, int num_sms) {
  const double live = (double)std::min(a.groups, a.rows);
  auto time = [&](int high, double more) {
    const double m = (double)a.rows / high;
    return std::ceil((a.groups == 1 ? std::ceil(m) : std::max(m + 0.5 * live + more, live)) * tiles_n / num_sms) * (PT_ROWS + high);
  };
  int best = 256;
  double least = (a.groups == 1 ? 1.0 : 0.94) * time(256, 0.0);
  for (int high = 240; high >= 128; high -= 16) {
    const double t = time(high, 0.58 * std::sqrt(live));
    if (t < least) best = high, least = t;
  }
  return best;
}

// Rows of a tile: 32, 64, 128 (e4m3; with 16 bits two CTAs of 64 were as fast) with the rows on the N side, two CTAs of the first two
// on an SM, or up to 256 (16-bit operands; e4m3: the wide form, 128 rows on the M side and 256 weights).  By the time that the tiles take
// in rounds of what is resident, from the measured times of a k-step, in hundredths of a microsecond.  (us with 32, 64 and 256 rows in
// bf16, 32, 64, 128 and 256 in e4m3: 4096 rows, N = 1000, K = 4096 63 45 32 and 60 46 37 25; 300 rows 15 15 19 and 15 14 14 22; 2000 rows
// in eight groups 37 29 31 and 34 26 36 24; 5000 in 32 89 74 66 and 76 64 60 48.)  Rows chosen by an index are copied at 18 bytes a
// cycle of an SM, whatever the form: 16-bit tiles of 256 rows would wait for them and do without an index (16384 rows in 32 groups, gated,
// 1024 x 2048 bf16: 32, 64 and 256 rows 259 199 264; without an index 266 172 144; later 195 and 141 for what is taken).
int choose_rows(const ProductArgs &a, bool scaled, bool gated, int kblocks, int num_sms) {
#ifdef OCCAMY_TUNING
  if (const char *e = getenv("OCCAMY_PT_BN")) return !scaled && a.index ? std::min(atoi(e), 64) : atoi(e);
#endif
  static const int rows_of[4] = {32, 64, 128, 256};
  static const int steps[3][4] = {{24, 32, 0, 40}, {43, 63, 50, 56}, {28, 42, 0, 0}};
  const int *step = steps[scaled ? 1 : a.index ? 2 : 0];
  const double live = (double)std::min(a.groups, a.rows);
  int best = 0;
  double least = 0;
  for (int i = 0; i < 4; ++i) {
    if (!step[i]) continue;
    const bool wide = scaled && i == 3;
    const double n = (wide ? 256 : PT_ROWS) / (gated ? 2 : 1);
    const int high = scaled || i < 3 ? rows_of[i] : tile_height(a, (int)std::ceil(a.N / n), num_sms);
    const double m = wide ? 128 : high;
    const double tiles = std::max(a.groups == 1 ? std::ceil(a.rows / m) : a.rows / m + 0.5 * live, live) * std::ceil(a.N / n);
    const double slots = (double)num_sms * (i < 2 ? 2 : 1);
    const int shares = i < 3 ? shares_of_k((int64_t)tiles, (int64_t)slots, kblocks) : 1;
    const double full = tiles * shares / slots, rounds = std::max(1.0, 0.5 * (full + std::ceil(full)));
    const double t = rounds * ((kblocks + shares - 1) / shares) * step[i] * (PT_ROWS + high) / (PT_ROWS + rows_of[i]) + (shares > 1 ? 300 : 0);
    if (i == 0 || t < least) best = i, least = t;
  }
  return rows_of[best];
}

template <int BN, bool SCALED, bool GATED>
cudaError_t launch_tiles(PtParams &p, int64_t most_tiles, int num_sms, cudaStream_t s) {
  constexpr size_t LIMIT = BN <= 64 ? TC_SMEM_DUO : TC_SMEM_LIMIT;
  constexpr int EW = PT_EPI_WARPS;
  p.bufs = BN == 256 ? 2 : 4;
  const size_t misc = EW * 1024 + (SCALED ? p.bufs * ((GATED ? 2 : 1) * BN * 8 + 24) + 16 : 0) + 8 * 3 * 4 + 16 +
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
    cudaFuncSetAttribute(block_product_kernel<BN, SCALED, GATED>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  });
  const int64_t resident = (int64_t)num_sms * (BN <= 64 ? 2 : 1);
  p.splits = BN <= 128 ? shares_of_k(most_tiles, resident, p.kblocks) : 1;
#ifdef OCCAMY_TUNING
  if (const char *e = getenv("OCCAMY_PT_SPLITS")) p.splits = atoi(e);
#endif
  if (p.splits > 1) count(CNT_PRODUCT_SHARED);
  const int64_t grid = p.splits > 1 ? most_tiles * p.splits : std::min<int64_t>(most_tiles, resident);
  return launch_after(block_product_kernel<BN, SCALED, GATED>, dim3((unsigned)grid), dim3(PT_THREADS), smem, s,
                      p.splits, p);
}

template <int BN, bool SCALED>
cudaError_t launch_width(PtParams &p, bool gated, int64_t most_tiles, int num_sms, cudaStream_t s) {
  return gated ? launch_tiles<BN, SCALED, true>(p, most_tiles, num_sms, s)
               : launch_tiles<BN, SCALED, false>(p, most_tiles, num_sms, s);
}

}  // namespace

cudaError_t launch_product(const ProductArgs &a, int num_sms, cudaStream_t s) {
  PtParams p;
  memset(&p, 0, sizeof(p));
  const bool scaled = a.type == ELEM_E4M3, gated = a.act == ACT_GATED_SILU;
  const int es = elem_size(a.type), bk = 128 / es;
  p.kblocks = (int)((a.K + bk - 1) / bk);
  const int BN = choose_rows(a, scaled, gated, p.kblocks, num_sms);
  const bool wide = scaled && BN == 256;
  p.a = (const uint8_t *)a.a;
  p.a_ld16 = (uint32_t)(a.lda * es / 16);
  p.k_bytes = (int)(a.K * es);
  if (!a.index) {
    const cuuint64_t dims[2] = {(cuuint64_t)a.K, (cuuint64_t)a.a_rows}, strides[1] = {(cuuint64_t)a.lda * es};
    const cuuint32_t box[2] = {(cuuint32_t)bk, (cuuint32_t)PT_BOX};
    if (!encode(&p.ta, a.type, a.a, 2, dims, strides, box)) return cudaErrorInvalidValue;
  }
  const cuuint32_t weights = wide ? 256 : 128;   // of one copy
  if (gated) {
    // eight rows of the first matrix, the same eight of the second, and so on: both halves of a result are near each other
    const cuuint64_t ld = (cuuint64_t)a.ldb * es;
    const cuuint64_t dims[5] = {(cuuint64_t)a.K, 8, 2, (cuuint64_t)a.N / 8, (cuuint64_t)a.groups};
    const cuuint64_t strides[4] = {ld, ld * a.N, ld * 8, ld * a.N * 2};
    const cuuint32_t box[5] = {(cuuint32_t)bk, 8, 2, weights / 16, 1};
    if (!encode(&p.tb, a.type, a.b, 5, dims, strides, box)) return cudaErrorInvalidValue;
  } else {
    const cuuint64_t dims[2] = {(cuuint64_t)a.K, (cuuint64_t)(a.N * a.groups)}, strides[1] = {(cuuint64_t)a.ldb * es};
    const cuuint32_t box[2] = {(cuuint32_t)bk, weights};
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
  p.blocks_n = (int)scale_blocks(a.N);
  // F32 accumulator; the type of A and B (f16 0, bf16 1, e4m3 0); M = 128
  const uint32_t fmt = a.type == ELEM_BF16 ? 1u : 0u;
  p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(128 >> 4) << 24);
  p.vec_out = (uintptr_t)a.out % 16 == 0 && a.ldo * elem_size(a.out_type) % 16 == 0;
  p.err = a.err;
#ifdef OCCAMY_TC_TIMERS
  p.timers = tc_timer_words();
#endif
  const int tile_n = (wide ? 256 : PT_ROWS) / (gated ? 2 : 1);
  p.tiles_n = (int)((a.N + tile_n - 1) / tile_n);
  p.height = BN == 256 ? tile_height(a, p.tiles_n, num_sms) : BN;
#ifdef OCCAMY_TUNING
  if (const char *e = getenv("OCCAMY_PT_HEIGHT")) p.height = std::min(atoi(e), BN);
#endif
  const int tile_m = wide ? 128 : p.height;
  // (rows of g groups fill at most so many tiles)
  const int64_t most_tiles =
      std::min<int64_t>((a.rows + std::min(a.groups, a.rows) * (tile_m - 1)) / tile_m * p.tiles_n, 1 << 28);
  count((Counter)(CNT_PRODUCT_32 + (BN == 32 ? 0 : BN == 64 ? 1 : BN == 128 ? 2 : 3)));
  if (scaled) {
    switch (BN) {
      case 32: return launch_width<32, true>(p, gated, most_tiles, num_sms, s);
      case 64: return launch_width<64, true>(p, gated, most_tiles, num_sms, s);
      case 128: return launch_width<128, true>(p, gated, most_tiles, num_sms, s);
      default: return launch_product_wide(p, gated, most_tiles, num_sms, s);
    }
  }
  switch (BN) {
    case 32: return launch_width<32, false>(p, gated, most_tiles, num_sms, s);
    case 64: return launch_width<64, false>(p, gated, most_tiles, num_sms, s);
    default: return launch_width<256, false>(p, gated, most_tiles, num_sms, s);
  }
}

}  // namespace occ
