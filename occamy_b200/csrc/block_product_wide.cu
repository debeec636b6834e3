// Block-scaled products of many rows: tiles of 128 rows (a pair of CTAs: 256) x 256 weights.
//
// The rows are the M side, one to a TMEM lane, so that a k-step's scale is one number for each epilogue thread: with the rows on
// the N side (block_product.cu) every column has its own, which would have to come from shared memory, 128 bytes a cycle for MMA
// operands, copies and scales together.  A thread holds 128 sums of its row.  For each k-step it waits for the TMEM buffer, reads
// 64 columns at a time and adds them, scaled: 256 cycles of fp32 arithmetic and 150 of TMEM reads on an SM against the 512 that
// the tensor core takes for the k-step; the two epilogue warps of each quarter of the SM fill in for each other.
#include <algorithm>
#include <mutex>

#include "block_product_dev.cuh"

namespace occ {
namespace {

constexpr int PW_THREADS = 384, PW_EPI_WARPS = 8;   // loads, MMAs, two idle warps; two epilogue warps for each TMEM quadrant
constexpr int PW_WEIGHTS = 256;
constexpr int PW_STAGE_OUT = 4096;                  // of each epilogue warp: 32 rows x 32 sums

template <bool GATED, bool PAIR>
__global__ void __launch_bounds__(PW_THREADS, 1) block_product_wide_kernel(const __grid_constant__ PtParams p) {
  constexpr int SETS = GATED ? 2 : 1;
  constexpr int TILE_N = PW_WEIGHTS / SETS, TILE_M = PAIR ? 256 : 128;
  constexpr uint32_t A_BYTES = 128 * 128, B_BYTES = (PAIR ? 128 : 256) * 128;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if ((smem_u32(smem_raw) & 1023u) != 0u) {
    if (threadIdx.x == 0) atomicExch(p.err, 1007);
    return;
  }
  const int stages = p.stages;
  const uint32_t sA = smem_u32(smem_raw), sB = sA + stages * A_BYTES;
  uint8_t *stage_out = smem_raw + stages * (A_BYTES + B_BYTES);
  uint64_t *bars = reinterpret_cast<uint64_t *>(stage_out + PW_EPI_WARPS * PW_STAGE_OUT);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (stages + s); };
  auto tfull_bar = [&](int b) { return bar0 + 8u * (2 * stages + b); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * stages + 2 + b); };
  int32_t *words = reinterpret_cast<int32_t *>(bars + 2 * stages + 4);
  volatile uint32_t *tmem_holder = reinterpret_cast<volatile uint32_t *>(words);
  volatile int *abort_flag = words + 1;
  const PtGroups groups = {words + 4, words + 4 + p.groups, words + 4 + 2 * p.groups};

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;   // 0: the CTA that issues the MMAs
  if (threadIdx.x == 0) {
    tma_prefetch_map(&p.ta);
    tma_prefetch_map(&p.tb);
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), (PAIR ? 2 : 1) * PW_EPI_WARPS);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32((const void *)tmem_holder))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32((const void *)tmem_holder))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  pdl_launch_dependents();
  pdl_wait();
  pt_read_groups<PW_THREADS>(p, groups);
  __syncthreads();
  if (warp == 0) pt_count_tiles<TILE_M>(p, groups, lane);
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();   // both CTAs' barriers exist before either signals the other's
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int total = pt_total(p, groups);
  const int tile0 = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, tstep = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const int kblocks = p.kblocks;
  int err_code = 0;
  auto decode = [&](int tile) { return pt_decode<TILE_M, TILE_N>(p, groups, tile); };
  // rows of the tile in CTA r of a pair
  auto rows_of = [&](const PtTile &tl, int r) { return PAIR ? min(max(tl.rows - 128 * r, 0), 128) : tl.rows; };
  auto bytes_of = [&](int rows) {
    return B_BYTES + (p.index ? (uint32_t)((rows + 3) / 4) * 512u : (uint32_t)((rows + PT_BOX - 1) / PT_BOX) * (PT_BOX * 128u));
  };

  // The sums' warps take the registers that the others do without: 128 x 88 + 256 x 208 = 384 x 168.  (Each at the head of its
  // roles: behind a point where both come together the compiler keeps to the smaller number.)
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 0) {
    // ------------------------------------------------------------ loads
    TCT_DECL
    int stage = 0;
    uint32_t phase = 0;
    for (int tile = tile0; tile < total && !err_code; tile += tstep) {
      const PtTile tl = decode(tile);
      const int mine = rows_of(tl, rank), m0 = tl.m0 + 128 * rank;
      int4 rows4 = make_int4(0, 0, 0, 0);
      const int n4 = (mine + 3) / 4, boxes = (mine + PT_BOX - 1) / PT_BOX;
      if (p.index) rows4 = four_rows(p, m0, mine, lane);
      const uint32_t bytes = bytes_of(mine) + (PAIR ? bytes_of(rows_of(tl, 1)) : 0u);   // (of both CTAs, for rank 0)
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!TCT_WAIT(0, mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag))) {
          err_code = 1;
          break;
        }
        const int k = kb * 128;
        const uint32_t bar = PAIR ? cluster_map(full_bar(stage), 0) : full_bar(stage);
        if (rank == 0) expect_tx_warp(full_bar(stage), bytes);
        if constexpr (GATED) load_5d_warp<PAIR>(sB + stage * B_BYTES, &p.tb, bar, k, tl.n0 / 8 + 8 * rank, tl.g);
        else load_2d_warp<PAIR>(sB + stage * B_BYTES, &p.tb, bar, k, tl.g * p.N + tl.n0 + 128 * rank);
        const uint32_t dst = sA + stage * A_BYTES;
        if (p.index) {
          if (lane < n4) gather_4_rows<PAIR>(dst + lane * 512u, &p.ta, bar, k, rows4);
          __syncwarp();
        } else {
          for (int b = 0; b < boxes; ++b) load_2d_warp<PAIR>(dst + b * (PT_BOX * 128u), &p.ta, bar, k, m0 + b * PT_BOX);
        }
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
    if (rank == 0) {
      TCT_DECL
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      const uint64_t a0 = make_smem_desc(sA, 64), b0 = make_smem_desc(sB, 64);
      const uint32_t hi = (uint32_t)(a0 >> 32), a_lo = (uint32_t)a0, b_lo = (uint32_t)b0;
      for (int tile = tile0; tile < total && !err_code; tile += tstep) {
        const PtTile tl = decode(tile);
        // one CTA: no more weights than there are (a pair's halves stay where they are)
        const int n = PAIR ? PW_WEIGHTS : min(PW_WEIGHTS, ((p.N - tl.n0) * SETS + 15) / 16 * 16);
        const uint32_t idesc = p.idesc | ((uint32_t)(n >> 3) << 17);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!TCT_WAIT(0, mbar_wait_warp(tempty_bar(buf), buf_phase ^ 1u, abort_flag))) {
            err_code = 2;
            break;
          }
          if (!TCT_WAIT(1, mbar_wait_warp(full_bar(stage), phase, abort_flag))) {
            err_code = 3;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(buf * PW_WEIGHTS);
          const uint32_t a = a_lo + (uint32_t)stage * (A_BYTES >> 4), b = b_lo + (uint32_t)stage * (B_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) pt_mma<true, PAIR>(d, a + 2u * kk, hi, b + 2u * kk, hi, idesc, kk ? 1u : 0u);
          if constexpr (PAIR) {
            commit_pair_warp(empty_bar(stage));
            commit_pair_warp(tfull_bar(buf));
          } else {
            commit_warp(empty_bar(stage));
            commit_warp(tfull_bar(buf));
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
          if (++buf == 2) {
            buf = 0;
            buf_phase ^= 1u;
          }
        }
      }
      TCT_FLUSH(1)
    }
  }
  } else {
    // ------------------------------------------------------------ sums and results
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    TCT_DECL
    const int ew = warp - 4, quad = ew & 3, half = ew >> 2;   // TMEM lanes, columns 128 * half ...
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int tile = tile0; tile < total && !err_code; tile += tstep) {
      const PtTile tl = decode(tile);
      const int mine = rows_of(tl, rank), m0 = tl.m0 + 128 * rank, m = quad * 32 + lane;
      const int r = m < mine ? (p.index ? p.index[m0 + m] : m0 + m) : -1;
      const bool there = r >= 0 && r < p.a_rows;
      const float *sa = p.scale_a + (there ? (int64_t)r * kblocks : 0);
      // the scale block of this warp's weights; of a gated tile's 128 + 128 there is one each
      const int block_n = min(tl.n0 / SCALE_BLOCK + (GATED ? 0 : half), p.blocks_n - 1);
      const float *sb = p.scale_b + ((int64_t)tl.g * SETS * p.blocks_n + block_n) * kblocks;
      const int64_t second = (int64_t)p.blocks_n * kblocks;
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
      // scales two k-steps ahead
      auto scale_at = [&](int kb, int h) {
        return there && kb < kblocks ? __ldg(sa + kb) * __ldg(sb + (h ? second : 0) + kb) : 0.0f;
      };
      float now[SETS], next[SETS];
#pragma unroll
      for (int h = 0; h < SETS; ++h) now[h] = scale_at(0, h), next[h] = scale_at(1, h);
      for (int kb = 0; kb < kblocks; ++kb) {
        float then[SETS];
#pragma unroll
        for (int h = 0; h < SETS; ++h) then[h] = scale_at(kb + 2, h);
        if (!TCT_WAIT(1, mbar_wait_warp(tfull_bar(buf), buf_phase, abort_flag))) {
          err_code = 5;
          break;
        }
        tc_fence_after();
        const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * PW_WEIGHTS + half * 128);
        uint64_t f[SETS];
#pragma unroll
        for (int h = 0; h < SETS; ++h) f[h] = f2_pack(now[h], now[h]);
#pragma unroll
        for (int s = 0; s < 128; s += 64) {
          uint32_t v[64];
          tc_ld32(from + s, v);
          tc_ld32(from + s + 32, v + 32);
          tc_ld_wait();
          if (s) {   // the last of this buffer has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (PAIR) mbar_arrive_cluster(cluster_map(tempty_bar(buf), 0));
              else mbar_arrive(tempty_bar(buf));
            }
          }
#pragma unroll
          for (int i = 0; i < 32; ++i)
            acc[s / 2 + i] = f2_fma(pair_of(v[2 * i], v[2 * i + 1]), f[GATED ? (i >> 2) & 1 : 0], acc[s / 2 + i]);
        }
#pragma unroll
        for (int h = 0; h < SETS; ++h) now[h] = next[h], next[h] = then[h];
        if (++buf == 2) {
          buf = 0;
          buf_phase ^= 1u;
        }
      }
      if (err_code) break;
      // 32 sums of each row at a time through shared memory, so that neighbouring lanes store neighbouring results; pieces of 16
      // bytes are moved around by the row so that neither side meets in a bank.  One copy of the code behind it (block_product.cu).
      const int n_tile = min(TILE_N, p.N - tl.n0), n_half = half * (128 / SETS);
      uint8_t *own = stage_out + ew * PW_STAGE_OUT;
      const float *bias = p.bias ? p.bias + (int64_t)tl.g * SETS * p.N + tl.n0 : nullptr;
      const int out_size = p.out_type == ELEM_F32 ? 4 : 2;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        const int n_chunk = n_half + c * (32 / SETS);
        if (n_chunk >= n_tile || quad * 32 >= mine) break;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i == c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float4 v;
              f2_unpack(acc[i * 16 + 2 * j], v.x, v.y);
              f2_unpack(acc[i * 16 + 2 * j + 1], v.z, v.w);
              *reinterpret_cast<float4 *>(own + lane * 128 + ((j ^ (lane & 7)) * 16)) = v;
            }
        __syncwarp();
        constexpr int UNITS = 4 / SETS;   // of eight results in a row
#pragma unroll 1
        for (int i = lane; i < 32 * UNITS; i += 32) {
          const int row = i / UNITS, unit = i % UNITS, n = n_chunk + unit * 8;
          if (quad * 32 + row >= mine || n >= n_tile) continue;
          auto piece = [&](int j) {
            return *reinterpret_cast<const float4 *>(own + row * 128 + ((j ^ (row & 7)) * 16));
          };
          float t[8];
          if constexpr (GATED) {
            const float4 a0 = piece(unit * 4), a1 = piece(unit * 4 + 1), b0 = piece(unit * 4 + 2), b1 = piece(unit * 4 + 3);
            const float x[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
            const float y[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
            for (int j = 0; j < 8; ++j)   // (N % 8 == 0)
              t[j] = silu(x[j] + (bias ? bias[n + j] : 0.0f)) * (y[j] + (bias ? bias[p.N + n + j] : 0.0f));
          } else {
            const float4 a0 = piece(unit * 2), a1 = piece(unit * 2 + 1);
            const float x[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = x[j] + (bias && n + j < n_tile ? bias[n + j] : 0.0f);
            if (p.act != ACT_IDENTITY) {
#pragma unroll
              for (int j = 0; j < 8; ++j) t[j] = activate(t[j], p.act);
            }
          }
          store_row<8>(p, (uint8_t *)p.out + ((int64_t)(m0 + quad * 32 + row) * p.ldo + tl.n0 + n) * out_size, t, n_tile - n);
        }
      }
    }
    if (ew == 0 || ew == PW_EPI_WARPS - 1) { TCT_FLUSH(ew ? 4 : 3) }
  }
  if (err_code) {
    *abort_flag = 1;
    if (lane == 0) atomicExch(p.err, 1000 + err_code);
  }
  tc_fence_before();
  __syncthreads();
  // neither CTA of a pair leaves (or frees TMEM) while the other may still signal its barriers or have MMAs reading its memory
  if constexpr (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <bool GATED, bool PAIR>
cudaError_t launch(PtParams &p, int64_t most_tiles, int num_sms, cudaStream_t s) {
  const size_t misc = PW_EPI_WARPS * PW_STAGE_OUT + 8 * 4 + 16 + (3 * (size_t)p.groups + 1) * 4;
  const size_t stage = (PAIR ? 256 : 384) * 128 + 16;
  p.stages = (int)((TC_SMEM_LIMIT - misc) / stage);
  p.bufs = 2;
  p.splits = 1;
  static std::once_flag once[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::call_once(once[dev & 63], [] {
    cudaFuncSetAttribute(block_product_wide_kernel<GATED, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, TC_SMEM_LIMIT);
  });
  const int64_t grid = PAIR ? 2 * std::min<int64_t>(most_tiles, num_sms / 2) : std::min<int64_t>(most_tiles, num_sms);
  return launch_after(block_product_wide_kernel<GATED, PAIR>, dim3((unsigned)grid), dim3(PW_THREADS), p.stages * stage + misc, s,
                      PAIR ? 2 : 1, p);
}

}  // namespace

cudaError_t launch_product_wide(PtParams &p, bool gated, bool pair, int64_t most_tiles, int num_sms, cudaStream_t s) {
  if (gated) return pair ? launch<true, true>(p, most_tiles, num_sms, s) : launch<true, false>(p, most_tiles, num_sms, s);
  return pair ? launch<false, true>(p, most_tiles, num_sms, s) : launch<false, false>(p, most_tiles, num_sms, s);
}

}  // namespace occ
