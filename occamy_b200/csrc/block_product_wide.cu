// Block-scaled products of many rows: tiles of 128 rows x 256 weights.
//
// The rows are the M side, one to a TMEM lane, so that a k-step's scale is one number for each epilogue thread: with the rows on
// the N side (block_product.cu) every column has its own, which would have to come from shared memory, 128 bytes a cycle for MMA
// operands, copies and scales together.  A thread holds 128 sums of its row.  For each k-step it waits for the TMEM buffer, reads
// 16 columns at a time and adds them, scaled.  On an SM that is 256 cycles of fp32 arithmetic and 150 of TMEM reads against the 512
// that the tensor core takes for the k-step, but all eight warps go through it together, from one TMEM buffer's barrier to the
// next, and with what they wait on the way a k-step takes them 950: that is what bounds the kernel (8190 x 8192 x 4096: 275 us, 2.0
// PFLOP/s.  Before it looked for factors out of range 271; then, without the sums 250, without the TMEM reads 254, without both 224, and of
// that the loads alone took 167, 19 TB/s out of L2).
// Tried: sixteen warps of 64 columns (310: no registers for their loads), loads of 32 or 64 columns (spills), either half of the weights
// committed by itself (291 against 280 then), pairs of CTAs (cta_group::2, 288 to 330: less to load, but the second CTA's sums hold up
// both).
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "block_product_dev.cuh"

namespace occ {
namespace {

constexpr int PW_ROWS = 128, PW_WEIGHTS = 256;      // of a tile
constexpr int PW_COLUMNS = PW_WEIGHTS / (PT_EPI_WARPS / 4);   // of an epilogue warp
constexpr int PW_STAGE_OUT = 1024;                  // of each epilogue warp: 32 rows x 32 bytes
constexpr int PW_BATCH = 4;                         // k-steps whose scales come together
constexpr int PW_SCALES = PW_BATCH * 2 * 128;       // of a slot: [k-step][half of the tile's weights, or matrix][row]
constexpr int PW_SLOT = 2 * PW_SCALES * 4 + 8;      // bytes, with what goes with factors out of range, and whether there are any

template <bool GATED>
__global__ void __launch_bounds__(PT_THREADS, 1) block_product_wide_kernel(const __grid_constant__ PtParams p) {
  constexpr int SETS = GATED ? 2 : 1;
  constexpr int V_COLUMNS = 16;          // of one TMEM load: with more of them the sums run out of registers
  constexpr int TILE_N = PW_WEIGHTS / SETS;
  constexpr uint32_t A_BYTES = 128 * 128, B_BYTES = PW_WEIGHTS * 128;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if ((smem_u32(smem_raw) & 1023u) != 0u) {
    if (threadIdx.x == 0) atomicExch(p.err, 1007);
    return;
  }
  const int stages = p.stages;
  const uint32_t sA = smem_u32(smem_raw), sB = sA + stages * A_BYTES;
  uint8_t *stage_out = smem_raw + stages * (A_BYTES + B_BYTES);
  float *scales = reinterpret_cast<float *>(stage_out + PT_EPI_WARPS * PW_STAGE_OUT);   // two slots
  float *powers = scales + 2 * PW_SCALES;
  uint2 *any_power = reinterpret_cast<uint2 *>(powers + 2 * PW_SCALES);   // of either scale warp
  uint64_t *bars = reinterpret_cast<uint64_t *>(any_power + 2);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (stages + s); };
  auto tfull_bar = [&](int b) { return bar0 + 8u * (2 * stages + b); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * stages + 2 + b); };
  auto sfull_bar = [&](int b) { return bar0 + 8u * (2 * stages + 4 + b); };
  auto sempty_bar = [&](int b) { return bar0 + 8u * (2 * stages + 6 + b); };
  int32_t *words = reinterpret_cast<int32_t *>(bars + 2 * stages + 8);
  volatile uint32_t *tmem_holder = reinterpret_cast<volatile uint32_t *>(words);
  volatile int *abort_flag = words + 1;
  const PtGroups groups = {words + 4, words + 4 + p.groups, words + 4 + 2 * p.groups};

  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    if (!p.index) tma_prefetch_map(&p.ta);
    tma_prefetch_map(&p.tb);
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), p.index ? 1 + 32 * PT_GATHERERS : 1);   // loads, lanes that copy rows chosen by an index
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), PT_EPI_WARPS);
      mbar_init(sfull_bar(b), 2);
      mbar_init(sempty_bar(b), PT_EPI_WARPS);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32((const void *)tmem_holder))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    // (not before: a CTA of the next kernel that took the columns first would keep them until this one ends)
    pdl_launch_dependents();
  }
  pdl_wait();
  pt_read_groups<PT_THREADS>(p, groups);
  __syncthreads();
  if (warp == 0) pt_count_tiles<PW_ROWS>(p, groups, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int total = pt_total(p, groups);
  const int tile0 = (int)blockIdx.x, tstep = (int)gridDim.x;
  const int kblocks = p.kblocks;
  int err_code = 0;
  auto decode = [&](int tile) { return pt_decode<PW_ROWS, TILE_N>(p, groups, tile); };
  // The sums' warps take the registers that the others do without: 256 x 48 + 256 x 208 = 512 x 128.  (Each at the head of its
  // roles: behind a point where both come together the compiler keeps to the smaller number.)
  if (warp < PT_EPI_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 0) {
      // ------------------------------------------------------------ loads
      TCT_DECL
      int stage = 0;
      uint32_t phase = 0;
      for (int tile = tile0; tile < total && !err_code; tile += tstep) {
        const PtTile tl = decode(tile);
        const int boxes = p.index ? 0 : (tl.rows + PT_BOX - 1) / PT_BOX;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!TCT_WAIT(0, mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag))) {
            err_code = 1;
            break;
          }
          const int k = kb * 128;
          expect_tx_warp(full_bar(stage), B_BYTES + (uint32_t)boxes * (PT_BOX * 128u));
          if constexpr (GATED) load_5d_warp(sB + stage * B_BYTES, &p.tb, full_bar(stage), k, tl.n0 / 8, tl.g);
          else load_2d_warp(sB + stage * B_BYTES, &p.tb, full_bar(stage), k, tl.g * p.N + tl.n0);
          for (int b = 0; b < boxes; ++b)
            load_2d_warp(sA + stage * A_BYTES + b * (PT_BOX * 128u), &p.ta, full_bar(stage), k, tl.m0 + b * PT_BOX);
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
      const uint64_t a0 = make_smem_desc(sA, 64), b0 = make_smem_desc(sB, 64);
      const uint32_t hi = (uint32_t)(a0 >> 32), a_lo = (uint32_t)a0, b_lo = (uint32_t)b0;
      for (int tile = tile0; tile < total && !err_code; tile += tstep) {
        const PtTile tl = decode(tile);
        const int n = min(PW_WEIGHTS, ((p.N - tl.n0) * SETS + 15) / 16 * 16);   // no more weights than there are
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
          if (p.index) fence_async_smem();
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(buf * PW_WEIGHTS);
          const uint32_t a = a_lo + (uint32_t)stage * (A_BYTES >> 4), b = b_lo + (uint32_t)stage * (B_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) pt_mma<true>(d, a + 2u * kk, hi, b + 2u * kk, hi, idesc, kk ? 1u : 0u);
          commit_warp(empty_bar(stage));
          commit_warp(tfull_bar(buf));
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
    } else if (warp >= PT_GATHER_WARP) {
      // ------------------------------------------------------------ rows chosen by an index
      if (p.index)
        err_code = pt_gather_role<PW_ROWS, PT_GATHERERS>(p, tile0, total, tstep, 0, kblocks, sA, stages, warp - PT_GATHER_WARP, lane,
                                                         abort_flag, decode, full_bar, empty_bar);
    } else {
      // ------------------------------------------------------------ scales
      // sA * sB of every row, with the scale of either half of the tile's weights (gated: of either matrix).
      TCT_DECL
      const int t = threadIdx.x - 64;
      int slot = 0;
      uint32_t slot_phase = 0;
      for (int tile = tile0; tile < total && !err_code; tile += tstep) {
        const PtTile tl = decode(tile);
        const float *sa[2], *sb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int m = t + 64 * i, r = m < tl.rows ? (p.index ? p.index[tl.m0 + m] : tl.m0 + m) : -1;
          sa[i] = r >= 0 && r < p.a_rows ? p.scale_a + (int64_t)r * kblocks : nullptr;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int block = GATED ? h * p.blocks_n + tl.n0 / SCALE_BLOCK : min(tl.n0 / SCALE_BLOCK + h, p.blocks_n - 1);
          sb[h] = p.scale_b + ((int64_t)tl.g * SETS * p.blocks_n + block) * kblocks;
        }
        float va[2][PW_BATCH], vb[2][PW_BATCH];
        auto fetch = [&](int kq) {   // 1 where there is none (the numbers of a row that an index does not give are zeros)
#pragma unroll
          for (int j = 0; j < PW_BATCH; ++j) {
#pragma unroll
            for (int i = 0; i < 2; ++i) va[i][j] = sa[i] && kq + j < kblocks ? __ldg(sa[i] + kq + j) : 1.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) vb[h][j] = kq + j < kblocks ? __ldg(sb[h] + kq + j) : 1.0f;
          }
        };
        fetch(0);
        for (int kq = 0; kq < kblocks; kq += PW_BATCH) {
          uint32_t range = 0;
#pragma unroll
          for (int j = 0; j < PW_BATCH; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 2; ++i) range = max(range, pt_range(va[i][j], vb[h][j]));
          const bool look = __any_sync(0xffffffffu, range > PT_RANGE);
          if (!TCT_WAIT(0, mbar_wait_warp(sempty_bar(slot), slot_phase ^ 1u, abort_flag))) {
            err_code = 4;
            break;
          }
          float *dst = scales + slot * PW_SCALES + t;
#pragma unroll
          for (int j = 0; j < PW_BATCH; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 2; ++i) dst[(j * 2 + h) * 128 + 64 * i] = va[i][j] * vb[h][j];
          bool met = false;
          if (look) {
            float *pow = powers + slot * PW_SCALES + t;
#pragma unroll
            for (int j = 0; j < PW_BATCH; ++j)
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  float f;
                  const float power = pt_factor(va[i][j], vb[h][j], f);
                  met = met || power != 1.0f;
                  dst[(j * 2 + h) * 128 + 64 * i] = f, pow[(j * 2 + h) * 128 + 64 * i] = power;
                }
            met = __any_sync(0xffffffffu, met);
          }
          if (lane == 0) reinterpret_cast<uint32_t *>(any_power + slot)[warp - 2] = met;
          __syncwarp();
          if (lane == 0) mbar_arrive(sfull_bar(slot));
          if (++slot == 2) {
            slot = 0;
            slot_phase ^= 1u;
          }
          if (kq + PW_BATCH < kblocks) fetch(kq + PW_BATCH);   // there when the next slot is free
        }
      }
      if (warp == 2) { TCT_FLUSH(2) }
    }
  } else {
    // ------------------------------------------------------------ sums and results
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    TCT_DECL
    const int ew = warp - PT_EPI_WARP, quad = ew & 3, c0 = (ew >> 2) * PW_COLUMNS, half = c0 / 128;   // TMEM lanes, columns c0 ...
    int buf = 0, slot = 0;
    uint32_t buf_phase = 0, slot_phase = 0;
    for (int tile = tile0; tile < total && !err_code; tile += tstep) {
      const PtTile tl = decode(tile);
      float acc[PW_COLUMNS];   // from the bias on
#pragma unroll
      for (int i = 0; i < PW_COLUMNS; ++i) acc[i] = 0.0f;
      const int n_tile = min(TILE_N, p.N - tl.n0);
      const bool any = quad * 32 < tl.rows && c0 / SETS < n_tile;
      if (p.bias && any) {
        const float *bias = p.bias + (int64_t)tl.g * SETS * p.N + tl.n0 + c0 / SETS;
        const int left = n_tile - c0 / SETS;
#pragma unroll
        for (int i = 0; i < PW_COLUMNS; ++i) {
          const int n = GATED ? (i >> 4) * 8 + (i & 7) : i;
          if (n < left) acc[i] = __ldg(bias + (GATED && (i & 8) ? p.N : 0) + n);
        }
      }
      // A k-step's columns are read V_COLUMNS at a time, the next ones under way while these are added; its last ones are added
      // while the first of the next k-step arrive.
      constexpr int STEPS = PW_COLUMNS / V_COLUMNS;
      auto add = [&](const uint32_t *x, int s, const float *w) {
#pragma unroll
        for (int i = 0; i < V_COLUMNS; ++i)
          acc[s * V_COLUMNS + i] = fmaf(__uint_as_float(x[i]), w[GATED ? ((s * V_COLUMNS + i) >> 3) & 1 : 0], acc[s * V_COLUMNS + i]);
      };
      for (int kq = 0; kq < kblocks && !err_code; kq += PW_BATCH) {
        if (!mbar_wait_warp(sfull_bar(slot), slot_phase, abort_flag)) {
          err_code = 6;
          break;
        }
        const float *src = scales + slot * PW_SCALES + quad * 32 + lane;
        // (gated: the scales of one k-step at a time, there are no registers for more)
        constexpr int AHEAD = GATED ? 1 : PW_BATCH;
        float f[AHEAD][SETS];
        auto take = [&](int j) {
#pragma unroll
          for (int h = 0; h < SETS; ++h) f[j % AHEAD][h] = src[(j * 2 + (GATED ? h : half)) * 128];
        };
        auto taken = [&] {   // all of the slot
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty_bar(slot));
          if (++slot == 2) {
            slot = 0;
            slot_phase ^= 1u;
          }
        };
        // One k-step: its columns into the sums, each times its factor `w` (odd: times `power` first).
        auto step = [&](const float *w, auto odd, const float *power) {
          if (!TCT_WAIT(1, mbar_wait_warp(tfull_bar(buf), buf_phase, abort_flag))) {
            err_code = 5;
            return;
          }
          tc_fence_after();
          const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * PW_WEIGHTS + c0);
          if (any) {   // rows and columns that the tile does not have are not looked at
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
              uint32_t v[V_COLUMNS];
#pragma unroll
              for (int i = 0; i < V_COLUMNS; i += 32) tc_ld<V_COLUMNS < 32 ? V_COLUMNS : 32>(from + s * V_COLUMNS + i, v + i);
              pt_ld_wait<V_COLUMNS>(v);
              if (s + 1 == STEPS) {   // all of this buffer has been read
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty_bar(buf));
              }
              if constexpr (decltype(odd)::value) {
#pragma unroll
                for (int i = 0; i < V_COLUMNS; ++i)
                  v[i] = __float_as_uint(__uint_as_float(v[i]) * power[GATED ? ((s * V_COLUMNS + i) >> 3) & 1 : 0]);
              }
              add(v, s, w);
            }
          } else if (lane == 0) {
            mbar_arrive(tempty_bar(buf));
          }
          if (++buf == 2) {
            buf = 0;
            buf_phase ^= 1u;
          }
        };
        const uint2 odd = any_power[slot];
        if (quad & 1 ? odd.y : odd.x) {   // (of the scale warp that has this quadrant's rows)
#pragma unroll 1
          for (int j = 0; j < PW_BATCH && kq + j < kblocks && !err_code; ++j) {
            float w[SETS], power[SETS];
#pragma unroll
            for (int h = 0; h < SETS; ++h) {
              const int at = (j * 2 + (GATED ? h : half)) * 128;
              w[h] = src[at];
              power[h] = src[powers - scales + at];
            }
            step(w, std::true_type(), power);
          }
          taken();
          continue;
        }
        if constexpr (!GATED) {
#pragma unroll
          for (int j = 0; j < PW_BATCH; ++j) take(j);
          taken();
        }
#pragma unroll
        for (int j = 0; j < PW_BATCH; ++j) {
          if (kq + j >= kblocks || err_code) continue;
          if constexpr (GATED) take(j);
          step(f[j % AHEAD], std::false_type(), nullptr);
        }
        if constexpr (GATED) taken();
      }
      if (err_code) break;
      // Results go through shared memory, so that neighbouring lanes store neighbouring ones: 32 bytes of each row at a time, the
      // halves moved around by the row so that neither side meets in a bank.
      if (!any) continue;
      const int n_warp = c0 / SETS;
      uint8_t *own = stage_out + ew * PW_STAGE_OUT;
      const bool f32 = p.out_type == ELEM_F32;
      const int out_size = f32 ? 4 : 2, each = f32 ? 4 : 8;   // results of 16 bytes
      const int64_t ld = p.ldo * out_size;
      const int row0 = lane >> 1, piece = lane & 1, turn = (lane >> 2) & 1;
      const bool row_in[2] = {quad * 32 + row0 < tl.rows, quad * 32 + row0 + 16 < tl.rows};
      uint8_t *const out = (uint8_t *)p.out + ((int64_t)(tl.m0 + quad * 32 + row0) * p.ldo + tl.n0) * out_size;
      // 32 bytes of each row, of results n, n + 1, ...
      auto put = [&](int half_row, uint4 w) { *reinterpret_cast<uint4 *>(own + lane * 32 + (half_row ^ turn) * 16) = w; };
      auto flush = [&](int n_first, bool vec) {
        __syncwarp();
        const int n = n_first + piece * each;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!row_in[i] || n >= n_tile) continue;
          const uint4 w = *reinterpret_cast<const uint4 *>(own + (row0 + 16 * i) * 32 + (piece ^ ((row0 >> 2) & 1)) * 16);
          uint8_t *dst = out + 16 * i * ld + n * out_size;
          if (vec) {
            *reinterpret_cast<uint4 *>(dst) = w;
          } else {
            const uint32_t e[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (n + j >= n_tile) break;
              if (!f32) ((uint16_t *)dst)[j] = (uint16_t)(e[j >> 1] >> (16 * (j & 1)));
              else if (j < 4) ((uint32_t *)dst)[j] = e[j];
            }
          }
        }
        __syncwarp();
      };
      auto words = [&](const float *r) {
        return make_uint4(pack16(r[0], r[1], p.out_type), pack16(r[2], r[3], p.out_type), pack16(r[4], r[5], p.out_type),
                          pack16(r[6], r[7], p.out_type));
      };
      constexpr int UNITS = PW_COLUMNS / (8 * SETS);   // of eight results of this lane's row
      if (p.vec_out && (GATED || p.act == ACT_IDENTITY || p.act == ACT_RELU) && n_warp + UNITS * 8 <= n_tile) {
        // straight through all sums: a loop over them, as below, takes 9000 cycles a tile
        const float floor = !GATED && p.act == ACT_RELU ? 0.0f : -INFINITY;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          float r[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            r[j] = acc[u * 8 * SETS + j];
            if constexpr (GATED) r[j] = silu(r[j]) * acc[u * 16 + 8 + j];
            else asm("max.NaN.f32 %0, %0, %1;" : "+f"(r[j]) : "f"(floor));
          }
          if (f32) {
            put(0, make_uint4(__float_as_uint(r[0]), __float_as_uint(r[1]), __float_as_uint(r[2]), __float_as_uint(r[3])));
            put(1, make_uint4(__float_as_uint(r[4]), __float_as_uint(r[5]), __float_as_uint(r[6]), __float_as_uint(r[7])));
            flush(n_warp + u * 8, true);
          } else {
            put(u & 1, words(r));
            if (u & 1) flush(n_warp + u * 8 - 8, true);
          }
        }
        continue;
      }
      // other activations and edges: one copy of the code, the sums chosen by a branch (block_product.cu)
#pragma unroll 1
      for (int u = 0; u < UNITS; ++u) {
        const int n_unit = n_warp + u * 8;
        if (n_unit >= n_tile) break;
        float r[8 * SETS];
#pragma unroll
        for (int i = 0; i < UNITS; ++i)
          if (i == u) {
#pragma unroll
            for (int j = 0; j < 8 * SETS; ++j) r[j] = acc[i * 8 * SETS + j];
          }
        if constexpr (GATED) {
#pragma unroll
          for (int j = 0; j < 8; ++j) r[j] = silu(r[j]) * r[8 + j];
        } else if (p.act == ACT_RELU) {
#pragma unroll
          for (int j = 0; j < 8; ++j) r[j] = r[j] < 0.0f ? 0.0f : r[j];
        } else if (p.act != ACT_IDENTITY) {
#pragma unroll
          for (int j = 0; j < 8; ++j) r[j] = activate(r[j], p.act);
        }
        if (f32) {
          put(0, make_uint4(__float_as_uint(r[0]), __float_as_uint(r[1]), __float_as_uint(r[2]), __float_as_uint(r[3])));
          put(1, make_uint4(__float_as_uint(r[4]), __float_as_uint(r[5]), __float_as_uint(r[6]), __float_as_uint(r[7])));
          flush(n_unit, p.vec_out && n_unit + 8 <= n_tile);
        } else {
          put(u & 1, words(r));
          if ((u & 1) || n_unit + 8 >= n_tile) flush(n_unit - (u & 1) * 8, p.vec_out && n_unit + 8 <= n_tile);
        }
      }
    }
    if (ew == 0 || ew == PT_EPI_WARPS - 1) { TCT_FLUSH(ew ? 4 : 3) }
  }
  if (err_code) {
    *abort_flag = 1;
    if (lane == 0) atomicExch(p.err, 1000 + err_code);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <bool GATED>
cudaError_t launch(PtParams &p, int64_t most_tiles, int num_sms, cudaStream_t s) {
  const size_t misc = PT_EPI_WARPS * PW_STAGE_OUT + 8 * 8 + 16 + 2 * PW_SLOT + (3 * (size_t)p.groups + 1) * 4;
  const size_t stage = (PW_ROWS + PW_WEIGHTS) * 128 + 16;
  p.stages = (int)((TC_SMEM_LIMIT - misc) / stage);
  // the attribute is the device's: set for each once
  static std::once_flag once[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::call_once(once[dev & 63], [] {
    cudaFuncSetAttribute(block_product_wide_kernel<GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, TC_SMEM_LIMIT);
    cudaFuncSetAttribute(block_product_wide_kernel<GATED>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  });
  return launch_after(block_product_wide_kernel<GATED>, dim3((unsigned)std::min<int64_t>(most_tiles, num_sms)), dim3(PT_THREADS),
                      p.stages * stage + misc, s, 1, p);
}

}  // namespace

cudaError_t launch_product_wide(PtParams &p, bool gated, int64_t most_tiles, int num_sms, cudaStream_t s) {
  return gated ? launch<true>(p, most_tiles, num_sms, s) : launch<false>(p, most_tiles, num_sms, s);
}

}  // namespace occ
