// Device side shared by the two forms of the block-scaled and grouped products (block_product.cu, block_product_wide.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "conv_tc_dev.cuh"
#include "expert_ops.h"

namespace occ {

constexpr int PT_BOX = 32;             // rows of one copy
constexpr int PT_RASTER = 16;          // row tiles that go through all weights together

// Warps of either form: 0 loads, 1 MMAs, 2 and 3 scales, four that copy rows chosen by an index, eight of the epilogue, two
// for each TMEM quadrant.
constexpr int PT_GATHER_WARP = 4, PT_GATHERERS = 4, PT_EPI_WARP = 8, PT_EPI_WARPS = 8;
constexpr int PT_THREADS = 32 * (PT_EPI_WARP + PT_EPI_WARPS);

struct alignas(64) PtParams {
  CUtensorMap ta, tb;                  // (ta: without an index)
  const uint8_t *a;                    // with an index: A, units of 16 bytes from row to row, bytes in a row
  uint32_t a_ld16;
  int k_bytes;
  const int32_t *index, *offsets;
  const float *scale_a, *scale_b, *bias;
  void *out;
  int64_t ldo;
  int a_rows, rows, groups, N, act, out_type;
  int kblocks;                         // k-steps: blocks of 128 bytes along K
  int blocks_n;                        // scale blocks of a matrix along N
  int tiles_n, stages, splits, bufs;
  int height;                          // rows of a tile, in the form of 256 up to so many
  uint32_t idesc;                      // instruction descriptor without N
  int vec_out;                         // 16-byte stores of the result are possible
  int *err;
#ifdef OCCAMY_TC_TIMERS
  long long *timers;   // as TcParams::timers: loads, MMAs, scales, two epilogue warps
#endif
};

// A tile of the result.
struct PtTile {
  int g, m0, rows, n0;   // group, first row, rows in the tile, first weight (of a gated pair)
};

// kind::f16, or kind::f8f6f4 for e4m3.
template <bool E4M3>
__device__ __forceinline__ void pt_mma(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                       uint32_t idesc, uint32_t accumulate) {
  if constexpr (E4M3)
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

// Waits for a thread's TMEM loads; the values are not to be used before.
template <int V>
__device__ __forceinline__ void pt_ld_wait(uint32_t *v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < V; ++i) asm volatile("" : "+r"(v[i])::"memory");
}

// ---- scales
// A k-step's sums v (0, or 2^-18 to 2^25) are multiplied by sA * sB, which fp32 does not hold for all scales although v sA sB fits: 2^-75
// and 2^-75 would give 0, 2^64 and 2^64 infinity, and NaN where v is 0.  Such a factor is kept as f 2^p instead, p = -96 below
// 2^-126 (unless fp32 has that number) and 64 from 2^128 on, where f is in range or far enough out of it; v 2^p is exact, and v 2^p f
// rounded once.  That is rare: the exponents say whether any of four k-steps may be so, which is looked at then alone.  (One factor is
// left as fp32 rounds it, to a multiple of 2^-149: that of the scale 2^-126, a block of zeros or of numbers below 2^-117.  Padded rows
// have nothing else, and what is lost is below 2^-125.)
constexpr float PT_DOWN = 1.262177448e-29f, PT_UP = 18446744073709551616.0f;   // 2^-96, 2^64
// Above PT_RANGE where a * b may not be a normal number (by the exponents; also where either is 0 or subnormal) and a is not 2^-126.
constexpr uint32_t PT_RANGE = 250u << 23;
__device__ __forceinline__ uint32_t pt_range(float a, float b) {
  const uint32_t u = __float_as_uint(a), e = u == 0x00800000u ? 127u << 23 : u & 0x7f800000u;
  return e + (__float_as_uint(b) & 0x7f800000u) - (129u << 23);
}
// f = sA * sB or as above; returns 2^p.
__device__ __forceinline__ float pt_factor(float a, float b, float &f) {
  const float most = 3.402823466e38f;
  f = a * b;
  const float m = fabsf(f);
  if ((m >= 1.175494351e-38f && m <= most) || a == 0.0f || b == 0.0f || !(fabsf(a) <= most) || !(fabsf(b) <= most)) return 1.0f;
  if (m < 1.0f) {
    if (a == 1.175494351e-38f || b == 1.175494351e-38f) return 1.0f;
    const float g = (a * 281474976710656.0f) * (b * 281474976710656.0f);   // 2^48
    if (f * 79228162514264337593543950336.0f == g) return 1.0f;            // 2^96
    f = g;
    return PT_DOWN;
  }
  f = fminf(fmaxf((a * 2.328306437e-10f) * (b * 2.328306437e-10f), -most), most);   // 2^-32
  return PT_UP;
}

// This warp's TMEM lanes, 16 columns from `from` on: times `power`, a number for each column.
__device__ __forceinline__ void pt_rescale(uint32_t from, const float *power) {
  uint32_t v[16];
  tc_ld<16>(from, v);
  pt_ld_wait<16>(v);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const float2 w = *reinterpret_cast<const float2 *>(power + i);
    v[i] = __float_as_uint(__uint_as_float(v[i]) * w.x);
    v[i + 1] = __float_as_uint(__uint_as_float(v[i + 1]) * w.y);
  }
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(from),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// ---- rows chosen by an index
// Four warps copy them, 16 bytes a lane, in the swizzled order that the tensor core reads.  (TMA's own gather of four rows
// takes 75 cycles an instruction, 2400 for the 128 rows of a k-step; a cp.async of a warp takes that warp 30 cycles, a k-step
// by one warp 960 and with the epilogue beside it 3300.)  The copies arrive at the k-step's barrier by themselves, one arrival for
// each lane, and the warp that issues the MMAs makes them visible to the tensor core.
// The role of these warps, warp `warp` of WARPS.  A lane holds where its rows (4 j WARPS + 4 warp + lane / 8) begin,
// in units of 16 bytes, for a whole tile.  Returns an error code.
template <int ROWS, int WARPS, typename Decode, typename Full, typename Empty>
__device__ __forceinline__ int pt_gather_role(const PtParams &p, int tile0, int total, int tstep, int k0, int k1, uint32_t sR,
                                              int stages, int warp, int lane, volatile int *abort_flag, Decode &&decode,
                                              Full &&full_bar, Empty &&empty_bar) {
  constexpr int MINE = ROWS / (4 * WARPS);
  static_assert(MINE <= 32, "a bit for each row");
  int stage = 0, err = 0;
  uint32_t phase = 0;
  const int row0 = warp * 4 + (lane >> 3), chunk = lane & 7;
  for (int tile = tile0; tile < total && !err; tile += tstep) {
    const PtTile tl = decode(tile);
    uint32_t begin[MINE], there = 0;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int i = row0 + j * 4 * WARPS;
      const int r = i < tl.rows ? p.index[tl.m0 + i] : -1;
      const bool in = r >= 0 && r < p.a_rows;        // one that there is not reads as zeros
      begin[j] = in ? (uint32_t)r * p.a_ld16 : 0u;
      there |= (uint32_t)in << j;
    }
    const int mine = (tl.rows - row0 + 4 * WARPS - 1) / (4 * WARPS);   // (none: not positive)
    for (int kb = k0; kb < k1; ++kb) {
      if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag)) {
        err = 7;
        break;
      }
      const int at = kb * 128 + chunk * 16;
      const uint32_t have = (uint32_t)max(0, min(16, p.k_bytes - at));   // the rows end here: zeros behind them
      const uint8_t *base = p.a + (have ? at : 0);
      const uint32_t dst = sR + stage * (ROWS * 128u) + row0 * 128u;
#pragma unroll
      for (int j = 0; j < MINE; ++j)
        if (j < mine) {
          const uint32_t size = there >> j & 1u ? have : 0u;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                           dst + (uint32_t)(j * WARPS * 512) + (uint32_t)((chunk ^ ((row0 + j * 4 * WARPS) & 7)) << 4)),
                       "l"(base + ((uint64_t)begin[j] << 4)), "r"(size)
                       : "memory");
        }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full_bar(stage)) : "memory");
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");   // nothing may be under way when the CTA ends
  return err;
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
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + expf(-v)); }
__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case ACT_SIGMOID: return __fdividef(1.0f, 1.0f + expf(-v));
    case ACT_RELU: return v < 0.0f ? 0.0f : v;
    case ACT_TANH: return tanhf(v);
    case ACT_CLIP: return fminf(fmaxf(v, 0.0f), 6.0f);
    case ACT_SILU: return silu(v);
    default: return v;
  }
}
__device__ __forceinline__ uint32_t pack16(float a, float b, int type) {
  return type == ELEM_F16 ? f2_to_bf16x2<true>(f2_pack(a, b)) : f2_to_bf16x2<false>(f2_pack(a, b));
}
// W results of one row, the first `have` of them; `out` is their address.
template <int W, bool WHOLE = false>
__device__ __forceinline__ void store_row(const PtParams &p, uint8_t *out, const float *r, int have) {
  if (WHOLE || (p.vec_out && have >= W)) {
    if (p.out_type == ELEM_F32) {
#pragma unroll
      for (int j = 0; j < W; j += 4) *reinterpret_cast<float4 *>(out + j * 4) = make_float4(r[j], r[j + 1], r[j + 2], r[j + 3]);
    } else if constexpr (W == 4) {
      *reinterpret_cast<uint2 *>(out) = make_uint2(pack16(r[0], r[1], p.out_type), pack16(r[2], r[3], p.out_type));
    } else {
      *reinterpret_cast<uint4 *>(out) = make_uint4(pack16(r[0], r[1], p.out_type), pack16(r[2], r[3], p.out_type),
                                                   pack16(r[4], r[5], p.out_type), pack16(r[6], r[7], p.out_type));
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (j < have) {
        if (p.out_type == ELEM_F32) ((float *)out)[j] = r[j];
        else ((uint16_t *)out)[j] = (uint16_t)pack16(r[j], 0.0f, p.out_type);
      }
  }
}

// Shared memory: first and last + 1 row of each group, row tiles before it.
struct PtGroups {
  int32_t *first, *last, *before;
};
// By all threads; they have to meet before anything is read.  Offsets are cut off at [0, rows].
template <int THREADS>
__device__ __forceinline__ void pt_read_groups(const PtParams &p, const PtGroups &t) {
  for (int g = threadIdx.x; g < p.groups; g += THREADS) {
    t.first[g] = p.offsets ? min(max(p.offsets[g], 0), p.rows) : 0;
    t.last[g] = p.offsets ? min(max(p.offsets[g + 1], 0), p.rows) : p.rows;
  }
}
// By one warp, behind that: how many row tiles come before each group.  An offset below one in front of it counts as that one: no
// row is in two groups, whatever the offsets are.
template <int ROWS>
__device__ __forceinline__ void pt_count_tiles(const PtParams &p, const PtGroups &t, int lane) {
  int sum = 0, top = t.first[0];
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    const int g = g0 + lane;
    int end = g < p.groups ? max(t.last[g], top) : top;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end = max(end, o);
    }
    int begin = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) begin = top;
    top = __shfl_sync(0xffffffffu, end, 31);
    const int high = ROWS == 256 ? p.height : ROWS;
    const int n = g < p.groups ? (end - begin + high - 1) / high : 0;
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    if (g < p.groups) {
      t.first[g] = begin;
      t.last[g] = end;
      t.before[g] = sum + upto - n;
    }
    sum += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) t.before[p.groups] = sum;
}
template <int ROWS, int WEIGHTS>
__device__ __forceinline__ PtTile pt_decode(const PtParams &p, const PtGroups &t, int tile) {
  const int mt = tile / p.tiles_n;
  int lo = 0, hi = p.groups - 1;          // last group with before[g] <= mt
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.before[mid] <= mt) lo = mid;
    else hi = mid - 1;
  }
  const int local = tile - t.before[lo] * p.tiles_n, all = t.before[lo + 1] - t.before[lo];
  const int band = local / (PT_RASTER * p.tiles_n), in_band = local - band * PT_RASTER * p.tiles_n;
  const int height = min(PT_RASTER, all - band * PT_RASTER), n = in_band / height;
  const int m = band * PT_RASTER + in_band - n * height;
  const int high = ROWS == 256 ? p.height : ROWS;
  PtTile tl;
  tl.g = lo;
  tl.m0 = t.first[lo] + m * high;
  tl.rows = min(high, t.last[lo] - tl.m0);
  tl.n0 = n * WEIGHTS;
  return tl;
}
__device__ __forceinline__ int pt_total(const PtParams &p, const PtGroups &t) {
  return (int)min((int64_t)t.before[p.groups] * p.tiles_n, (int64_t)0x7fffffff);
}

// block_product_wide.cu
cudaError_t launch_product_wide(PtParams &p, bool gated, int64_t most_tiles, int num_sms, cudaStream_t s);

}  // namespace occ
