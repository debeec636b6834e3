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

struct alignas(64) PtParams {
  CUtensorMap ta, tb;
  const int32_t *index, *offsets;
  const float *scale_a, *scale_b, *bias;
  void *out;
  int64_t ldo;
  int a_rows, rows, groups, N, act, out_type;
  int kblocks;                         // k-steps: blocks of 128 bytes along K
  int blocks_n;                        // scale blocks of a matrix along N
  int tiles_n, stages, splits, bufs;
  uint32_t idesc;                      // instruction descriptor without N
  int vec_out;                         // 16-byte stores of the result are possible
  int *err;
#ifdef OCCAMY_TC_TIMERS
  long long *timers;   // as TcParams::timers: loads, MMAs, scales, two epilogue warps
#endif
};

// kind::f16, or kind::f8f6f4 for e4m3; by one CTA or a pair.
template <bool E4M3, bool PAIR>
__device__ __forceinline__ void pt_mma(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                       uint32_t idesc, uint32_t accumulate) {
  if constexpr (E4M3 && PAIR)
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 da, db;\n"
        "elect.sync _|q, 0xffffffff;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "mov.b64 da, {%1, %2};\n"
        "mov.b64 db, {%3, %4};\n"
        "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %5, p;\n}" ::"r"(d_tmem),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
  else if constexpr (E4M3)
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 da, db;\n"
        "elect.sync _|q, 0xffffffff;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "mov.b64 da, {%1, %2};\n"
        "mov.b64 db, {%3, %4};\n"
        "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n}" ::"r"(d_tmem),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
  else if constexpr (PAIR)
    mma_pair_warp(d_tmem, a_lo, a_hi, b_lo, b_hi, idesc, accumulate);
  else
    mma_warp(d_tmem, a_lo, a_hi, b_lo, b_hi, idesc, accumulate);
}
// Copies of two- and five-dimensional boxes; PAIR: counted on a barrier that may be the other CTA's (a shared::cluster
// address; the data lands in the issuing CTA's own memory).
template <bool PAIR>
__device__ __forceinline__ void load_2d_warp(uint32_t dst, const CUtensorMap *m, uint32_t bar, int c0, int c1) {
  if constexpr (PAIR)
    asm volatile(
        "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
        "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4}], [%2];\n}" ::"r"(dst),
        "l"(m), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
        "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n}" ::"r"(dst),
        "l"(m), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void load_5d_warp(uint32_t dst, const CUtensorMap *m, uint32_t bar, int c0, int c3, int c4) {
  if constexpr (PAIR)
    asm volatile(
        "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
        "@q cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %6, %6, %4, %5}], [%2];\n}" ::"r"(dst),
        "l"(m), "r"(bar), "r"(c0), "r"(c3), "r"(c4), "r"(0)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
        "@q cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %6, %6, %4, %5}], [%2];\n}" ::"r"(dst),
        "l"(m), "r"(bar), "r"(c0), "r"(c3), "r"(c4), "r"(0)
        : "memory");
}
// Four rows, by the executing lane.
template <bool PAIR>
__device__ __forceinline__ void gather_4_rows(uint32_t dst, const CUtensorMap *m, uint32_t bar, int c0, int4 r) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
        "l"(m), "r"(bar), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
        "l"(m), "r"(bar), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w)
        : "memory");
}
// Rows 4 i .. 4 i + 3 of a tile that begins at row m0 and has `rows`: where they are in A.  One that there is not, or none,
// reads as zeros.
__device__ __forceinline__ int4 four_rows(const PtParams &p, int m0, int rows, int i) {
  int r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = i * 4 + j;
    r[j] = m < rows ? p.index[m0 + m] : -1;
    if (r[j] < 0 || r[j] >= p.a_rows) r[j] = p.a_rows;
  }
  return make_int4(r[0], r[1], r[2], r[3]);
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
template <int W>
__device__ __forceinline__ void store_row(const PtParams &p, uint8_t *out, const float *r, int have) {
  if (p.vec_out && have >= W) {
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

// Which rows a tile has, and whose.  Shared memory: first and last + 1 row of each group, row tiles before it.
struct PtTile {
  int g, m0, rows, n0;   // group, first row, rows in the tile, first weight (of a gated pair)
};
struct PtGroups {
  int32_t *first, *last, *before;
};
// By all threads; they have to meet before anything is read.  Offsets are cut off at [0, rows].
template <int THREADS>
__device__ __forceinline__ void pt_read_groups(const PtParams &p, const PtGroups &t) {
  for (int g = threadIdx.x; g < p.groups; g += THREADS) {
    const int lo = p.offsets ? min(max(p.offsets[g], 0), p.rows) : 0;
    t.first[g] = lo;
    t.last[g] = p.offsets ? min(max(p.offsets[g + 1], lo), p.rows) : p.rows;
  }
}
// By one warp, behind that.
template <int ROWS>
__device__ __forceinline__ void pt_count_tiles(const PtParams &p, const PtGroups &t, int lane) {
  int sum = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    const int g = g0 + lane, n = g < p.groups ? (t.last[g] - t.first[g] + ROWS - 1) / ROWS : 0;
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    if (g < p.groups) t.before[g] = sum + upto - n;
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
  PtTile tl;
  tl.g = lo;
  tl.m0 = t.first[lo] + m * ROWS;
  tl.rows = min(ROWS, t.last[lo] - tl.m0);
  tl.n0 = n * WEIGHTS;
  return tl;
}
__device__ __forceinline__ int pt_total(const PtParams &p, const PtGroups &t) {
  return (int)min((int64_t)t.before[p.groups] * p.tiles_n, (int64_t)0x7fffffff);
}

// block_product_wide.cu.  Rows of its tiles' M side; launch.
cudaError_t launch_product_wide(PtParams &p, bool gated, bool pair, int64_t most_tiles, int num_sms, cudaStream_t s);

}  // namespace occ
