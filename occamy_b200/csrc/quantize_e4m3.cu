// Rows or weights to e4m3 with a power-of-two scale for each block (occamy_quantize_e4m3).
//
//   s_b = 2^e, e the smallest integer >= -126 with max|x| over block b <= 448 * 2^e;   q = e4m3(x / s_b)
//
// A power of two costs e4m3 no precision (its steps are relative down to 2^-6, i.e. over 2^14 below the largest
// value) and makes x / s_b exact: q is x rounded once, to nearest even, whatever the order of operations, and the
// reciprocal is a product.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "expert_ops.h"
#include "kernels.h"

namespace occ {
namespace {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// Infinities and NaN, which e4m3 cannot hold as they are, become NaN and do not count for the scale.  fmaxf() passes over a NaN, and
// the conversion keeps it: only a block whose maximum comes out infinite is looked at element by element.
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }
__device__ __forceinline__ float finite_or_nan(float v) { return finite(v) ? v : __int_as_float(0x7fffffff); }
template <int N>
__device__ __forceinline__ float max_of(const float *v, float amax) {
#pragma unroll
  for (int j = 0; j < N; ++j) amax = fmaxf(amax, fabsf(v[j]));
  return amax;
}
template <int N>
__device__ __forceinline__ float finite_max_of(const float *v, float amax) {
#pragma unroll
  for (int j = 0; j < N; ++j) amax = fmaxf(amax, finite(v[j]) ? fabsf(v[j]) : 0.0f);
  return amax;
}

// amax = 1.m * 2^E <= 448 * 2^e = 1.75 * 2^(8 + e): e = E - 8, one more when 1.m is above 1.75.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -126);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack4(const float *v, float inv) {
  return pack2(v[0] * inv, v[1] * inv) | pack2(v[2] * inv, v[3] * inv) << 16;
}

// Eight consecutive elements from 16-byte pieces.
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];
  template <bool ONCE>   // nothing reads them again
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint4 *from = reinterpret_cast<const uint4 *>(p) + i;
      w[i] = ONCE ? __ldcs(from) : __ldg(from);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void values(float *v) const {
    const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_float(e[j]);
  }
  __device__ __forceinline__ void nan_unless_finite() {
    T *e = reinterpret_cast<T *>(w);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (!finite(to_float(e[j]))) e[j] = (T)__int_as_float(0x7fffffff);
  }
  // The largest magnitude, NaN passed over; 16-bit types two at a time.
  static __device__ __forceinline__ float largest(const Eight *e, int n) {
    if constexpr (sizeof(T) == 4) {
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        float v[8];
        e[i].values(v);
        amax = max_of<8>(v, amax);
      }
      return amax;
    } else {
      using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
      T2 m = __habs2(reinterpret_cast<const T2 *>(e[0].w)[0]);
#pragma unroll
      for (int i = 0; i < 4 * n; ++i)
        if (i) m = __hmax2(m, __habs2(reinterpret_cast<const T2 *>(e[i >> 2].w)[i & 3]));
      return fmaxf(fmaxf(to_float(m.x), to_float(m.y)), 0.0f);   // (of nothing but NaN: 0)
    }
  }
  // In e4m3, times a power of two that leaves no magnitude above 448.  In bf16 that product is exact down to 2^-126, far below what
  // e4m3 tells from 0 (2^-10), and takes two elements at a time.  (fp16 does not hold all the powers.)
  __device__ __forceinline__ uint2 packed(float inv) const {
    float v[8];
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162 by = __float2bfloat162_rn(inv);
      Eight scaled;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        reinterpret_cast<__nv_bfloat162 *>(scaled.w)[j] = __hmul2(reinterpret_cast<const __nv_bfloat162 *>(w)[j], by);
      scaled.values(v);
      inv = 1.0f;
    } else {
      values(v);
    }
    return make_uint2(pack4(v, inv), pack4(v + 4, inv));
  }
};

// A few threads for each block of 128 elements of a row: four of 32 elements (fp32: eight of sixteen) in runs of eight when rows
// allow 16-byte loads (VEC), else every fourth (eighth) element.  A pass of a CTA covers 2^lanes_log blocks of some rows; a thread
// keeps its place in the row and goes from row to row, the next one's elements on their way while it works on these.
// WHOLE: VEC and no block is cut off.  What bounds it is the first-level cache (77 %: lines come in halves) and instructions (61 % of the
// issue slots): 16384 gathered rows of 4096 bf16 27 us, eight threads a block with all arithmetic in 32 bits 31, without the next
// row on its way and two CTAs more on an SM 29, eight threads for two blocks (lines read whole, more registers) 31.
template <typename T>
constexpr int QR_LANES = sizeof(T) == 4 ? 8 : 4;
template <typename T, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(256, 4) quantize_rows_kernel(QuantArgs a, int blocks, int lanes_log) {
  chain_begin();
  constexpr int LANES = QR_LANES<T>, RUNS = SCALE_BLOCK / (8 * LANES), RUN = 8 * LANES;
  const int t = threadIdx.x % LANES, unit = threadIdx.x / LANES;
  const int block = (blockIdx.x << lanes_log) + (unit & ((1 << lanes_log) - 1));
  const int rows_pass = (256 / LANES) >> lanes_log;
  const int left = (int)min((int64_t)SCALE_BLOCK, a.cols - (int64_t)block * SCALE_BLOCK);   // elements of the block
  const T *x = (const T *)a.x + (int64_t)block * SCALE_BLOCK;
  const int64_t step = (int64_t)gridDim.y * rows_pass;
  const int rows = (int)a.rows, x_rows = (int)a.x_rows;
  auto column = [&](int j) { return VEC ? (j >> 3) * RUN + t * 8 + (j & 7) : t + LANES * j; };
  auto source = [&](int64_t row) {   // -1: none
    if (row >= rows || left <= 0) return -1;
    const int from = a.index ? __ldg(a.index + row) : (int)row;
    return from < x_rows ? from : -1;
  };
  auto fetch = [&](int from, Eight<T> *e) {
    if (from < 0) return;
    const T *p = x + (int64_t)from * a.ldx;
    if (WHOLE || (VEC && left == SCALE_BLOCK)) {
#pragma unroll
      for (int i = 0; i < RUNS; ++i) e[i].template load<false>(p + i * RUN + t * 8);
    } else {
#pragma unroll
      for (int i = 0; i < RUNS; ++i) e[i].clear();
      T *w = reinterpret_cast<T *>(e[0].w);
#pragma unroll
      for (int j = 0; j < RUNS * 8; ++j)
        if (column(j) < left) w[j] = p[column(j)];
    }
  };
  int64_t row = blockIdx.y * (int64_t)rows_pass + (unit >> lanes_log);
  uint8_t *q = a.q + row * a.ldq + (int64_t)block * SCALE_BLOCK;
  float *scale = a.scales + row * blocks + block;
  const int64_t q_step = step * a.ldq, scale_step = step * blocks;
  Eight<T> e[RUNS], next[RUNS];
#pragma unroll
  for (int i = 0; i < RUNS; ++i) e[i].clear();
  int from = source(row), from_next = source(row + step);
  fetch(from, e);
  const int64_t row0 = row - (unit >> lanes_log);   // the CTA's threads go round together
  for (int64_t r = row0; r < rows; r += step) {
    fetch(from_next, next);
    const int from_then = source(row + 2 * step);
    float amax = Eight<T>::largest(e, RUNS);
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    if (__any_sync(0xffffffffu, !finite(amax))) {
      amax = 0.0f;
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        float v[8];
        e[i].values(v);
        amax = finite_max_of<8>(v, amax);
        e[i].nan_unless_finite();
      }
#pragma unroll
      for (int d = LANES / 2; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    }
    if (from >= 0) {
      const int ex = scale_exponent(amax);
      const float inv = power_of_two(-ex);
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        const uint2 w = e[i].packed(inv);
        if (WHOLE || (VEC && left == SCALE_BLOCK)) {
          *reinterpret_cast<uint2 *>(q + i * RUN + t * 8) = w;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (column(i * 8 + j) < left) q[column(i * 8 + j)] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
        }
      }
      if (t == 0) *scale = power_of_two(ex);
    }
    q += q_step;
    scale += scale_step;
    row += step;
    from = from_next;
    from_next = from_then;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) e[i] = next[i];
  }
}

__device__ __forceinline__ float cta_max(float v, float *part) {   // of 256 threads
#pragma unroll
  for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) v = fmaxf(v, part[w]);
  return v;
}

// One CTA of 256 threads for each block of 128 x 128, which stays in registers between its maximum and its results when rows
// allow 16-byte loads (VEC); else it is read twice.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(QuantArgs a, int64_t blocks, int64_t total) {
  chain_begin();
  __shared__ float part[8];
  const T *x = (const T *)a.x;
  for (int64_t i = blockIdx.x; i < total; i += gridDim.x) {
    const int64_t r0 = i / blocks * SCALE_BLOCK, c0 = i % blocks * SCALE_BLOCK;
    const int rows = (int)min((int64_t)SCALE_BLOCK, a.rows - r0), cols = (int)min((int64_t)SCALE_BLOCK, a.cols - c0);
    float amax = 0.0f;
    if constexpr (VEC) {
      const int t = threadIdx.x & 15, row = threadIdx.x >> 4;
      Eight<T> e[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        e[k].clear();
        const T *p = x + (r0 + row + 16 * k) * a.ldx + c0 + t * 8;
        if (row + 16 * k < rows && t * 8 + 8 <= cols) {
          e[k].template load<true>(p);
        } else if (row + 16 * k < rows) {
          T *w = reinterpret_cast<T *>(e[k].w);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (t * 8 + j < cols) w[j] = p[j];
        }
      }
      amax = cta_max(Eight<T>::largest(e, 8), part);
      const bool odd = !finite(amax);   // the same for all threads
      if (odd) {
        amax = 0.0f;
#pragma unroll 1
        for (int k = 0; k < 8; ++k)
          for (int j = 0; j < 8; ++j)
            if (row + 16 * k < rows && t * 8 + j < cols) {
              const float v = to_float(x[(r0 + row + 16 * k) * a.ldx + c0 + t * 8 + j]);
              amax = finite_max_of<1>(&v, amax);
            }
        amax = cta_max(amax, part);
      }
      const int ex = scale_exponent(amax);
      const float inv = power_of_two(-ex);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (row + 16 * k >= rows) break;
        if (odd) e[k].nan_unless_finite();
        const uint2 w = e[k].packed(inv);
        uint8_t *q = a.q + (r0 + row + 16 * k) * a.ldq + c0 + t * 8;
        if (t * 8 + 8 <= cols) {
          *reinterpret_cast<uint2 *>(q) = w;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (t * 8 + j < cols) q[j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
        }
      }
      if (threadIdx.x == 0) a.scales[i] = power_of_two(ex);
    } else {
      const int c = threadIdx.x & 127;
      for (int r = threadIdx.x >> 7; r < rows; r += 2)
        if (c < cols) {
          const float v = to_float(x[(r0 + r) * a.ldx + c0 + c]);
          amax = finite_max_of<1>(&v, amax);
        }
      amax = cta_max(amax, part);
      const int ex = scale_exponent(amax);
      const float inv = power_of_two(-ex);
      for (int r = threadIdx.x >> 7; r < rows; r += 2)
        if (c < cols)
          a.q[(r0 + r) * a.ldq + c0 + c] = (uint8_t)pack2(finite_or_nan(to_float(x[(r0 + r) * a.ldx + c0 + c])) * inv, 0.0f);
      if (threadIdx.x == 0) a.scales[i] = power_of_two(ex);
    }
  }
}

template <typename T, bool VEC>
cudaError_t launch_form(const QuantArgs &a, int num_sms, cudaStream_t s) {
  const int64_t blocks = scale_blocks(a.cols);
  if (a.block_rows == 1) {
    int lanes_log = sizeof(T) == 4 ? 5 : 6;
    while (lanes_log > 0 && blocks <= 1 << (lanes_log - 1)) --lanes_log;
    const int64_t x = (blocks + (1 << lanes_log) - 1) >> lanes_log, rows = 256 / QR_LANES<T> >> lanes_log;
    // four rows a thread, and no more CTAs than eight for each SM
    int64_t y = (a.rows + 4 * rows - 1) / (4 * rows);
    y = y * x < num_sms * 8 ? (a.rows + rows - 1) / rows : y;
    const int64_t most = num_sms * 8 / x > 1 ? num_sms * 8 / x : 1;
    const dim3 grid((unsigned)x, (unsigned)(y < most ? y : most));
    if (VEC && a.cols % SCALE_BLOCK == 0)
      return launch_after(quantize_rows_kernel<T, VEC, VEC>, grid, dim3(256), 0, s, 1, a, (int)blocks, lanes_log);
    return launch_after(quantize_rows_kernel<T, VEC, false>, grid, dim3(256), 0, s, 1, a, (int)blocks, lanes_log);
  }
  const int64_t total = scale_blocks(a.rows) * blocks, most = (int64_t)num_sms * 64;
  return launch_after(quantize_blocks_kernel<T, VEC>, dim3((unsigned)(total < most ? total : most)), dim3(256), 0, s, 1, a,
                      blocks, total);
}

template <typename T>
cudaError_t launch_typed(const QuantArgs &a, int num_sms, cudaStream_t s) {
  const bool vec = (uintptr_t)a.x % 16 == 0 && a.ldx * sizeof(T) % 16 == 0 && (uintptr_t)a.q % 8 == 0 && a.ldq % 8 == 0;
  return vec ? launch_form<T, true>(a, num_sms, s) : launch_form<T, false>(a, num_sms, s);
}

}  // namespace

cudaError_t launch_quantize_e4m3(const QuantArgs &a, int num_sms, cudaStream_t s) {
  if (a.type == ELEM_F32) return launch_typed<float>(a, num_sms, s);
  if (a.type == ELEM_BF16) return launch_typed<__nv_bfloat16>(a, num_sms, s);
  return launch_typed<__half>(a, num_sms, s);
}

}  // namespace occ
