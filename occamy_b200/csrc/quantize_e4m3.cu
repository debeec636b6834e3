// Rows or weights to e4m3 with a power-of-two scale for each block (occamy_quantize_e4m3).
//
//   s_b = 2^e, e the smallest integer >= -126 with max|x| over block b <= 448 * 2^e;   q = e4m3(x / s_b)
//
// A power of two costs e4m3 no precision (its steps are relative down to 2^-6, i.e. over 2^14 below the largest
// value) and makes x / s_b exact: q is x rounded once, to nearest even, whatever the order of operations, and the
// reciprocal is a product.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
};

// Eight threads for each block of 128 elements of a row, sixteen elements for each: two runs of eight, 64 apart, when rows allow
// 16-byte loads (VEC), else every eighth.  A pass of a CTA covers 2^lanes_log blocks of 32 >> lanes_log rows; a thread keeps its
// place in the row and goes from row to row, the next one's elements on their way while it works on these.
// WHOLE: VEC and no block is cut off.  What bounds it is instructions: with eight elements a thread and everything computed anew for each
// row 64 % of the issue slots (16384 gathered rows of 4096 bf16: 55 us, this way 32).
constexpr int QR_LANES = 8;
template <typename T, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 4 : 5) quantize_rows_kernel(QuantArgs a, int blocks, int lanes_log) {
  chain_begin();
  const int t = threadIdx.x % QR_LANES, unit = threadIdx.x / QR_LANES;
  const int block = (blockIdx.x << lanes_log) + (unit & ((1 << lanes_log) - 1));
  const int rows_pass = (256 / QR_LANES) >> lanes_log;
  const int left = (int)min((int64_t)SCALE_BLOCK, a.cols - (int64_t)block * SCALE_BLOCK);   // elements of the block
  const T *x = (const T *)a.x + (int64_t)block * SCALE_BLOCK;
  const int64_t step = (int64_t)gridDim.y * rows_pass;
  const int rows = (int)a.rows, x_rows = (int)a.x_rows;
  auto column = [&](int j) { return VEC ? (j >> 3) * 64 + t * 8 + (j & 7) : t + QR_LANES * j; };
  auto source = [&](int64_t row) {   // -1: none
    if (row >= rows || left <= 0) return -1;
    const int from = a.index ? __ldg(a.index + row) : (int)row;
    return from < x_rows ? from : -1;
  };
  auto fetch = [&](int from, Eight<T> *e) {
    if (from < 0) return;
    const T *p = x + (int64_t)from * a.ldx;
    if (WHOLE || (VEC && left == SCALE_BLOCK)) {
      e[0].template load<false>(p + t * 8);
      e[1].template load<false>(p + 64 + t * 8);
    } else {
      e[0].clear();
      e[1].clear();
      T *w = reinterpret_cast<T *>(e[0].w);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (column(j) < left) w[j] = p[column(j)];
    }
  };
  int64_t row = blockIdx.y * (int64_t)rows_pass + (unit >> lanes_log);
  uint8_t *q = a.q + row * a.ldq + (int64_t)block * SCALE_BLOCK;
  float *scale = a.scales + row * blocks + block;
  const int64_t q_step = step * a.ldq, scale_step = step * blocks;
  Eight<T> e[2], next[2];
  e[0].clear();
  e[1].clear();
  int from = source(row), from_next = source(row + step);
  fetch(from, e);
  const int64_t row0 = row - (unit >> lanes_log);   // the CTA's threads go round together
  for (int64_t r = row0; r < rows; r += step) {
    fetch(from_next, next);
    const int from_then = source(row + 2 * step);
    float v[16];
    e[0].values(v);
    e[1].values(v + 8);
    float amax = max_of<16>(v, 0.0f);
#pragma unroll
    for (int d = QR_LANES / 2; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    if (__any_sync(0xffffffffu, !finite(amax))) {
      amax = finite_max_of<16>(v, 0.0f);
#pragma unroll
      for (int d = QR_LANES / 2; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = finite_or_nan(v[j]);
    }
    if (from >= 0) {
      const int ex = scale_exponent(amax);
      const float inv = power_of_two(-ex);
      if (WHOLE || (VEC && left == SCALE_BLOCK)) {
        *reinterpret_cast<uint2 *>(q + t * 8) = make_uint2(pack4(v, inv), pack4(v + 4, inv));
        *reinterpret_cast<uint2 *>(q + 64 + t * 8) = make_uint2(pack4(v + 8, inv), pack4(v + 12, inv));
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (column(j) < left) q[column(j)] = (uint8_t)pack2(v[j] * inv, 0.0f);
      }
      if (t == 0) *scale = power_of_two(ex);
    }
    q += q_step;
    scale += scale_step;
    row += step;
    from = from_next;
    from_next = from_then;
    e[0] = next[0];
    e[1] = next[1];
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
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float v[8];
        e[k].values(v);
        amax = max_of<8>(v, amax);
      }
      amax = cta_max(amax, part);
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
        float v[8];
        e[k].values(v);
        if (odd) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = finite_or_nan(v[j]);
        }
        const uint2 w = make_uint2(pack4(v, inv), pack4(v + 4, inv));
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
    int lanes_log = 5;
    while (lanes_log > 0 && blocks <= 1 << (lanes_log - 1)) --lanes_log;
    const int64_t x = (blocks + (1 << lanes_log) - 1) >> lanes_log, rows = 256 / QR_LANES >> lanes_log;
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
