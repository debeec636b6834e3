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

// Infinities and NaN, which e4m3 cannot hold as they are, become NaN and do not count for the scale.
__device__ __forceinline__ float magnitude(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.0f;
}
__device__ __forceinline__ float finite_or_nan(float v) {
  return fabsf(v) <= 3.402823466e38f ? v : __int_as_float(0x7fffffff);
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

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// One warp for each block of 128 elements of a row, four of them for each lane.
template <typename T>
__global__ void quantize_rows_kernel(QuantArgs a, int64_t blocks, int64_t total) {
  chain_begin();
  const int lane = threadIdx.x & 31;
  const T *x = (const T *)a.x;
  for (int64_t i = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5); i < total;
       i += (int64_t)gridDim.x * (blockDim.x >> 5)) {
    const int64_t row = i / blocks, block = i % blocks;
    const int64_t from = a.index ? a.index[row] : row;
    if (from < 0 || from >= a.x_rows) continue;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = block * SCALE_BLOCK + lane + 32 * j;
      v[j] = c < a.cols ? to_float(x[from * a.ldx + c]) : 0.0f;
    }
    const float amax = warp_max(fmaxf(fmaxf(magnitude(v[0]), magnitude(v[1])), fmaxf(magnitude(v[2]), magnitude(v[3]))));
    const int e = scale_exponent(amax);
    const float inv = power_of_two(-e);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = block * SCALE_BLOCK + lane + 32 * j;
      if (c < a.cols) a.q[row * a.ldq + c] = (uint8_t)pack2(finite_or_nan(v[j]) * inv, 0.0f);
    }
    if (lane == 0) a.scales[row * blocks + block] = power_of_two(e);
  }
}

// One CTA of 256 threads for each block of 128 x 128.
template <typename T>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(QuantArgs a, int64_t blocks, int64_t total) {
  chain_begin();
  __shared__ float part[8];
  const T *x = (const T *)a.x;
  for (int64_t i = blockIdx.x; i < total; i += gridDim.x) {
    const int64_t r0 = i / blocks * SCALE_BLOCK, c0 = i % blocks * SCALE_BLOCK;
    const int64_t c = c0 + (threadIdx.x & 127);
    float amax = 0.0f;
    for (int r = threadIdx.x >> 7; r < SCALE_BLOCK; r += 2)
      if (r0 + r < a.rows && c < a.cols) amax = fmaxf(amax, magnitude(to_float(x[(r0 + r) * a.ldx + c])));
    amax = warp_max(amax);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
    __syncthreads();
    for (int w = 0; w < 8; ++w) amax = fmaxf(amax, part[w]);
    const int e = scale_exponent(amax);
    const float inv = power_of_two(-e);
    for (int r = threadIdx.x >> 7; r < SCALE_BLOCK; r += 2)
      if (r0 + r < a.rows && c < a.cols)
        a.q[(r0 + r) * a.ldq + c] = (uint8_t)pack2(finite_or_nan(to_float(x[(r0 + r) * a.ldx + c])) * inv, 0.0f);
    if (threadIdx.x == 0) a.scales[i] = power_of_two(e);
  }
}

template <typename T>
cudaError_t launch_typed(const QuantArgs &a, int num_sms, cudaStream_t s) {
  const int64_t blocks = scale_blocks(a.cols);
  if (a.block_rows == 1) {
    const int64_t total = a.rows * blocks, want = (total + 7) / 8, most = (int64_t)num_sms * 32;
    return launch_after(quantize_rows_kernel<T>, dim3((unsigned)(want < most ? want : most)), dim3(256), 0, s, 1, a, blocks,
                        total);
  }
  const int64_t total = scale_blocks(a.rows) * blocks, most = (int64_t)num_sms * 32;
  return launch_after(quantize_blocks_kernel<T>, dim3((unsigned)(total < most ? total : most)), dim3(256), 0, s, 1, a,
                      blocks, total);
}

}  // namespace

cudaError_t launch_quantize_e4m3(const QuantArgs &a, int num_sms, cudaStream_t s) {
  if (a.type == ELEM_F32) return launch_typed<float>(a, num_sms, s);
  if (a.type == ELEM_BF16) return launch_typed<__nv_bfloat16>(a, num_sms, s);
  return launch_typed<__half>(a, num_sms, s);
}

}  // namespace occ
