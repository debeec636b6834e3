// Products of rows with weights, act(A B^T + bias): block-scaled e4m3, and rows in ragged groups that each have a matrix
// of their own (occamy_matmul_e4m3, occamy_matmul_grouped).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "expert_ops.h"
#include "kernels.h"

namespace occ {
namespace {

__device__ __forceinline__ float load_elem(const void *p, int64_t i, int type) {
  if (type == ELEM_BF16) return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
  if (type == ELEM_F16) return __half2float(((const __half *)p)[i]);
  return (float)((const __nv_fp8_e4m3 *)p)[i];
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

// One thread for each result.
__global__ void product_simple_kernel(ProductArgs p) {
  chain_begin();
  const int64_t n = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  const int64_t blocks_k = (p.K + SCALE_BLOCK - 1) / SCALE_BLOCK, blocks_n = (p.N + SCALE_BLOCK - 1) / SCALE_BLOCK;
  const int both = p.act == ACT_GATED_SILU ? 2 : 1;
  for (int64_t m = blockIdx.y; m < p.rows; m += gridDim.y) {
    int64_t g = 0;
    if (p.offsets) {
      while (g < p.groups && p.offsets[g + 1] <= m) ++g;
      if (g == p.groups || p.offsets[g] > m) continue;
    }
    if (n >= p.N) continue;
    const int64_t row = p.index ? p.index[m] : m;
    const bool there = row >= 0 && row < p.a_rows;
    float r[2];
    for (int h = 0; h < both; ++h) {
      const int64_t mat = g * both + h, brow = mat * p.N + n;
      float sum = 0.0f;
      for (int64_t kb = 0; there && kb < blocks_k; ++kb) {
        float part = 0.0f;
        for (int64_t k = kb * SCALE_BLOCK; k < p.K && k < (kb + 1) * SCALE_BLOCK; ++k)
          part = fmaf(load_elem(p.a, row * p.lda + k, p.type), load_elem(p.b, brow * p.ldb + k, p.type), part);
        if (p.scale_a)
          part *= p.scale_a[row * blocks_k + kb] * p.scale_b[(mat * blocks_n + n / SCALE_BLOCK) * blocks_k + kb];
        sum += part;
      }
      r[h] = sum + (p.bias ? p.bias[mat * p.N + n] : 0.0f);
    }
    float v = activate(r[0], p.act);
    if (both == 2) v *= r[1];
    const int64_t at = m * p.ldo + n;
    if (p.out_type == ELEM_F32) ((float *)p.out)[at] = v;
    else if (p.out_type == ELEM_BF16) ((__nv_bfloat16 *)p.out)[at] = __float2bfloat16_rn(v);
    else ((__half *)p.out)[at] = __float2half_rn(v);
  }
}

}  // namespace

cudaError_t launch_product(const ProductArgs &a, int, cudaStream_t s) {
  const dim3 grid((unsigned)((a.N + 127) / 128), (unsigned)(a.rows < 65535 ? a.rows : 65535));
  return launch_after(product_simple_kernel, grid, dim3(128), 0, s, a);
}

}  // namespace occ
