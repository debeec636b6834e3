// Launchers of the 8-bit and grouped operators (expert_api.cu checks their arguments).  Each enqueues on the given
// stream and returns what the launch returned; none allocates, waits, or keeps anything from one call for the next.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace occ {

// Element types as they cross the ABI.
enum ElemType { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2, ELEM_E4M3 = 3 };
inline int elem_size(int t) { return t == ELEM_F32 ? 4 : (t == ELEM_E4M3 ? 1 : 2); }

constexpr int SCALE_BLOCK = 128;   // elements along a row (and rows of a weight) that share a scale
inline int64_t scale_blocks(int64_t n) { return (n + SCALE_BLOCK - 1) / SCALE_BLOCK; }

// Activations beyond those of kernels.h (Act).
constexpr int ACT_SILU = 6;          // x * sigmoid(x)
constexpr int ACT_GATED_SILU = 7;    // silu(first matrix's result) * second matrix's

struct QuantArgs {
  const void *x;
  int type;
  int64_t x_rows, cols, ldx;
  const int32_t *index;   // row i of q is row index[i] of x, or null
  int64_t rows;
  int block_rows;         // 1 or SCALE_BLOCK
  uint8_t *q;
  int64_t ldq;
  float *scales;          // [rows / block_rows][scale_blocks(cols)]
};

struct ProductArgs {
  const void *a, *b;
  int type;                             // of a and b
  int64_t a_rows, lda, ldb;             // in elements
  const float *scale_a, *scale_b;       // e4m3, else null
  const float *bias;
  const int32_t *index, *offsets;       // offsets null: one group of all rows
  int64_t groups, rows, N, K;
  int act;
  void *out;
  int out_type;
  int64_t ldo;
  int *err;                             // word that bounded waits report into
};

struct RouteArgs {
  const void *logits;
  int type;
  int64_t tokens, experts, ldl;
  int k;
  int normalise;
  int32_t *chosen;
  float *weights;
  int32_t *offsets, *order, *position;
  int32_t *counts;        // [blocks][experts]
};

struct CombineArgs {
  const void *y;
  int type;
  int64_t y_rows, ldy;
  const int32_t *position;
  const float *weights;
  int64_t tokens, k, N;
  void *out;
  int out_type;
  int64_t ldo;
};

cudaError_t launch_quantize_e4m3(const QuantArgs &a, int num_sms, cudaStream_t s);
cudaError_t launch_product(const ProductArgs &a, int num_sms, cudaStream_t s);
cudaError_t launch_route(const RouteArgs &a, cudaStream_t s);
size_t route_workspace(int64_t tokens, int64_t experts, int64_t k);
int route_kernels(int64_t tokens);   // that launch_route() launches
cudaError_t launch_combine(const CombineArgs &a, int num_sms, cudaStream_t s);

#ifdef OCCAMY_TC_TIMERS
long long *tc_timer_words();   // conv_tc.cu
#endif

// A launch that may start while the kernel before it is still running: the kernel begins with chain_begin().  `cluster`: CTAs
// that run together.
template <typename... P, typename... A>
inline cudaError_t launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace occ
