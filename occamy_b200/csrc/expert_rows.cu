// Which expert a token's row goes to, and the weighted sum of what comes back (occamy_route_experts,
// occamy_combine_experts).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "expert_ops.h"
#include "kernels.h"

namespace occ {
namespace {

constexpr int RT_THREADS = 1024, RT_WARPS = RT_THREADS / 32;
constexpr int RT_TOKENS = 128;       // of a block, more when there would be over RT_BLOCKS of them
constexpr int RT_BLOCKS = 256;
constexpr int RT_MOST_EXPERTS = 1024;

inline int64_t tokens_of_block(int64_t tokens) {
  const int64_t even = (tokens + RT_BLOCKS - 1) / RT_BLOCKS;
  return even > RT_TOKENS ? even : RT_TOKENS;
}

__device__ __forceinline__ float load_logit(const void *p, int64_t i, int type) {
  if (type == ELEM_F32) return ((const float *)p)[i];
  if (type == ELEM_BF16) return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
  return __half2float(((const __half *)p)[i]);
}
// Unsigned keys in the order of the values; both zeros alike, every NaN above everything.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t KEY_NONE = 0x007fffffu;   // of -inf: an expert that is not to be taken, and all below it

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// The k largest logits of token t, by one warp; lane j gets the j-th choice.  V = ceil(experts / 32).
template <int V>
__device__ __forceinline__ void choose(const RouteArgs &a, int64_t t, int lane) {
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 32 + lane;
    key[v] = e < a.experts ? key_of(load_logit(a.logits, t * a.ldl + e, a.type)) : 0u;
  }
  uint32_t mine = 0;
  int expert = -1;
  float top = 0.0f, total = 0.0f;
  for (int j = 0; j < a.k; ++j) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v] > best) best = key[v], at = v * 32 + lane;
    const uint32_t high = __reduce_max_sync(0xffffffffu, best);
    if (high <= KEY_NONE) break;
    const int e = (int)__reduce_min_sync(0xffffffffu, best == high ? (uint32_t)at : 0xffffffffu);
    if (j == 0) {
      top = value_of(high);
      if (!a.normalise) {
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (key[v] > KEY_NONE) sum += expf(value_of(key[v]) - top);
        total = warp_sum(sum);
      }
    }
    if (lane == j) mine = high, expert = e;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e == v * 32 + lane) key[v] = 0;
  }
  float w = expert >= 0 ? expf(value_of(mine) - top) : 0.0f;
  if (a.normalise) total = warp_sum(w);
  if (expert >= 0) w /= total;
  if (lane < a.k) {
    a.chosen[t * a.k + lane] = expert;
    a.weights[t * a.k + lane] = w;
  }
}

template <int V>
__device__ __forceinline__ void choose_block(const RouteArgs &a, int64_t t0, int64_t t1) {
  for (int64_t t = t0 + (threadIdx.x >> 5); t < t1; t += RT_WARPS) choose<V>(a, t, threadIdx.x & 31);
}

// Rows of this block's (token, choice) slots: they go behind base[expert] in the order of the slots.  Each warp counts its
// share of the slots first; after that every one knows where its own begin.  cnt: [warps][experts] in shared memory.
__device__ __forceinline__ void place_block(const RouteArgs &a, int64_t s0, int64_t s1, const int32_t *base, int32_t *cnt,
                                            int warps) {
  const int E = (int)a.experts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t share = ((s1 - s0 + warps - 1) / warps + 31) / 32 * 32;
  const int64_t w0 = s0 + warp * share, w1 = w0 + share < s1 ? w0 + share : s1;
  for (int i = threadIdx.x; i < warps * E; i += RT_THREADS) cnt[i] = 0;
  __syncthreads();
  if (warp < warps)
    for (int64_t s = w0 + lane; s < w1; s += 32) {
      const int e = a.chosen[s];
      if (e >= 0) atomicAdd(&cnt[warp * E + e], 1);
    }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += RT_THREADS) {
    int at = base[e];
    for (int w = 0; w < warps; ++w) {
      const int n = cnt[w * E + e];
      cnt[w * E + e] = at;
      at += n;
    }
  }
  __syncthreads();
  if (warp < warps)
    for (int64_t s = w0; s < w1; s += 32) {
      const bool in = s + lane < w1;
      const int e = in ? a.chosen[s + lane] : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      const int before = __popc(same & ((1u << lane) - 1u));
      int at = -1;
      if (e >= 0) at = cnt[warp * E + e] + before;
      __syncwarp();
      if (e >= 0 && before == 0) cnt[warp * E + e] += __popc(same);
      __syncwarp();
      if (in) a.position[s + lane] = at;
      if (at >= 0) a.order[at] = (int32_t)((s + lane) / a.k);
    }
}

inline __host__ __device__ int place_warps(int64_t experts) { return experts <= 256 ? RT_WARPS : 8; }

template <int V>
__global__ void __launch_bounds__(RT_THREADS) route_choose_kernel(RouteArgs a, int64_t per_block) {
  extern __shared__ int32_t cnt[];
  chain_begin();
  const int64_t t0 = blockIdx.x * per_block, t1 = t0 + per_block < a.tokens ? t0 + per_block : a.tokens;
  for (int e = threadIdx.x; e < a.experts; e += RT_THREADS) cnt[e] = 0;
  choose_block<V>(a, t0, t1);
  __syncthreads();
  for (int64_t s = t0 * a.k + threadIdx.x; s < t1 * a.k; s += RT_THREADS) {
    const int e = a.chosen[s];
    if (e >= 0) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += RT_THREADS) a.counts[blockIdx.x * a.experts + e] = cnt[e];
}

__global__ void __launch_bounds__(RT_THREADS) route_place_kernel(RouteArgs a, int64_t per_block) {
  extern __shared__ int32_t sm[];
  chain_begin();
  const int E = (int)a.experts;
  int32_t *base = sm, *total = sm + E, *cnt = sm + 2 * E;
  for (int e = threadIdx.x; e < 2 * E; e += RT_THREADS) sm[e] = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < (int64_t)gridDim.x * E; i += RT_THREADS) {
    const int e = (int)(i % E), n = a.counts[i];
    if (!n) continue;
    atomicAdd(&total[e], n);
    if (i / E < blockIdx.x) atomicAdd(&base[e], n);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int at = 0;
    for (int e = 0; e < E; ++e) {
      if (blockIdx.x == 0) a.offsets[e] = at;
      base[e] += at;
      at += total[e];
    }
    if (blockIdx.x == 0) a.offsets[E] = at;
    total[0] = at;
  }
  __syncthreads();
  const int64_t used = total[0], all = a.tokens * a.k;
  for (int64_t i = used + blockIdx.x * (int64_t)RT_THREADS + threadIdx.x; i < all; i += (int64_t)gridDim.x * RT_THREADS)
    a.order[i] = -1;
  const int64_t t0 = blockIdx.x * per_block, t1 = t0 + per_block < a.tokens ? t0 + per_block : a.tokens;
  place_block(a, t0 * a.k, t1 * a.k, base, cnt, place_warps(E));
}

template <int V>
cudaError_t launch_choose(const RouteArgs &a, unsigned blocks, int64_t per_block, cudaStream_t s) {
  return launch_after(route_choose_kernel<V>, dim3(blocks), dim3(RT_THREADS), (size_t)a.experts * 4, s, 1, a, per_block);
}

// ---------------------------------------------------------------- weighted sum
template <typename T>
__device__ __forceinline__ float as_float(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else return (float)v;
}
template <typename T>
struct Row8 {   // eight elements of a row, in 16-byte pieces
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
  }
  __device__ __forceinline__ void add(float f, float *sum) const {
    const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = fmaf(f, as_float(e[j]), sum[j]);
  }
};
template <typename T>
__device__ __forceinline__ void put8(T *p, const float *v) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = (T)v[j];
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(t);
  }
}

// Eight results a thread, the rows of four choices on their way together; `per_row` threads for each token.  Needs rows that begin
// at multiples of 16 bytes; the last threads' elements beyond N one by one.
template <typename T, typename O>
__global__ void __launch_bounds__(256) combine_kernel(CombineArgs a, int per_row) {
  chain_begin();
  const T *y = (const T *)a.y;
  O *out = (O *)a.out;
  const int64_t total = a.tokens * per_row;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t t = total <= 0x7fffffff ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row;
    const int64_t n = (i - t * per_row) * 8;
    const int32_t *position = a.position + t * a.k;
    const float *weights = a.weights + t * a.k;
    float sum[8] = {};
    if (n + 8 <= a.N) {
      for (int j0 = 0; j0 < a.k; j0 += 4) {
        Row8<T> r[4];
        bool there[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int32_t at = j0 + j < a.k ? position[j0 + j] : -1;
          there[j] = at >= 0 && at < a.y_rows;
          if (there[j]) r[j].load(y + at * a.ldy + n);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (there[j]) r[j].add(weights[j0 + j], sum);
      }
      put8(out + t * a.ldo + n, sum);
    } else {
      for (int e = 0; n + e < a.N; ++e) {
        float v = 0.0f;
        for (int j = 0; j < a.k; ++j) {
          const int32_t at = position[j];
          if (at >= 0 && at < a.y_rows) v = fmaf(weights[j], as_float(y[at * a.ldy + n + e]), v);
        }
        out[t * a.ldo + n + e] = (O)v;
      }
    }
  }
}
// Rows that begin anywhere: one result a thread.
template <typename T, typename O>
__global__ void __launch_bounds__(256) combine_plain_kernel(CombineArgs a) {
  chain_begin();
  const T *y = (const T *)a.y;
  const int64_t total = a.tokens * a.N;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / a.N, n = i % a.N;
    float sum = 0.0f;
    for (int j = 0; j < a.k; ++j) {
      const int32_t at = a.position[t * a.k + j];
      if (at >= 0 && at < a.y_rows) sum = fmaf(a.weights[t * a.k + j], as_float(y[at * a.ldy + n]), sum);
    }
    ((O *)a.out)[t * a.ldo + n] = (O)sum;
  }
}

template <typename T, typename O>
cudaError_t launch_sum(const CombineArgs &a, int num_sms, cudaStream_t s) {
  const bool vec = (uintptr_t)a.y % 16 == 0 && a.ldy * sizeof(T) % 16 == 0 && (uintptr_t)a.out % 16 == 0 &&
                   a.ldo * sizeof(O) % 16 == 0;
  const int per_row = vec ? (int)((a.N + 7) / 8) : (int)a.N;
  const int64_t want = (a.tokens * per_row + 255) / 256, most = (int64_t)num_sms * 64;
  const dim3 grid((unsigned)(want < most ? want : most));
  return vec ? launch_after(combine_kernel<T, O>, grid, dim3(256), 0, s, 1, a, per_row)
             : launch_after(combine_plain_kernel<T, O>, grid, dim3(256), 0, s, 1, a);
}
template <typename T>
cudaError_t launch_sum_of(const CombineArgs &a, int num_sms, cudaStream_t s) {
  if (a.out_type == ELEM_F32) return launch_sum<T, float>(a, num_sms, s);
  if (a.out_type == ELEM_BF16) return launch_sum<T, __nv_bfloat16>(a, num_sms, s);
  return launch_sum<T, __half>(a, num_sms, s);
}

}  // namespace

size_t route_workspace(int64_t tokens, int64_t experts, int64_t) {
  const int64_t per = tokens_of_block(tokens);
  return (size_t)((tokens + per - 1) / per) * (size_t)experts * 4;
}

cudaError_t launch_route(const RouteArgs &a, cudaStream_t s) {
  const int64_t per = tokens_of_block(a.tokens);
  const unsigned blocks = (unsigned)((a.tokens + per - 1) / per);
  cudaError_t e;
  if (a.experts <= 32) e = launch_choose<1>(a, blocks, per, s);
  else if (a.experts <= 64) e = launch_choose<2>(a, blocks, per, s);
  else if (a.experts <= 128) e = launch_choose<4>(a, blocks, per, s);
  else if (a.experts <= 256) e = launch_choose<8>(a, blocks, per, s);
  else e = launch_choose<32>(a, blocks, per, s);
  if (e != cudaSuccess) return e;
  const size_t smem = (size_t)a.experts * 4 * (2 + place_warps(a.experts));
  return launch_after(route_place_kernel, dim3(blocks), dim3(RT_THREADS), smem, s, 1, a, per);
}

cudaError_t launch_combine(const CombineArgs &a, int num_sms, cudaStream_t s) {
  if (a.type == ELEM_F32) return launch_sum_of<float>(a, num_sms, s);
  if (a.type == ELEM_BF16) return launch_sum_of<__nv_bfloat16>(a, num_sms, s);
  return launch_sum_of<__half>(a, num_sms, s);
}

}  // namespace occ
