// Which expert a token's row goes to, and the weighted sum of what comes back (occamy_route_experts,
// occamy_combine_experts).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "expert_ops.h"
#include "kernels.h"

namespace occ {
namespace {

constexpr int RT_THREADS = 1024, RT_WARPS = RT_THREADS / 32;
constexpr int RT_TOKENS = 128;       // of a block, more when there would be over RT_BLOCKS of them
constexpr int RT_BLOCKS = 256;
constexpr int PL_WARPS = 8;          // that count and place a block's rows

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
// The same for 16-bit logits, whose key leaves room for the expert (the lower one the larger) in the same word: one comparison
// of words does both.
template <typename T>
__device__ __forceinline__ uint32_t word_of(T v, int e) {
  uint32_t b = *reinterpret_cast<const uint16_t *>(&v);
  const float f = (float)v;
  if (b == 0x8000u) b = 0;
  b = f != f ? 0xffffu : (b & 0x8000u ? ~b & 0xffffu : b | 0x8000u);
  return b << 16 | (0xffffu - (uint32_t)e);
}
template <typename T>
__device__ __forceinline__ float value_of_word(uint32_t w) {
  const uint32_t k = w >> 16;
  const uint16_t b = (uint16_t)(k & 0x8000u ? k & 0x7fffu : ~k);
  return (float)*reinterpret_cast<const T *>(&b);
}
// of -inf and the largest expert number: below every word of a value
template <typename T>
constexpr uint32_t WORD_NONE = std::is_same<T, __half>::value ? 0x03ffffffu : 0x007fffffu;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// ---- up to eight choices of up to 256 experts (fp32: 128): eight lanes a token
// A lane holds V neighbouring experts' keys, each with its expert in the low half, so that no two are alike, and sorts them. A choice
// then looks at the first of each lane alone: three exchanges for the largest, and the lane that had it moves on.  With a token for a
// whole warp the instructions were few lanes' work: 460 a token, 16384 tokens of 128 experts, k = 8, 17 us; this way 11.
template <typename T>
struct KeyOf {   // 16-bit logits
  typedef uint32_t type;
  static constexpr type NONE = WORD_NONE<T>;
  static __device__ __forceinline__ type make(T v, int e) { return word_of(v, e); }
  static __device__ __forceinline__ float value(type k) { return value_of_word<T>(k); }
  static __device__ __forceinline__ int expert(type k) { return (int)(0xffffu - (k & 0xffffu)); }
};
template <>
struct KeyOf<float> {
  typedef unsigned long long type;
  static constexpr type NONE = (type)KEY_NONE << 32 | 0xffffffffu;
  static __device__ __forceinline__ type make(float v, int e) { return (type)key_of(v) << 32 | (0xffffffffu - (uint32_t)e); }
  static __device__ __forceinline__ float value(type k) { return value_of((uint32_t)(k >> 32)); }
  static __device__ __forceinline__ int expert(type k) { return (int)(0xffffffffu - (uint32_t)k); }
};
// Batcher's odd-even merge sort of V = 2^n values, largest first.
template <int V, typename K>
__device__ __forceinline__ void sort_down(K *key) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int i = 0; i + k < V; ++i) {
        // i and i + k, where i is in the first half of its run of 2 k, counted from k % p, and both in the same run of 2 p
        const int from = i - k % p;
        if (from >= 0 && from / k % 2 == 0 && i / (2 * p) == (i + k) / (2 * p)) {
          const K hi = max(key[i], key[i + k]), lo = min(key[i], key[i + k]);
          key[i] = hi;
          key[i + k] = lo;
        }
      }
}
constexpr int EIGHT = 8;
template <typename T, int V>
__device__ __forceinline__ void choose_by_eight(const RouteArgs &a, int64_t t0, int64_t t1) {
  typedef KeyOf<T> Key;
  typedef typename Key::type K;
  const int l = threadIdx.x % EIGHT;
  // (all lanes of a warp go round together: the exchanges are theirs)
  for (int64_t w = t0 + threadIdx.x / 32 * 4; w < t1; w += RT_THREADS / EIGHT) {
    const int64_t t = w + (threadIdx.x % 32) / EIGHT;
    const bool in = t < t1;
    const T *logits = (const T *)a.logits + t * a.ldl;
    K key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = l * V + v;
      key[v] = in && e < a.experts ? Key::make(logits[e], e) : 0;
    }
    float top = 0.0f, total = 0.0f;
    if (!a.normalise) {
      K m = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) m = max(m, key[v]);
#pragma unroll
      for (int d = EIGHT / 2; d; d /= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
      top = Key::value(m);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (key[v] > Key::NONE) total += expf(Key::value(key[v]) - top);
    }
    sort_down<V>(key);
    K mine = 0;
    for (int j = 0; j < a.k; ++j) {
      K m = key[0];
#pragma unroll
      for (int d = EIGHT / 2; d; d /= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
      if (j == 0) top = Key::value(m);
      if (l == j) mine = m;
      if (key[0] == m) {
#pragma unroll
        for (int v = 0; v + 1 < V; ++v) key[v] = key[v + 1];
        key[V - 1] = 0;
      }
    }
    const bool taken = mine > Key::NONE;
    float p = taken ? expf(Key::value(mine) - top) : 0.0f;
    if (a.normalise) total = p;
#pragma unroll
    for (int d = EIGHT / 2; d; d /= 2) total += __shfl_xor_sync(0xffffffffu, total, d);
    if (in && l < a.k) {
      a.chosen[t * a.k + l] = taken ? Key::expert(mine) : -1;
      a.weights[t * a.k + l] = taken ? p / total : 0.0f;
    }
  }
}

// ---- any other number of them: a warp a token, lane j gets the j-th choice.  V = ceil(experts / 32), the numbers of a lane.
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

// V: the numbers of a lane; negative: of eight lanes a token.
template <typename T, int V>
__device__ __forceinline__ void choose_block(const RouteArgs &a, int64_t t0, int64_t t1) {
  if constexpr (V < 0)
    choose_by_eight<T, -V>(a, t0, t1);
  else
    for (int64_t t = t0 + (threadIdx.x >> 5); t < t1; t += RT_WARPS) choose<V>(a, t, threadIdx.x & 31);
}

// Exclusive prefix sums of one number for each thread; `sums`: 32 words of shared memory.  The last thread's result and number
// make the total.
__device__ __forceinline__ int scan_block(int n, int32_t *sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int upto = n;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  if (warp == 0) {
    int t = sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, t, d);
      if (lane >= d) t += o;
    }
    sums[lane] = t;
  }
  __syncthreads();
  return upto - n + (warp ? sums[warp - 1] : 0);
}

// The slots (token, choice) [s0, s1) of a block, shared out to `warps` of its warps in whole groups of 32.
struct Slots {
  int64_t from, to;
};
__device__ __forceinline__ Slots slots_of(int64_t s0, int64_t s1, int warp, int warps) {
  const int64_t share = ((s1 - s0 + warps - 1) / warps + 31) / 32 * 32;
  const int64_t from = s0 + warp * share, to = from + share;
  return {from, to < s1 ? to : s1};
}
// cnt [warps][experts], in shared memory: how many rows each warp's slots bring to each expert.
__device__ __forceinline__ void count_slots(const RouteArgs &a, int64_t s0, int64_t s1, int32_t *cnt) {
  const int E = (int)a.experts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < PL_WARPS * E; i += RT_THREADS) cnt[i] = 0;
  __syncthreads();
  if (warp < PL_WARPS) {
    const Slots mine = slots_of(s0, s1, warp, PL_WARPS);
    for (int64_t s = mine.from + lane; s < mine.to; s += 32) {
      const int e = a.chosen[s];
      if (e >= 0) atomicAdd(&cnt[warp * E + e], 1);
    }
  }
  __syncthreads();
}
// Their rows: those of expert e go behind base (this thread's, e == threadIdx.x) in the order of the slots.
__device__ __forceinline__ void place_slots(const RouteArgs &a, int64_t s0, int64_t s1, int base, int32_t *cnt) {
  const int E = (int)a.experts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e0 = threadIdx.x;
  if (e0 < E) {
    int n[PL_WARPS];
#pragma unroll
    for (int w = 0; w < PL_WARPS; ++w) n[w] = cnt[w * E + e0];
#pragma unroll
    for (int w = 0; w < PL_WARPS; ++w) {
      cnt[w * E + e0] = base;
      base += n[w];
    }
  }
  __syncthreads();
  if (warp >= PL_WARPS) return;
  const Slots mine = slots_of(s0, s1, warp, PL_WARPS);
  for (int64_t s = mine.from; s < mine.to; s += 32) {
    const bool in = s + lane < mine.to;
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
// All of it, for tokens that one block takes.
template <typename T, int V>
__global__ void __launch_bounds__(RT_THREADS) route_one_kernel(RouteArgs a) {
  extern __shared__ int32_t cnt[];
  __shared__ int32_t sums[32];
  chain_begin();
  const int E = (int)a.experts, e = threadIdx.x;
  const int64_t slots = a.tokens * a.k;
  choose_block<T, V>(a, 0, a.tokens);
  __syncthreads();
  count_slots(a, 0, slots, cnt);
  int n = 0;
  if (e < E) {
#pragma unroll
    for (int w = 0; w < PL_WARPS; ++w) n += cnt[w * E + e];
  }
  const int base = scan_block(n, sums);
  if (e < E) a.offsets[e] = base;
  const int used = sums[31];
  if (e == 0) a.offsets[E] = used;
  for (int64_t i = used + e; i < slots; i += RT_THREADS) a.order[i] = -1;
  place_slots(a, 0, slots, base, cnt);
}

template <typename T, int V>
__global__ void __launch_bounds__(RT_THREADS) route_choose_kernel(RouteArgs a, int64_t per_block) {
  extern __shared__ int32_t cnt[];
  chain_begin();
  const int64_t t0 = blockIdx.x * per_block, t1 = t0 + per_block < a.tokens ? t0 + per_block : a.tokens;
  for (int e = threadIdx.x; e < a.experts; e += RT_THREADS) cnt[e] = 0;
  choose_block<T, V>(a, t0, t1);
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
  __shared__ int32_t sums[32];
  chain_begin();
  const int E = (int)a.experts, e0 = threadIdx.x;
  int32_t *front = sm, *total = sm + E, *cnt = sm + 2 * E;
  for (int e = threadIdx.x; e < 2 * E; e += RT_THREADS) sm[e] = 0;
  __syncthreads();
  // rows of each expert in front of this block's, and of all: each thread adds up every RT_THREADS / E-th block
  const int parts = RT_THREADS / E, part = e0 / E, e = e0 - part * E;
  if (part < parts) {
    int before = 0, all = 0;
#pragma unroll 4
    for (int b = part; b < (int)gridDim.x; b += parts) {
      const int n = a.counts[b * E + e];
      all += n;
      before += b < (int)blockIdx.x ? n : 0;
    }
    atomicAdd(&front[e], before);
    atomicAdd(&total[e], all);
  }
  const int64_t t0 = blockIdx.x * per_block, t1 = t0 + per_block < a.tokens ? t0 + per_block : a.tokens;
  count_slots(a, t0 * a.k, t1 * a.k, cnt);   // (its barriers come between the sums above and what follows)
  const int first = scan_block(e0 < E ? total[e0] : 0, sums);
  const int used = sums[31];
  if (blockIdx.x == 0) {
    if (e0 < E) a.offsets[e0] = first;
    if (e0 == 0) a.offsets[E] = used;
  }
  const int64_t all = a.tokens * a.k;
  for (int64_t i = used + blockIdx.x * (int64_t)RT_THREADS + threadIdx.x; i < all; i += (int64_t)gridDim.x * RT_THREADS)
    a.order[i] = -1;
  place_slots(a, t0 * a.k, t1 * a.k, first + (e0 < E ? front[e0] : 0), cnt);
}

template <typename T, int V>
cudaError_t launch_route_of(const RouteArgs &a, cudaStream_t s) {
  const int64_t per = tokens_of_block(a.tokens);
  const unsigned blocks = (unsigned)((a.tokens + per - 1) / per);
  const size_t cnt = (size_t)a.experts * 4 * PL_WARPS;
  if (blocks == 1) return launch_after(route_one_kernel<T, V>, dim3(1), dim3(RT_THREADS), cnt, s, 1, a);
  const cudaError_t e =
      launch_after(route_choose_kernel<T, V>, dim3(blocks), dim3(RT_THREADS), (size_t)a.experts * 4, s, 1, a, per);
  if (e != cudaSuccess) return e;
  return launch_after(route_place_kernel, dim3(blocks), dim3(RT_THREADS), cnt + (size_t)a.experts * 8, s, 1, a, per);
}

template <typename T>
cudaError_t launch_route_typed(const RouteArgs &a, cudaStream_t s) {
  if (a.k <= EIGHT) {
    if (a.experts <= 32) return launch_route_of<T, -4>(a, s);
    if (a.experts <= 64) return launch_route_of<T, -8>(a, s);
    if (a.experts <= 128) return launch_route_of<T, -16>(a, s);
    if constexpr (sizeof(T) == 2)
      if (a.experts <= 256) return launch_route_of<T, -32>(a, s);
  }
  if (a.experts <= 256) return launch_route_of<float, 8>(a, s);
  return launch_route_of<float, 32>(a, s);
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

int route_kernels(int64_t tokens) { return tokens <= tokens_of_block(tokens) ? 1 : 2; }

cudaError_t launch_route(const RouteArgs &a, cudaStream_t s) {
  if (a.type == ELEM_F32) return launch_route_typed<float>(a, s);
  if (a.type == ELEM_BF16) return launch_route_typed<__nv_bfloat16>(a, s);
  return launch_route_typed<__half>(a, s);
}

cudaError_t launch_combine(const CombineArgs &a, int num_sms, cudaStream_t s) {
  if (a.type == ELEM_F32) return launch_sum_of<float>(a, num_sms, s);
  if (a.type == ELEM_BF16) return launch_sum_of<__nv_bfloat16>(a, num_sms, s);
  return launch_sum_of<__half>(a, num_sms, s);
}

}  // namespace occ
