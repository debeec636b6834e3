// Entry points of the 8-bit and grouped operators: argument checks, the order between the caller's stream and the
// runtime's, launches.
#include <climits>
#include <cstdarg>
#include <mutex>
#include <vector>

#include "expert_ops.h"
#include "graph_replay.h"
#include "kernels.h"
#include "runtime.h"

extern "C" void occamy_internal_opaque_call(void);

using namespace occ;

namespace {

constexpr int MAX_DEVICES = 64;
constexpr int NO_DEVICE = -1, TOO_SMALL = -2, BAD_ARGUMENT = -3, FAILED = -4, BAD_POINTER = -5, CAPTURED = -6;
constexpr int64_t MOST_EXPERTS = 1024, MOST_CHOICES = 32, MOST_ROWS = (1ll << 31) - 1024;

// Calls may come from several host threads; what they share (the tensor registry, counters, first-use set-up) is
// not made for that.
std::mutex g_mutex;

int refuse(int code, const char *who, const char *why, ...) {
  char text[256];
  va_list ap;
  va_start(ap, why);
  vsnprintf(text, sizeof(text), why, ap);
  va_end(ap);
  fprintf(stderr, "[occamy_b200] %s: %s\n", who, text);
  return code;
}

// One call: the current device, the pointers it was given, and the runtime's own stream.
//
// Memory that the runtime knows (wrapDNNMalloc, a pool) may not hold yet what it stands for: a zero fill or an upload that
// is put off, a result kept in another format, a convolution held back, a recorded inference whose calls wait for their graph.
// Such tensors are brought up to date first, on the runtime's stream; the caller's stream waits for that, and the runtime's for
// the call.
class Call {
 public:
  Call(const char *who, cudaStream_t stream) : who_(who), stream_(stream) {}

  int open() {
    if (cudaGetDevice(&device_) != cudaSuccess || device_ < 0 || device_ >= MAX_DEVICES)
      return refuse(NO_DEVICE, who_, "no usable current device");
    static int sms[MAX_DEVICES] = {};
    if (!sms[device_]) {
      int major = 0;
      if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device_) != cudaSuccess || major != 10)
        return refuse(NO_DEVICE, who_, "device %d is not sm_100", device_);
      if (cudaDeviceGetAttribute(&sms[device_], cudaDevAttrMultiProcessorCount, device_) != cudaSuccess)
        return refuse(NO_DEVICE, who_, "cannot read the number of SMs");
    }
    num_sms_ = sms[device_];
    // the runtime's state is set up by the first call of any kind, which a stream that is captured does not allow
    static bool ready = false;
    if (!ready) {
      if (capturing(stream_)) return refuse(CAPTURED, who_, "the first call cannot be captured");
      rt();
      ready = true;
    }
    if (stream_ == rt().stream && !capturing(stream_)) {   // (what is put off is no part of the caller's graph)
      occamy_internal_opaque_call();
      settled_ = true;
    }
    return 0;
  }
  // `bytes` of device memory that the call reads / writes; null is passed over.  `align`: of the address, in bytes.
  // `whole`: a result without gaps between its rows.
  int in(const void *p, int64_t bytes, size_t align) { return use(p, bytes, align, false, false); }
  int out(void *p, int64_t bytes, size_t align, bool whole = true) { return use(p, bytes, align, true, whole); }

  // When all memory is known and nothing can be refused any more but a capture, before the launches: nothing has been enqueued so far.
  int begin() {
    bool tracked = false;
    // (a tensor of an inference that is being replayed is not on record until its calls are made one by one)
    for (int i = 0; i < count_ && !tracked; ++i) tracked = in_live_pool(uses_[i].p) || !records(uses_[i]).empty();
    if (!tracked) return 0;
    // Bringing it up to date would be done by every replay, or not at all, and a replay cannot put on record what it wrote.
    if (capturing(stream_) || capturing(rt().stream))
      return refuse(CAPTURED, who_, "memory of the runtime's own cannot be used while the stream, or occamy_stream(), is captured");
    if (!settled_) occamy_internal_opaque_call();
    tracked_ = true;
    // A result may leave parts of its memory as they were: they have to be there too.  (An operand may be several tensors.)
    // One that fusion left unwritten and the result replaces has nothing to keep: writing it is no error.
    for (int i = 0; i < count_; ++i)
      for (uintptr_t t : records(uses_[i]))
        if (!replaces(uses_[i], t)) ensure_f32((const void *)t);
    for (int i = 0; i < count_; ++i)
      if (uses_[i].written)
        for (uintptr_t t : records(uses_[i])) mark_f32((void *)t);
    return stream_ == rt().stream ? 0 : order(rt().stream, stream_);
  }
  // `e`: of the launches, of so many kernels.
  int end(cudaError_t e, int kernels = 1) {
    if (e != cudaSuccess) {
      cudaGetLastError();
      return refuse((int)e, who_, "%s", cudaGetErrorString(e));
    }
    count(CNT_LAUNCHES, kernels);
    if (!tracked_ || stream_ == rt().stream) return 0;
    return order(stream_, rt().stream);
  }
  int num_sms() const { return num_sms_; }
  const char *who() const { return who_; }

 private:
  struct Use {
    const void *p;
    int64_t bytes;
    bool written, whole;
  };
  static std::vector<uintptr_t> records(const Use &u) { return reg_within(u.p, (size_t)u.bytes); }
  static bool replaces(const Use &u, uintptr_t t) {
    const TensorRec *rec = reg_find((const void *)t);
    return u.whole && rec && rec->fmt == FMT_ELIDED && t >= (uintptr_t)u.p && t + rec->bytes <= (uintptr_t)u.p + (uintptr_t)u.bytes;
  }
  int use(const void *p, int64_t bytes, size_t align, bool written, bool whole) {
    if (!p) return 0;
    if ((uintptr_t)p % align) return refuse(BAD_ARGUMENT, who_, "an address is not a multiple of %zu bytes", align);
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
      cudaGetLastError();
      return refuse(BAD_POINTER, who_, "an address is not known to CUDA");
    }
    if (at.type != cudaMemoryTypeManaged && (at.type != cudaMemoryTypeDevice || at.device != device_))
      return refuse(BAD_POINTER, who_, "an address is not memory of the current device");
    uses_[count_++] = {p, bytes, written, whole};
    return 0;
  }
  static bool capturing(cudaStream_t s) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(s, &st) == cudaSuccess && st == cudaStreamCaptureStatusNone) return false;
    cudaGetLastError();
    return true;
  }
  int order(cudaStream_t first, cudaStream_t then) {
    cudaEvent_t ev;
    cudaError_t e = cudaEventCreateWithFlags(&ev, cudaEventDisableTiming);
    if (e == cudaSuccess) {
      e = cudaEventRecord(ev, first);
      if (e == cudaSuccess) e = cudaStreamWaitEvent(then, ev, 0);
      cudaEventDestroy(ev);
    }
    if (e == cudaSuccess) return 0;
    cudaGetLastError();
    return refuse((int)e, who_, "%s", cudaGetErrorString(e));
  }

  const char *who_;
  cudaStream_t stream_;
  int device_ = -1, num_sms_ = 0;
  bool settled_ = false, tracked_ = false;
  Use uses_[8];
  int count_ = 0;
};

bool extent(int64_t v) { return v >= 0 && v <= INT_MAX; }
bool real_type(int t) { return t == ELEM_F32 || t == ELEM_BF16 || t == ELEM_F16; }
// Rows `ld` elements apart, `cols` of them used: within 40 bits of bytes, as the copy engine's strides are.
bool row_length(int64_t ld, int64_t cols, int64_t rows, int size) {
  return ld >= cols && ld <= INT64_MAX / 16 && ld * size < (1ll << 40) && (rows <= 1 || ld <= INT64_MAX / 16 / rows);
}
// From the first element of such rows to the last, in bytes.
int64_t span(int64_t rows, int64_t ld, int64_t cols, int size) { return rows ? ((rows - 1) * ld + cols) * size : 0; }
bool linear_act(int64_t mode) {
  return mode == ACT_SIGMOID || mode == ACT_RELU || mode == ACT_TANH || mode == ACT_CLIP || mode == ACT_IDENTITY ||
         mode == ACT_SILU;
}

#define TRY(expr)               \
  do {                          \
    if (int c_ = (expr)) return c_; \
  } while (0)

// The products' common part.  `rows`: of the result.
int product(Call &call, ProductArgs &p, cudaStream_t stream) {
  const char *who = call.who();
  if (!extent(p.a_rows) || !extent(p.rows) || !extent(p.N) || !extent(p.groups) || p.K < 1 || p.K > INT_MAX / 2)
    return refuse(BAD_ARGUMENT, who, "extent out of range");
  const int both = p.act == ACT_GATED_SILU ? 2 : 1, es = elem_size(p.type);
  const int64_t mats = p.groups * both;
  if (!real_type(p.out_type)) return refuse(BAD_ARGUMENT, who, "type of the result");
  // (the kernels' 32-bit row and weight numbers go up to a tile past the end)
  if (p.rows > MOST_ROWS || mats * p.N > MOST_ROWS) return refuse(BAD_ARGUMENT, who, "more than 2^31 - 1024 rows of A or of weights");
  if (!row_length(p.lda, p.K, p.a_rows, es) || !row_length(p.ldb, p.K, mats * p.N, es) || !row_length(p.ldo, p.N, p.rows, 4))
    return refuse(BAD_ARGUMENT, who, "distance between rows out of range");
  if (p.lda * es % 16 || p.ldb * es % 16)
    return refuse(BAD_ARGUMENT, who, "rows of the operands have to start at multiples of 16 bytes");
  if (p.index && p.a_rows * (p.lda * es / 16) > (int64_t)UINT32_MAX)
    return refuse(BAD_ARGUMENT, who, "A of more than 64 GiB cannot be indexed");
  if (both == 2 && p.N % 8) return refuse(BAD_ARGUMENT, who, "a gated product needs N %% 8 == 0");
  const bool scaled = p.type == ELEM_E4M3;
  if (p.rows == 0 || p.N == 0) return 0;
  if (p.a_rows == 0) return refuse(BAD_ARGUMENT, who, "A has no rows");
  if (!p.a || !p.b || !p.out || (scaled && (!p.scale_a || !p.scale_b)))
    return refuse(BAD_ARGUMENT, who, "null pointer");
  if (!scaled) p.scale_a = p.scale_b = nullptr;
  TRY(call.open());
  const int64_t blocks_k = scale_blocks(p.K);
  TRY(call.in(p.a, span(p.a_rows, p.lda, p.K, es), 16));
  TRY(call.in(p.b, span(mats * p.N, p.ldb, p.K, es), 16));
  TRY(call.in(p.scale_a, p.a_rows * blocks_k * 4, 4));
  TRY(call.in(p.scale_b, mats * scale_blocks(p.N) * blocks_k * 4, 4));
  TRY(call.in(p.bias, mats * p.N * 4, 4));
  TRY(call.in(p.index, p.rows * 4, 4));
  TRY(call.in(p.offsets, (p.groups + 1) * 4, 4));
  TRY(call.out(p.out, span(p.rows, p.ldo, p.N, elem_size(p.out_type)), elem_size(p.out_type), p.ldo == p.N));
  p.err = rt().dev_err;
  TRY(call.begin());
  return call.end(launch_product(p, call.num_sms(), stream));
}

}  // namespace

extern "C" {

int occamy_quantize_e4m3(const void *x, int xType, int64_t xRows, int64_t cols, int64_t ldx, const int32_t *index,
                         int64_t rows, int64_t blockRows, void *q, int64_t ldq, float *scales, cudaStream_t stream) try {
  std::lock_guard<std::mutex> lock(g_mutex);
  Call call("occamy_quantize_e4m3", stream);
  if (!real_type(xType)) return refuse(BAD_ARGUMENT, call.who(), "type of x");
  if (!extent(xRows) || !extent(cols) || !extent(rows)) return refuse(BAD_ARGUMENT, call.who(), "extent out of range");
  if (blockRows != 1 && blockRows != SCALE_BLOCK) return refuse(BAD_ARGUMENT, call.who(), "blockRows is 1 or 128");
  if (index && blockRows != 1) return refuse(BAD_ARGUMENT, call.who(), "an index needs blockRows 1");
  if (!index && rows != xRows) return refuse(BAD_ARGUMENT, call.who(), "rows other than xRows need an index");
  if (!row_length(ldx, cols, xRows, elem_size(xType)) || !row_length(ldq, cols, rows, 1))
    return refuse(BAD_ARGUMENT, call.who(), "distance between rows out of range");
  if (rows == 0 || cols == 0 || xRows == 0) return 0;
  if (!x || !q || !scales) return refuse(BAD_ARGUMENT, call.who(), "null pointer");
  TRY(call.open());
  TRY(call.in(x, span(xRows, ldx, cols, elem_size(xType)), elem_size(xType)));
  TRY(call.in(index, rows * 4, 4));
  TRY(call.out(q, span(rows, ldq, cols, 1), 1, ldq == cols));
  TRY(call.out(scales, (rows + blockRows - 1) / blockRows * scale_blocks(cols) * 4, 4));
  TRY(call.begin());
  QuantArgs a = {x, xType, xRows, cols, ldx, index, rows, (int)blockRows, (uint8_t *)q, ldq, scales};
  return call.end(launch_quantize_e4m3(a, call.num_sms(), stream));
} catch (...) {
  return FAILED;
}

int occamy_matmul_e4m3(const void *a, int64_t lda, const float *scaleA, const void *b, int64_t ldb, const float *scaleB,
                       const float *bias, int64_t M, int64_t N, int64_t K, int64_t activMode, void *out, int outType,
                       int64_t ldo, cudaStream_t stream) try {
  std::lock_guard<std::mutex> lock(g_mutex);
  Call call("occamy_matmul_e4m3", stream);
  if (!linear_act(activMode)) return refuse(BAD_ARGUMENT, call.who(), "activation mode (0, 1, 2, 3, 5 or 6)");
  ProductArgs p = {};
  p.a = a; p.b = b; p.type = ELEM_E4M3;
  p.a_rows = p.rows = M; p.lda = lda; p.ldb = ldb;
  p.scale_a = scaleA; p.scale_b = scaleB; p.bias = bias;
  p.groups = 1; p.N = N; p.K = K;
  p.act = (int)activMode; p.out = out; p.out_type = outType; p.ldo = ldo;
  return product(call, p, stream);
} catch (...) {
  return FAILED;
}

int occamy_matmul_grouped(const void *a, int type, int64_t aRows, int64_t lda, const float *scaleA, const int32_t *index,
                          const int32_t *offsets, int64_t groups, const void *b, int64_t ldb, const float *scaleB,
                          const float *bias, int64_t rows, int64_t N, int64_t K, int64_t activMode, void *out,
                          int outType, int64_t ldo, cudaStream_t stream) try {
  std::lock_guard<std::mutex> lock(g_mutex);
  Call call("occamy_matmul_grouped", stream);
  if (type != ELEM_BF16 && type != ELEM_F16 && type != ELEM_E4M3)
    return refuse(BAD_ARGUMENT, call.who(), "type of the operands");
  if (!linear_act(activMode) && activMode != ACT_GATED_SILU)
    return refuse(BAD_ARGUMENT, call.who(), "activation mode (0, 1, 2, 3, 5, 6 or 7)");
  if (groups < 0 || groups > MOST_EXPERTS) return refuse(BAD_ARGUMENT, call.who(), "0 to 1024 groups");
  if (!index && rows != aRows) return refuse(BAD_ARGUMENT, call.who(), "rows other than aRows need an index");
  if (rows > 0 && groups > 0 && !offsets) return refuse(BAD_ARGUMENT, call.who(), "null pointer");
  if (groups == 0) return 0;
  ProductArgs p = {};
  p.a = a; p.b = b; p.type = type;
  p.a_rows = aRows; p.rows = rows; p.lda = lda; p.ldb = ldb;
  p.scale_a = scaleA; p.scale_b = scaleB; p.bias = bias;
  p.index = index; p.offsets = offsets; p.groups = groups; p.N = N; p.K = K;
  p.act = (int)activMode; p.out = out; p.out_type = outType; p.ldo = ldo;
  return product(call, p, stream);
} catch (...) {
  return FAILED;
}

int64_t occamy_route_experts_workspace(int64_t tokens, int64_t experts, int64_t k) {
  if (!extent(tokens) || experts < 1 || experts > MOST_EXPERTS || k < 1 || k > MOST_CHOICES) return BAD_ARGUMENT;
  return (int64_t)route_workspace(tokens, experts, k);
}

int occamy_route_experts(const void *logits, int type, int64_t tokens, int64_t experts, int64_t ldl, int64_t k,
                         int normalise, int32_t *chosen, float *weights, int32_t *offsets, int32_t *order,
                         int32_t *position, void *workspace, int64_t workspaceBytes, cudaStream_t stream) try {
  std::lock_guard<std::mutex> lock(g_mutex);
  Call call("occamy_route_experts", stream);
  if (!real_type(type)) return refuse(BAD_ARGUMENT, call.who(), "type of the logits");
  if (!extent(tokens)) return refuse(BAD_ARGUMENT, call.who(), "extent out of range");
  if (experts < 1 || experts > MOST_EXPERTS) return refuse(BAD_ARGUMENT, call.who(), "1 to 1024 experts");
  if (k < 1 || k > MOST_CHOICES || k > experts)
    return refuse(BAD_ARGUMENT, call.who(), "1 to 32 choices, no more than experts");
  if (tokens * k > INT_MAX) return refuse(BAD_ARGUMENT, call.who(), "more than 2^31 - 1 rows");
  if (!row_length(ldl, experts, tokens, elem_size(type)))
    return refuse(BAD_ARGUMENT, call.who(), "distance between rows out of range");
  if (!offsets || (tokens && (!logits || !chosen || !weights || !order || !position)))
    return refuse(BAD_ARGUMENT, call.who(), "null pointer");
  const size_t need = route_workspace(tokens, experts, k);
  if (need && (!workspace || workspaceBytes < (int64_t)need))
    return refuse(TOO_SMALL, call.who(), "the workspace has to have %zu bytes", need);
  TRY(call.open());
  TRY(call.out(offsets, (experts + 1) * 4, 4));
  if (tokens == 0) {
    TRY(call.begin());
    rt().main_copies++;   // (that a later upload goes behind it: wrapDNNMemcpy)
    return call.end(cudaMemsetAsync(offsets, 0, (size_t)(experts + 1) * 4, stream), 0);
  }
  TRY(call.in(logits, span(tokens, ldl, experts, elem_size(type)), elem_size(type)));
  TRY(call.out(chosen, tokens * k * 4, 4));
  TRY(call.out(weights, tokens * k * 4, 4));
  TRY(call.out(order, tokens * k * 4, 4));
  TRY(call.out(position, tokens * k * 4, 4));
  TRY(call.out(workspace, (int64_t)need, 4));
  TRY(call.begin());
  RouteArgs a = {logits, type, tokens, experts, ldl, (int)k, normalise != 0, chosen, weights, offsets, order, position,
                 (int32_t *)workspace};
  return call.end(launch_route(a, stream), route_kernels(tokens));
} catch (...) {
  return FAILED;
}

int occamy_combine_experts(const void *y, int type, int64_t yRows, int64_t ldy, const int32_t *position,
                           const float *weights, int64_t tokens, int64_t k, int64_t N, void *out, int outType,
                           int64_t ldo, cudaStream_t stream) try {
  std::lock_guard<std::mutex> lock(g_mutex);
  Call call("occamy_combine_experts", stream);
  if (!real_type(type) || !real_type(outType)) return refuse(BAD_ARGUMENT, call.who(), "element type");
  if (!extent(yRows) || !extent(tokens) || !extent(N)) return refuse(BAD_ARGUMENT, call.who(), "extent out of range");
  if (k < 1 || k > MOST_CHOICES) return refuse(BAD_ARGUMENT, call.who(), "1 to 32 choices");
  if (!row_length(ldy, N, yRows, elem_size(type)) || !row_length(ldo, N, tokens, elem_size(outType)))
    return refuse(BAD_ARGUMENT, call.who(), "distance between rows out of range");
  if (tokens == 0 || N == 0) return 0;
  if ((yRows && !y) || !position || !weights || !out) return refuse(BAD_ARGUMENT, call.who(), "null pointer");
  TRY(call.open());
  if (yRows) TRY(call.in(y, span(yRows, ldy, N, elem_size(type)), elem_size(type)));
  TRY(call.in(position, tokens * k * 4, 4));
  TRY(call.in(weights, tokens * k * 4, 4));
  TRY(call.out(out, span(tokens, ldo, N, elem_size(outType)), elem_size(outType), ldo == N));
  TRY(call.begin());
  CombineArgs a = {y, type, yRows, ldy, position, weights, tokens, k, N, out, outType, ldo};
  return call.end(launch_combine(a, call.num_sms(), stream));
} catch (...) {
  return FAILED;
}

}  // extern "C"
