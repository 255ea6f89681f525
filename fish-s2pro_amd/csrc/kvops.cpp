// kvops.cpp -- the KV-cache operators behind the C ABI (include/s2hip.h,
// s2hip_kv_*): argument checks, the handle's workspace and the launches.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <memory>
#include <stdexcept>
#include <string>
#include <vector>

#include "kvops.h"
#include "s2hip.h"

namespace s2 {
namespace {

struct KvFailure : std::runtime_error {
  explicit KvFailure(const std::string& m) : std::runtime_error(m) {}
};
void hipc(hipError_t e, const char* what) {
  if (e != hipSuccess) throw KvFailure(std::string(what) + ": " + hipGetErrorString(e));
}
#define CHK(expr) hipc((expr), #expr)
[[noreturn]] void kfail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
void kfail(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  throw KvFailure(buf);
}

constexpr uint32_t KV_MAX_SLOTS = 32768, KV_MAX_REQUESTS = 256, KV_MAX_TOKENS = 65536, KV_MAX_REP = 64,
                   KV_MAX_HEADS = 1024, KV_MAX_LAYERS = 1024;

// The handle's device for the length of a call; the caller's afterwards.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    CHK(hipGetDevice(&was_));
    if (was_ != device) {
      CHK(hipSetDevice(device));
      moved_ = true;
    }
  }
  ~DeviceScope() {
    if (moved_) (void)hipSetDevice(was_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int was_ = 0;
  bool moved_ = false;
};

void need(const void* p, const char* name, size_t align) {
  if (!p) kfail("kv: %s is NULL", name);
  if (reinterpret_cast<uintptr_t>(p) % align) kfail("kv: %s is not aligned to %zu bytes", name, align);
}
void may(const void* p, const char* name, size_t align) {
  if (p) need(p, name, align);
}

// n words from p and m words from q have one in common.
bool meet(const void* p, size_t n, const void* q, size_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
  return x < y + 4 * m && y < x + 4 * n;
}
// out is in itself, or shares no word of `words` with it.
void same_or_apart(const void* in, const void* out, size_t words, const char* name) {
  if (in != out && meet(in, words, out, words)) kfail("kv: %s_out overlaps %s without being it", name, name);
}

// A dimension of the caches' layout.
struct Dim {
  uint64_t size, stride;
};
// Rows of `row` elements share none: sorted by stride, each dimension steps over all of those before it.
template <size_t N>
void check_apart(Dim (&dims)[N], uint64_t row) {
  std::sort(dims, dims + N, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
  uint64_t extent = row;
  for (const Dim& d : dims) {
    if (d.size == 1) continue;
    if (d.stride < extent) kfail("kv: the strides make caches overlap (one of %llu is less than the %llu elements below it)",
                                 (unsigned long long)d.stride, (unsigned long long)extent);
    extent += (d.size - 1) * d.stride;
  }
}

class KvOps {
 public:
  explicit KvOps(const s2hip_kv_config& c) {
    if (c.kv_heads == 0 || c.heads == 0 || c.heads % c.kv_heads)
      kfail("kv: heads %u is not a multiple of kv_heads %u", c.heads, c.kv_heads);
    if (c.heads / c.kv_heads > KV_MAX_REP || c.heads > KV_MAX_HEADS)
      kfail("kv: heads %u over kv_heads %u is not supported (at most %u times, at most %u heads)", c.heads, c.kv_heads,
            KV_MAX_REP, KV_MAX_HEADS);
    if (c.head_dim != 64 && c.head_dim != 128) kfail("kv: head_dim %u is not 64 or 128", c.head_dim);
    if (c.kv_f16 > 1) kfail("kv: kv_f16 is %u, not 0 or 1", c.kv_f16);
    if (c.max_requests == 0 || c.max_requests > KV_MAX_REQUESTS)
      kfail("kv: max_requests %u is not in 1..%u", c.max_requests, KV_MAX_REQUESTS);
    if (c.max_tokens == 0 || c.max_tokens > KV_MAX_TOKENS) kfail("kv: max_tokens %u is not in 1..%u", c.max_tokens, KV_MAX_TOKENS);
    if (!(c.rope_base > 0.0f) || !std::isfinite(c.rope_base)) kfail("kv: rope_base is not positive");
    if (!(c.eps >= 0.0f) || !std::isfinite(c.eps)) kfail("kv: eps is negative");
    if (!(c.scale >= 0.0f) || !std::isfinite(c.scale)) kfail("kv: scale is negative");
    cfg_ = c;
    int ndev = 0;
    CHK(hipGetDeviceCount(&ndev));
    if (c.device < 0 || c.device >= ndev) kfail("HIP device %d not present", c.device);
    DeviceScope on(c.device);
    shape_.H = c.heads;
    shape_.G = c.kv_heads;
    shape_.rep = c.heads / c.kv_heads;
    shape_.scale2 = float((c.scale != 0.0f ? double(c.scale) : 1.0 / std::sqrt(double(c.head_dim))) * 1.4426950408889634);
    shape_.eps = c.eps;
    std::vector<double> freq(c.head_dim / 2);
    for (size_t i = 0; i < freq.size(); ++i)
      freq[i] = std::pow(double(c.rope_base), -2.0 * double(i) / double(c.head_dim));
    double* f = alloc<double>(freq.size());
    CHK(hipMemcpy(f, freq.data(), freq.size() * sizeof(double), hipMemcpyHostToDevice));
    shape_.freq = f;
    shape_.err = alloc<uint32_t>(2);
    CHK(hipMemset(shape_.err, 0, 2 * sizeof(uint32_t)));
    work_.stat = alloc<float>(size_t(c.max_tokens) * c.heads * 2);
    work_.cap_parts = 8192;
    work_.part = alloc<float>(work_.cap_parts * 16 * c.head_dim);
    work_.part_ml = alloc<float>(work_.cap_parts * 16 * 2);
    work_.cap_weights = size_t(1) << 25;
    work_.weights = alloc<float>(work_.cap_weights);
    work_.moves = alloc<uint32_t>(size_t(KV_LISTS) * KV_LIST);
    work_.counts = alloc<uint32_t>(2 * KV_LISTS);
    CHK(hipDeviceSynchronize());
  }
  uint32_t errors(hipStream_t s) {
    DeviceScope on(cfg_.device);
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    CHK(hipStreamIsCapturing(s, &st));
    if (st != hipStreamCaptureStatusNone) kfail("kv: errors waits for its stream, which is being captured");
    uint32_t bits = 0;
    CHK(launch_kv_take_errors(shape_.err, shape_.err + 1, s));
    CHK(hipMemcpyAsync(&bits, shape_.err + 1, sizeof bits, hipMemcpyDeviceToHost, s));
    CHK(hipStreamSynchronize(s));
    return bits;
  }

  void append(const s2hip_kv_view& v, const float* qkv, uint32_t n, const int32_t* positions, const float* qn,
              const float* kn, float* q_out, float* scores, int32_t* slot_positions, hipStream_t s) {
    KvAppendArgs a{};
    a.c = caches(v, n, true, false);
    need(qkv, "qkv", 16);
    need(positions, "positions", 4);
    need(q_out, "q_out", 16);
    const size_t tokens = size_t(v.requests) * n;
    if (meet(qkv, tokens * (cfg_.heads + 2 * cfg_.kv_heads) * cfg_.head_dim, q_out, tokens * cfg_.heads * cfg_.head_dim))
      kfail("kv: q_out overlaps qkv");
    if (!qn != !kn) kfail("kv: q_norm and k_norm go together");
    may(qn, "q_norm", 16);
    may(kn, "k_norm", 16);
    may(scores, "scores", 4);
    may(slot_positions, "slot_positions", 4);
    a.s = shape_;
    a.qkv = qkv;
    a.positions = positions;
    a.q_norm = qn;
    a.k_norm = kn;
    a.q_out = q_out;
    a.scores = scores;
    a.slot_positions = slot_positions;
    DeviceScope on(cfg_.device);
    CHK(launch_kv_append(cfg_.head_dim, cfg_.kv_f16, a, s));
  }

  void attend(const s2hip_kv_view& v, const float* q, uint32_t n, float* out, bool weigh, const float* w_in, float* w_out,
              const float* pw_in, float* pw_out, hipStream_t s) {
    KvAttendArgs a{};
    a.c = caches(v, n, true, true);
    need(q, "q", 16);
    need(out, "out", 16);
    const size_t words = size_t(v.requests) * n * cfg_.heads * cfg_.head_dim;
    if (meet(q, words, out, words)) kfail("kv: out overlaps q");
    if (weigh) {
      need(w_out, "weights_out", 4);
      may(w_in, "weights_in", 4);
      may(pw_in, "prefix_weights_in", 4);
      may(pw_out, "prefix_weights_out", 4);
      if (w_in) same_or_apart(w_in, w_out, size_t(v.requests) * cfg_.kv_heads * v.capacity, "weights");
      if (pw_in && pw_out)
        same_or_apart(pw_in, pw_out, size_t(cfg_.kv_heads) * (v.prefix_capacity ? v.prefix_capacity : v.prefix_len), "prefix_weights");
      if (pw_in && !pw_out) kfail("kv: prefix_weights_in without prefix_weights_out");
      a.w_in = w_in;
      a.w_out = w_out;
      a.pw_in = pw_in;
      a.pw_out = v.prefix_len ? pw_out : nullptr;
      a.pw_stride = v.prefix_capacity ? v.prefix_capacity : v.prefix_len;
    }
    a.s = shape_;
    a.q = q;
    a.out = out;
    DeviceScope on(cfg_.device);
    CHK(launch_kv_attend(cfg_.head_dim, cfg_.kv_f16, a, work_, s));
  }

  void evict(const s2hip_kv_view& v, uint32_t layers, uint64_t layer_stride, uint32_t keep, uint32_t recent, uint32_t sinks,
             const float* scores, const int32_t* positions, float* scores_out, int32_t* positions_out, int32_t* lens_out,
             hipStream_t s) {
    KvEvictArgs a{};
    a.c = caches(v, 0, false, false);
    if (layers == 0 || layers > KV_MAX_LAYERS) kfail("kv: layers %u is not in 1..%u", layers, KV_MAX_LAYERS);
    if (keep == 0) kfail("kv: keep is 0");
    if (recent > keep) kfail("kv: recent %u is more than keep %u", recent, keep);
    stride(layer_stride, "layer_stride");
    need(scores, "scores", 4);
    need(positions, "positions", 4);
    need(scores_out, "scores_out", 4);
    need(positions_out, "positions_out", 4);
    need(lens_out, "lens_out", 4);
    const size_t words = size_t(layers) * v.requests * cfg_.kv_heads * v.capacity;
    same_or_apart(scores, scores_out, words, "scores");
    same_or_apart(positions, positions_out, words, "positions");
    same_or_apart(v.lens, lens_out, v.requests, "lens");
    a.s = shape_;
    a.layer_stride = layer_stride ? layer_stride : std::max({a.c.req_stride * v.requests, a.c.head_stride * cfg_.kv_heads, a.c.slot_stride * v.capacity});
    Dim dims[] = {{layers, a.layer_stride}, {v.requests, a.c.req_stride}, {cfg_.kv_heads, a.c.head_stride}, {v.capacity, a.c.slot_stride}};
    check_apart(dims, cfg_.head_dim);
    a.layers = layers;
    a.keep = keep;
    a.recent = recent;
    a.sinks = sinks;
    a.scores = scores;
    a.positions = positions;
    a.scores_out = scores_out;
    a.positions_out = positions_out;
    a.lens_out = lens_out;
    DeviceScope on(cfg_.device);
    a.elem = cfg_.kv_f16 ? 2 : 4;
    CHK(launch_kv_evict(a, work_, cfg_.head_dim, s));
  }

 private:
  struct Free {
    void operator()(void* p) const { (void)hipFree(p); }
  };
  template <class T>
  T* alloc(size_t n) {
    void* p = nullptr;
    CHK(hipMalloc(&p, n * sizeof(T)));
    std::unique_ptr<void, Free> own(p);
    owned_.push_back(std::move(own));
    return static_cast<T*>(p);
  }

  void stride(uint64_t n, const char* name) const {
    const uint64_t unit = cfg_.kv_f16 ? 8 : 4;
    if (n % unit) kfail("kv: %s %llu is not a multiple of 16 bytes", name, (unsigned long long)n);
    if (n >> 40) kfail("kv: %s %llu is too large", name, (unsigned long long)n);
  }

  // The view's checks; strides of 0 become those that step over all below.  tokens: a call with n per request.
  KvCaches caches(const s2hip_kv_view& v, uint32_t n, bool tokens, bool prefix) const {
    if (v.requests == 0 || v.requests > cfg_.max_requests)
      kfail("kv: requests %u is not in 1..max_requests %u", v.requests, cfg_.max_requests);
    if (tokens && (n == 0 || uint64_t(v.requests) * n > cfg_.max_tokens))
      kfail("kv: %u requests of n_tokens %u are not in 1..max_tokens %u", v.requests, n, cfg_.max_tokens);
    if (v.capacity == 0 || v.capacity > KV_MAX_SLOTS) kfail("kv: capacity %u is not in 1..%u", v.capacity, KV_MAX_SLOTS);
    need(v.k, "k", 16);
    need(v.v, "v", 16);
    need(v.lens, "lens", 4);
    may(v.new_lens, "new_lens", 4);
    stride(v.request_stride, "request_stride");
    stride(v.head_stride, "head_stride");
    stride(v.slot_stride, "slot_stride");
    KvCaches c{};
    c.k = v.k;
    c.v = v.v;
    c.lens = v.lens;
    c.new_lens = v.new_lens;
    c.slot_stride = v.slot_stride ? v.slot_stride : cfg_.head_dim;
    c.head_stride = v.head_stride ? v.head_stride : c.slot_stride * v.capacity;
    c.req_stride = v.request_stride ? v.request_stride : std::max(c.head_stride * cfg_.kv_heads, c.slot_stride * v.capacity);
    if (c.slot_stride >> 24) kfail("kv: slot_stride %llu is not below 2^24", (unsigned long long)c.slot_stride);
    if (c.slot_stride < cfg_.head_dim) kfail("kv: slot_stride %llu is below head_dim %u", (unsigned long long)c.slot_stride, cfg_.head_dim);
    if (c.head_stride < cfg_.head_dim) kfail("kv: head_stride %llu is below head_dim %u", (unsigned long long)c.head_stride, cfg_.head_dim);
    if (c.req_stride < cfg_.head_dim) kfail("kv: request_stride %llu is below head_dim %u", (unsigned long long)c.req_stride, cfg_.head_dim);
    Dim dims[] = {{v.requests, c.req_stride}, {cfg_.kv_heads, c.head_stride}, {v.capacity, c.slot_stride}};
    check_apart(dims, cfg_.head_dim);
    c.R = v.requests;
    c.cap = v.capacity;
    c.n = n;
    if (!prefix) return c;
    if (v.prefix_len > KV_MAX_SLOTS) kfail("kv: prefix_len %u is above %u", v.prefix_len, KV_MAX_SLOTS);
    if (v.prefix_capacity && (v.prefix_capacity < v.prefix_len || v.prefix_capacity > KV_MAX_SLOTS))
      kfail("kv: prefix_capacity %u is not in prefix_len %u..%u", v.prefix_capacity, v.prefix_len, KV_MAX_SLOTS);
    if (v.prefix_len == 0) return c;
    need(v.prefix_k, "prefix_k", 16);
    need(v.prefix_v, "prefix_v", 16);
    stride(v.prefix_head_stride, "prefix_head_stride");
    stride(v.prefix_slot_stride, "prefix_slot_stride");
    c.pk = v.prefix_k;
    c.pv = v.prefix_v;
    c.P = v.prefix_len;
    c.p_slot_stride = v.prefix_slot_stride ? v.prefix_slot_stride : cfg_.head_dim;
    c.p_head_stride = v.prefix_head_stride ? v.prefix_head_stride : c.p_slot_stride * (v.prefix_capacity ? v.prefix_capacity : v.prefix_len);
    if (c.p_slot_stride >> 24) kfail("kv: prefix_slot_stride %llu is not below 2^24", (unsigned long long)c.p_slot_stride);
    if (c.p_slot_stride < cfg_.head_dim)
      kfail("kv: prefix_slot_stride %llu is below head_dim %u", (unsigned long long)c.p_slot_stride, cfg_.head_dim);
    if (c.p_head_stride < cfg_.head_dim)
      kfail("kv: prefix_head_stride %llu is below head_dim %u", (unsigned long long)c.p_head_stride, cfg_.head_dim);
    return c;
  }

  s2hip_kv_config cfg_{};
  KvShape shape_{};
  KvWorkspace work_{};
  std::vector<std::unique_ptr<void, Free>> owned_;  // freed also where the constructor throws
};

}  // namespace
}  // namespace s2

struct s2hip_kv {
  std::unique_ptr<s2::KvOps> ops;
};

namespace {
template <class F>
int32_t kv_guarded(char* err, size_t cap, F&& f) {
  const char* what = "unknown error";
  try {
    f();
    return 1;
  } catch (const std::exception& ex) {
    if (err && cap) snprintf(err, cap, "%s", ex.what());
    return 0;
  } catch (...) {
  }
  if (err && cap) snprintf(err, cap, "%s", what);
  return 0;
}
void kv_args(const s2hip_kv* kv, const void* view) {
  if (!kv || !view) throw std::runtime_error("NULL argument");
}
hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }
}  // namespace

extern "C" {

s2hip_kv* s2hip_kv_open(const s2hip_kv_config* cfg, char* err, size_t err_cap) {
  s2hip_kv* h = nullptr;
  kv_guarded(err, err_cap, [&] {
    if (!cfg) throw std::runtime_error("config is NULL");
    std::unique_ptr<s2hip_kv> tmp(new s2hip_kv());
    tmp->ops.reset(new s2::KvOps(*cfg));
    h = tmp.release();
  });
  return h;
}

void s2hip_kv_close(s2hip_kv* kv) { delete kv; }

int32_t s2hip_kv_errors(s2hip_kv* kv, void* stream, uint32_t* bits, char* err, size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(kv, bits);
    *bits = kv->ops->errors(as_stream(stream));
  });
}

int32_t s2hip_kv_append(s2hip_kv* kv, const s2hip_kv_view* view, const float* qkv, uint32_t n_tokens,
                        const int32_t* positions, const float* q_norm, const float* k_norm, float* q_out,
                        float* scores, int32_t* slot_positions, void* stream, char* err, size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(kv, view);
    kv->ops->append(*view, qkv, n_tokens, positions, q_norm, k_norm, q_out, scores, slot_positions, as_stream(stream));
  });
}

int32_t s2hip_kv_attend(s2hip_kv* kv, const s2hip_kv_view* view, const float* q, uint32_t n_tokens, float* out,
                        void* stream, char* err, size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(kv, view);
    kv->ops->attend(*view, q, n_tokens, out, false, nullptr, nullptr, nullptr, nullptr, as_stream(stream));
  });
}

int32_t s2hip_kv_attend_weigh(s2hip_kv* kv, const s2hip_kv_view* view, const float* q, uint32_t n_tokens, float* out,
                              const float* weights_in, float* weights_out, const float* prefix_weights_in,
                              float* prefix_weights_out, void* stream, char* err, size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(kv, view);
    kv->ops->attend(*view, q, n_tokens, out, true, weights_in, weights_out, prefix_weights_in, prefix_weights_out,
                    as_stream(stream));
  });
}

int32_t s2hip_kv_evict(s2hip_kv* kv, const s2hip_kv_view* view, uint32_t layers, uint64_t layer_stride, uint32_t keep,
                       uint32_t recent, uint32_t sinks, const float* scores, const int32_t* positions,
                       float* scores_out, int32_t* positions_out, int32_t* lens_out, void* stream, char* err,
                       size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(kv, view);
    kv->ops->evict(*view, layers, layer_stride, keep, recent, sinks, scores, positions, scores_out, positions_out, lens_out,
                   as_stream(stream));
  });
}

}  // extern "C"
