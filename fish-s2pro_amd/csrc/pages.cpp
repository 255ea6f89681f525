// pages.cpp -- the paged 4-bit KV cache behind the C ABI (include/s2hip.h,
// s2hip_pages_*): argument checks, the handle's workspace and the launches.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <stdexcept>
#include <string>
#include <vector>

#include "kv_host.h"
#include "pages.h"
#include "s2hip.h"

namespace s2 {
namespace {

constexpr uint32_t PG_MAX_PAGES = 1u << 20, PG_MAX_SLOTS = 1u << 20, PG_MAX_REQUESTS = 256, PG_MAX_TOKENS = 65536, PG_MAX_REP = 64,
                   PG_MAX_HEADS = 1024, PG_MAX_LAYERS = 1024, PG_MAX_ROPE_DIMS = 1u << 16;

struct Words {
  const void* p;
  size_t words;
  const char* name;
};
// No two of them share a word (those that are NULL share nothing).
void apart(const Words& x, const Words& y) {
  if (x.p && y.p && meet(x.p, x.words, y.p, y.words)) kfail("kv: %s overlaps %s", y.name, x.name);
}
template <size_t N>
void apart(const Words (&all)[N]) {
  for (size_t i = 0; i < N; ++i)
    for (size_t j = i + 1; j < N; ++j) apart(all[i], all[j]);
}

// An output that shares a word with an input.
template <size_t N, size_t M>
void outputs_apart(const Words (&outputs)[N], const Words (&inputs)[M]) {
  for (const Words& out : outputs)
    for (const Words& in : inputs) apart(in, out);
}
// A pool in every layer; what lies between the layers is the caller's.
struct Layers {
  const void* p;
  uint64_t bytes, stride;
  uint32_t n;
};
void pools_apart(const Layers& pools, const Words& x) {
  if (!x.p) return;
  const uint64_t base = reinterpret_cast<uintptr_t>(pools.p), at = reinterpret_cast<uintptr_t>(x.p), end = at + 4 * uint64_t(x.words);
  // the first layer that ends behind the array's beginning
  const uint64_t first = at < base + pools.bytes ? 0 : pools.n == 1 ? 1 : (at - base - pools.bytes) / pools.stride + 1;
  if (first < pools.n && base + first * pools.stride < end) kfail("kv: %s overlaps pool", x.name);
}
template <size_t N>
void pools_apart(const Layers& pools, const Words (&all)[N]) {
  for (const Words& x : all) pools_apart(pools, x);
}

class Pages : DeviceArrays {
 public:
  explicit Pages(const s2hip_pages_config& c) {
    if (c.kv_heads == 0 || c.heads == 0 || c.heads % c.kv_heads)
      kfail("kv: heads %u is not a multiple of kv_heads %u", c.heads, c.kv_heads);
    if (c.heads / c.kv_heads > PG_MAX_REP || c.heads > PG_MAX_HEADS)
      kfail("kv: heads %u over kv_heads %u is not supported (at most %u times, at most %u heads)", c.heads, c.kv_heads,
            PG_MAX_REP, PG_MAX_HEADS);
    if (c.head_dim != 64 && c.head_dim != 128) kfail("kv: head_dim %u is not 64 or 128", c.head_dim);
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128)
      kfail("kv: page_tokens %u is not 16, 32, 64 or 128", c.page_tokens);
    if (c.pages == 0 || c.pages > PG_MAX_PAGES) kfail("kv: pages %u is not in 1..%u", c.pages, PG_MAX_PAGES);
    if (c.table_pages == 0 || c.table_pages > PG_MAX_SLOTS / c.page_tokens)
      kfail("kv: table_pages %u is not in 1..%u", c.table_pages, PG_MAX_SLOTS / c.page_tokens);
    if (c.max_requests == 0 || c.max_requests > PG_MAX_REQUESTS)
      kfail("kv: max_requests %u is not in 1..%u", c.max_requests, PG_MAX_REQUESTS);
    if (c.max_tokens == 0 || c.max_tokens > PG_MAX_TOKENS) kfail("kv: max_tokens %u is not in 1..%u", c.max_tokens, PG_MAX_TOKENS);
    const uint32_t dims = c.rope_dims ? c.rope_dims : c.head_dim;
    if (c.rope_half > 1) kfail("kv: rope_half is %u, not 0 or 1", c.rope_half);
    if (dims > c.head_dim || dims % (c.rope_half ? 16 : 2))
      kfail("kv: rope_dims %u is not a multiple of %u up to head_dim %u", dims, c.rope_half ? 16 : 2, c.head_dim);
    if (!c.rope_freq && (!(c.rope_base > 0.0) || !std::isfinite(c.rope_base))) kfail("kv: rope_base is not positive");
    if (!(c.rope_gain >= 0.0) || !std::isfinite(c.rope_gain)) kfail("kv: rope_gain is negative");
    if (!(c.eps >= 0.0f) || !std::isfinite(c.eps)) kfail("kv: eps is negative");
    if (!(c.scale >= 0.0f) || !std::isfinite(c.scale)) kfail("kv: scale is negative");
    std::vector<double> turns(dims / 2);
    for (size_t i = 0; i < turns.size(); ++i) {
      const double f = c.rope_freq ? c.rope_freq[i] : std::pow(c.rope_base, -2.0 * double(i) / double(dims));
      if (!std::isfinite(f)) kfail("kv: rope_freq[%zu] is not finite", i);
      turns[i] = f / 6.283185307179586;
    }
    cfg_ = c;
    cfg_.rope_freq = nullptr;
    int ndev = 0;
    CHK(hipGetDeviceCount(&ndev));
    if (c.device < 0 || c.device >= ndev) kfail("HIP device %d not present", c.device);
    DeviceScope on(c.device);
    shape_.H = c.heads;
    shape_.G = c.kv_heads;
    shape_.rep = c.heads / c.kv_heads;
    shape_.scale2 = float((c.scale != 0.0f ? double(c.scale) : 1.0 / std::sqrt(double(c.head_dim))) * 1.4426950408889634);
    shape_.eps = c.eps;
    double* t = alloc<double>(turns.size());
    CHK(hipMemcpy(t, turns.data(), turns.size() * sizeof(double), hipMemcpyHostToDevice));
    rope_.turns = t;
    rope_.gain = c.rope_gain != 0.0 ? c.rope_gain : 1.0;
    rope_.dims = dims;
    rope_.half = c.rope_half;
    shape_.err = alloc<uint32_t>(2);
    CHK(hipMemset(shape_.err, 0, 2 * sizeof(uint32_t)));
    while ((1u << shift_) < c.page_tokens) ++shift_;
    chunk_ = c.page_tokens * (c.head_dim + c.head_dim / 8);
    work_.part = alloc<float>(size_t(PG_STATES) * 16 * c.head_dim);
    work_.part_ml = alloc<float>(size_t(PG_STATES) * 16 * 2);
    work_.ranges = alloc<uint2>(64);
    work_.refs = alloc<int32_t>(c.pages);
    work_.list = alloc<int32_t>(size_t(c.pages) * 2);
    work_.table = alloc<int32_t>(size_t(c.max_requests) * c.table_pages);
    work_.moves = alloc<int32_t>(2 * PG_MAX_REQUESTS);
    CHK(prepare_pg());
    CHK(hipDeviceSynchronize());
  }
  uint64_t bytes() const { return uint64_t(chunk_) * cfg_.kv_heads; }

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

  void append(const s2hip_pages_view& v, const float* qkv, uint32_t n, const int32_t* positions, const float* qn, const float* kn,
              float* q_out, float* k_held, float* v_held, hipStream_t s) {
    PgAppendArgs a{};
    a.p = pool(v);
    a.c = tokens(v, n);
    need(qkv, "qkv", 16);
    need(positions, "positions", 4);
    need(q_out, "q_out", 16);
    if (!qn != !kn) kfail("kv: q_norm and k_norm go together");
    may(qn, "q_norm", 16);
    may(kn, "k_norm", 16);
    may(k_held, "k_held", 16);
    may(v_held, "v_held", 16);
    const size_t rows = size_t(v.requests) * n, q = rows * cfg_.heads * cfg_.head_dim, kv = rows * cfg_.kv_heads * cfg_.head_dim;
    apart({{qkv, q + 2 * kv, "qkv"}, {q_out, q, "q_out"}, {k_held, kv, "k_held"}, {v_held, kv, "v_held"}});
    const Words outputs[] = {{q_out, q, "q_out"}, {k_held, kv, "k_held"}, {v_held, kv, "v_held"}};
    const Words inputs[] = {{positions, rows, "positions"}, {qn, cfg_.head_dim, "q_norm"}, {kn, cfg_.head_dim, "k_norm"}, {v.table, table_words(v), "table"},
                            {v.lens, v.requests, "lens"}, {v.new_lens, v.requests, "new_lens"}};
    outputs_apart(outputs, inputs);
    pools_apart(one_pool(v), outputs);
    pools_apart(one_pool(v), inputs);
    pools_apart(one_pool(v), Words{qkv, q + 2 * kv, "qkv"});
    a.s = shape_;
    a.rope = rope_;
    a.qkv = qkv;
    a.positions = positions;
    a.q_norm = qn;
    a.k_norm = kn;
    a.q_out = q_out;
    a.k_held = k_held;
    a.v_held = v_held;
    DeviceScope on(cfg_.device);
    CHK(launch_pg_append(cfg_.head_dim, a, s));
  }

  void attend(const s2hip_pages_view& v, const float* q, uint32_t n, float* out, hipStream_t s) {
    PgAttendArgs a{};
    a.p = pool(v);
    a.a.c = tokens(v, n);
    need(q, "q", 16);
    need(out, "out", 16);
    const size_t words = size_t(v.requests) * n * cfg_.heads * cfg_.head_dim;
    if (meet(q, words, out, words)) kfail("kv: out overlaps q");
    const Words outputs[] = {{out, words, "out"}};
    outputs_apart(outputs, {{v.table, table_words(v), "table"}, {v.lens, v.requests, "lens"}, {v.new_lens, v.requests, "new_lens"}});
    pools_apart(one_pool(v), outputs);
    a.a.s = shape_;
    a.a.q = q;
    a.a.out = out;
    DeviceScope on(cfg_.device);
    CHK(launch_pg_attend(cfg_.head_dim, a, work_, s));
  }

  void update(const s2hip_pages_view& v, uint32_t layers, uint64_t layer_stride, const int32_t* source, const int32_t* keep,
              const int32_t* add, const int32_t* refs, int32_t* refs_out, int32_t* table_out, int32_t* lens_out, hipStream_t s) {
    PgUpdateArgs a = rows(v, layers, layer_stride, refs, refs_out, table_out);
    may(source, "source", 4);
    may(keep, "keep", 4);
    may(add, "add", 4);
    need(lens_out, "lens_out", 4);
    same_or_apart(v.lens, lens_out, v.requests, "lens");
    const size_t R = v.requests, T = R * cfg_.table_pages, P = cfg_.pages;
    const Words r{refs_out, P, "refs_out"}, t{table_out, T, "table_out"}, l{lens_out, R, "lens_out"};
    apart({r, t, l});
    for (const Words& out : {r, t, l})
      for (const Words& in : {Words{source, R, "source"}, Words{keep, R, "keep"}, Words{add, R, "add"}, Words{out.p == refs_out ? nullptr : refs, P, "refs"},
                              Words{out.p == table_out ? nullptr : v.table, T, "table"}, Words{out.p == lens_out ? nullptr : v.lens, R, "lens"}})
        apart(in, out);
    pools_apart({v.pool, bytes() * P, a.layer_stride, layers},
                {r, t, l, {source, R, "source"}, {keep, R, "keep"}, {add, R, "add"}, {refs, P, "refs"}, {v.table, T, "table"}, {v.lens, R, "lens"}});
    a.source = source;
    a.keep = keep;
    a.add = add;
    a.lens_out = lens_out;
    DeviceScope on(cfg_.device);
    CHK(launch_pg_update(a, work_, uint32_t(bytes()), s));
  }

  void compact(const s2hip_pages_view& v, uint32_t layers, uint64_t layer_stride, const int32_t* refs, int32_t* refs_out,
               int32_t* table_out, int32_t* used_out, int32_t* moved_to, hipStream_t s) {
    PgUpdateArgs a = rows(v, layers, layer_stride, refs, refs_out, table_out);
    need(used_out, "used_out", 4);
    may(moved_to, "moved_to", 4);
    const size_t R = v.requests, T = R * cfg_.table_pages, P = cfg_.pages;
    const Words r{refs_out, P, "refs_out"}, t{table_out, T, "table_out"}, u{used_out, 1, "used_out"}, m{moved_to, P, "moved_to"};
    apart({r, t, u, m});
    for (const Words& out : {r, t, u, m})
      for (const Words& in : {Words{out.p == refs_out ? nullptr : refs, P, "refs"}, Words{out.p == table_out ? nullptr : v.table, T, "table"}, Words{v.lens, R, "lens"}})
        apart(in, out);
    pools_apart({v.pool, bytes() * P, a.layer_stride, layers}, {r, t, u, m, {refs, P, "refs"}, {v.table, T, "table"}, {v.lens, R, "lens"}});
    a.used_out = used_out;
    a.moved_to = moved_to;
    DeviceScope on(cfg_.device);
    CHK(launch_pg_compact(a, work_, uint32_t(bytes()), s));
  }

 private:
  PgPool pool(const s2hip_pages_view& v) const {
    if (v.requests == 0 || v.requests > cfg_.max_requests)
      kfail("kv: requests %u is not in 1..max_requests %u", v.requests, cfg_.max_requests);
    need(v.pool, "pool", 16);
    need(v.table, "table", 4);
    need(v.lens, "lens", 4);
    return {static_cast<uint8_t*>(v.pool), v.table, shift_, cfg_.pages, cfg_.table_pages, chunk_};
  }

  size_t table_words(const s2hip_pages_view& v) const { return size_t(v.requests) * cfg_.table_pages; }
  Layers one_pool(const s2hip_pages_view& v) const { return {v.pool, bytes() * cfg_.pages, bytes() * cfg_.pages, 1}; }

  KvCaches tokens(const s2hip_pages_view& v, uint32_t n) const {
    if (n == 0 || uint64_t(v.requests) * n > cfg_.max_tokens)
      kfail("kv: %u requests of n_tokens %u are not in 1..max_tokens %u", v.requests, n, cfg_.max_tokens);
    may(v.new_lens, "new_lens", 4);
    KvCaches c{};
    c.lens = v.lens;
    c.new_lens = v.new_lens;
    c.R = v.requests;
    c.n = n;
    c.cap = cfg_.table_pages << shift_;
    return c;
  }

  PgUpdateArgs rows(const s2hip_pages_view& v, uint32_t layers, uint64_t layer_stride, const int32_t* refs, int32_t* refs_out, int32_t* table_out) const {
    PgUpdateArgs a{};
    a.p = pool(v);
    const uint64_t all = bytes() * cfg_.pages;
    if (layers == 0 || layers > PG_MAX_LAYERS) kfail("kv: layers %u is not in 1..%u", layers, PG_MAX_LAYERS);
    if (layer_stride % 16) kfail("kv: layer_stride %llu is not a multiple of 16 bytes", (unsigned long long)layer_stride);
    if (layer_stride && layer_stride < all) kfail("kv: layer_stride %llu is below the %llu bytes of a pool", (unsigned long long)layer_stride, (unsigned long long)all);
    if (layer_stride >> 48) kfail("kv: layer_stride %llu is too large", (unsigned long long)layer_stride);
    need(refs, "refs", 4);
    need(refs_out, "refs_out", 4);
    need(table_out, "table_out", 4);
    same_or_apart(refs, refs_out, cfg_.pages, "refs");
    same_or_apart(v.table, table_out, size_t(v.requests) * cfg_.table_pages, "table");
    a.lens = v.lens;
    a.refs = refs;
    a.refs_out = refs_out;
    a.table_out = table_out;
    a.layers = layers;
    a.layer_stride = layer_stride ? layer_stride : all;
    a.R = v.requests;
    a.err = shape_.err;
    return a;
  }

  s2hip_pages_config cfg_{};
  KvShape shape_{};
  PgRope rope_{};
  PgWorkspace work_{};
  uint32_t shift_ = 0, chunk_ = 0;
};

}  // namespace
}  // namespace s2

struct s2hip_pages {
  std::unique_ptr<s2::Pages> ops;
};

extern "C" {

int32_t s2hip_rope_frequencies(uint32_t dims, double base, uint32_t scaling, double factor, double context, double low,
                               double high, double* freq, double* gain, char* err, size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    if (!freq || !gain) throw std::runtime_error("NULL argument");
    if (dims == 0 || dims % 2 || dims > s2::PG_MAX_ROPE_DIMS) s2::kfail("rope: dims %u is not an even number of 2..%u", dims, s2::PG_MAX_ROPE_DIMS);
    if (!(base > 0.0) || !std::isfinite(base)) s2::kfail("rope: base is not positive");
    if (scaling > S2HIP_ROPE_PARTS) s2::kfail("rope: scaling %u is not known", scaling);
    if (scaling != S2HIP_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) s2::kfail("rope: factor is not at least 1");
    if (scaling == S2HIP_ROPE_STRETCH && dims < 4) s2::kfail("rope: dims %u is too few to stretch", dims);
    if (scaling == S2HIP_ROPE_PARTS && (!(context > 0.0) || !std::isfinite(context))) s2::kfail("rope: context is not positive");
    if (scaling == S2HIP_ROPE_PARTS && (!(low >= 0.0) || !(low < high) || !std::isfinite(high))) s2::kfail("rope: low is not below high");
    const double n = double(dims), b = scaling == S2HIP_ROPE_STRETCH ? base * std::pow(factor, n / (n - 2.0)) : base;
    for (uint32_t i = 0; i < dims / 2; ++i) {
      double f = std::pow(b, -2.0 * double(i) / n);
      if (scaling == S2HIP_ROPE_LINEAR) f /= factor;
      if (scaling == S2HIP_ROPE_PARTS) {
        const double turns = context * f / 6.283185307179586, stays = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
        f = f / factor * (1.0 - stays) + f * stays;
      }
      freq[i] = f;
    }
    *gain = scaling == S2HIP_ROPE_PARTS ? 1.0 + 0.1 * std::log(factor) : 1.0;
  });
}

s2hip_pages* s2hip_pages_open(const s2hip_pages_config* cfg, char* err, size_t err_cap) {
  s2hip_pages* h = nullptr;
  kv_guarded(err, err_cap, [&] {
    if (!cfg) throw std::runtime_error("config is NULL");
    std::unique_ptr<s2hip_pages> tmp(new s2hip_pages());
    tmp->ops.reset(new s2::Pages(*cfg));
    h = tmp.release();
  });
  return h;
}

void s2hip_pages_close(s2hip_pages* pages) { delete pages; }

uint64_t s2hip_pages_bytes(const s2hip_pages* pages) { return pages ? pages->ops->bytes() : 0; }

int32_t s2hip_pages_errors(s2hip_pages* pages, void* stream, uint32_t* bits, char* err, size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(pages, bits);
    *bits = pages->ops->errors(as_stream(stream));
  });
}

int32_t s2hip_pages_append(s2hip_pages* pages, const s2hip_pages_view* view, const float* qkv, uint32_t n_tokens,
                           const int32_t* positions, const float* q_norm, const float* k_norm, float* q_out,
                           float* k_held, float* v_held, void* stream, char* err, size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(pages, view);
    pages->ops->append(*view, qkv, n_tokens, positions, q_norm, k_norm, q_out, k_held, v_held, as_stream(stream));
  });
}

int32_t s2hip_pages_attend(s2hip_pages* pages, const s2hip_pages_view* view, const float* q, uint32_t n_tokens,
                           float* out, void* stream, char* err, size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(pages, view);
    pages->ops->attend(*view, q, n_tokens, out, as_stream(stream));
  });
}

int32_t s2hip_pages_update(s2hip_pages* pages, const s2hip_pages_view* view, uint32_t layers, uint64_t layer_stride,
                           const int32_t* source, const int32_t* keep, const int32_t* add, const int32_t* refs,
                           int32_t* refs_out, int32_t* table_out, int32_t* lens_out, void* stream, char* err,
                           size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(pages, view);
    pages->ops->update(*view, layers, layer_stride, source, keep, add, refs, refs_out, table_out, lens_out, as_stream(stream));
  });
}

int32_t s2hip_pages_compact(s2hip_pages* pages, const s2hip_pages_view* view, uint32_t layers, uint64_t layer_stride,
                            const int32_t* refs, int32_t* refs_out, int32_t* table_out, int32_t* used_out,
                            int32_t* moved_to, void* stream, char* err, size_t err_cap) {
  return kv_guarded(err, err_cap, [&] {
    kv_args(pages, view);
    pages->ops->compact(*view, layers, layer_stride, refs, refs_out, table_out, used_out, moved_to, as_stream(stream));
  });
}

}  // extern "C"
