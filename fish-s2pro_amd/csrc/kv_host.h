// kv_host.h -- argument checks, errors and the C boundary that the KV-cache
// operators' handles share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <memory>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

namespace s2 {
namespace {

struct KvFailure : std::runtime_error {
  explicit KvFailure(const std::string& m) : std::runtime_error(m) {}
};
inline void hipc(hipError_t e, const char* what) {
  if (e != hipSuccess) throw KvFailure(std::string(what) + ": " + hipGetErrorString(e));
}
#define CHK(expr) hipc((expr), #expr)
[[noreturn]] inline void kfail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
inline void kfail(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  throw KvFailure(buf);
}

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

inline void need(const void* p, const char* name, size_t align) {
  if (!p) kfail("kv: %s is NULL", name);
  if (reinterpret_cast<uintptr_t>(p) % align) kfail("kv: %s is not aligned to %zu bytes", name, align);
}
inline void may(const void* p, const char* name, size_t align) {
  if (p) need(p, name, align);
}

// n words from p and m words from q have one in common.
inline bool meet(const void* p, size_t n, const void* q, size_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
  return x < y + 4 * m && y < x + 4 * n;
}
// out is in itself, or shares no word of `words` with it.
inline void same_or_apart(const void* in, const void* out, size_t words, const char* name) {
  if (in != out && meet(in, words, out, words)) kfail("kv: %s_out overlaps %s without being it", name, name);
}

// A handle's device memory, freed also where its constructor throws.
class DeviceArrays {
 protected:
  template <class T>
  T* alloc(size_t n) {
    void* p = nullptr;
    CHK(hipMalloc(&p, n * sizeof(T)));
    std::unique_ptr<void, Free> own(p);
    owned_.push_back(std::move(own));
    return static_cast<T*>(p);
  }

 private:
  struct Free {
    void operator()(void* p) const { (void)hipFree(p); }
  };
  std::vector<std::unique_ptr<void, Free>> owned_;
};

}  // namespace
}  // namespace s2

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
inline void kv_args(const void* kv, const void* view) {
  if (!kv || !view) throw std::runtime_error("NULL argument");
}
inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }
}  // namespace
