// kv_dev.h -- device code that the KV-cache operators' kernels share (gfx950,
// wave64): a request's lengths, lane exchanges, and the parts of an attention that
// do not depend on how keys and values are held.
#pragma once

#include <type_traits>

#include "kvops.h"
#include "s2hip.h"
#include "wave.h"

namespace s2 {
namespace {

// Slots in use and new tokens of a request; a request out of range has none.
// (Loaded and looked at apart, so that other loads can start in between.)
struct Request {
  uint32_t len, fresh;
};
struct RawRequest {
  int32_t len, fresh;
};
__device__ __forceinline__ RawRequest load_request(const KvCaches& c, uint32_t b) {
  return {c.lens[b], (c.new_lens ? c.new_lens : c.lens)[b]};
}
__device__ __forceinline__ Request checked(const KvCaches& c, RawRequest r, uint32_t* err) {
  if (!c.new_lens) r.fresh = r.len == 0 ? 0 : int32_t(c.n);
  const bool ok = r.len >= 0 && r.len <= int32_t(c.cap) && r.fresh >= 0 && r.fresh <= int32_t(c.n) && r.fresh <= r.len;
  if (!ok && err) atomicOr(err, S2HIP_KV_ERR_LENS);
  return ok ? Request{uint32_t(r.len), uint32_t(r.fresh)} : Request{0u, 0u};
}
__device__ __forceinline__ Request request_of(const KvCaches& c, uint32_t b, uint32_t* err) {
  return checked(c, load_request(c, b), err);
}

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int intx4 __attribute__((ext_vector_type(4)));

// Sum over lanes 0 .. l of the wave (all 64 active): shifts by 1, 2, 4, 8 within
// each 16 lanes, then their last lanes' sums to the rows behind them.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or_0(uint32_t x) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += dpp_or_0<0x111, 0xF>(x);  // row_shr:1
  x += dpp_or_0<0x112, 0xF>(x);
  x += dpp_or_0<0x114, 0xF>(x);
  x += dpp_or_0<0x118, 0xF>(x);
  x += dpp_or_0<0x142, 0xA>(x);  // row_bcast:15 to rows 1 and 3
  x += dpp_or_0<0x143, 0xC>(x);  // row_bcast:31 to rows 2 and 3
  return x;
}

// a value that is the same in all lanes, said so
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return uint32_t(__builtin_amdgcn_readfirstlane(int(x))); }

template <bool KH>
using Elem = std::conditional_t<KH, _Float16, float>;

// m follows a row's maximum only when it is SLACK behind: weights stay below
// 2^SLACK and the o registers are hardly ever rescaled.  It is a whole number, so
// that taking it off and the factors between states round nothing, and each row's
// goes by the keys that the row sees alone.  f16 parts of
// weights are of 2^(s - m + F16_LIFT), up to 2^14: the hi and the lo part of a small
// weight are exact to 2^-25 each, together 2^-30 of the largest.  The o of f32 values leave (and in
// kv_step_kernel grow) times F32_DOWN: 65536 weights then add no more than the
// largest value.
constexpr float SLACK = 8.0f, F16_LIFT = 6.0f, F32_DOWN = 0x1p-30f, F32_UP = 0x1p30f;

// max / sum over lanes l, l ^ 16, l ^ 32, l ^ 48
template <class Op>
__device__ __forceinline__ float quarter_reduce(float x, Op op) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quarter_max(float x) {
  return quarter_reduce(x, [](float p, float q) { return fmaxf(p, q); });
}
__device__ __forceinline__ float quarter_sum(float x) {
  return quarter_reduce(x, [](float p, float q) { return p + q; });
}

// op over lanes l and l ^ 32
template <class Op>
__device__ __forceinline__ float half_reduce(float x, Op op) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// a power of two r with max / r in [2^13, 2^14), and 1 / r; at least 2^LEAST.
// (Queries and keys: what the product of two such scales loses is of scores below
// 2^-80.  Values: times F32_DOWN and over a sum of weights it is a normal number.)
template <int LEAST = -126>
__device__ __forceinline__ void pow2_scale(float max, float& r, float& inv) {
  const int e = int((__float_as_uint(max) >> 23) & 255u) - 13;
  const uint32_t x = uint32_t(e < LEAST + 127 ? LEAST + 127 : e);
  r = __uint_as_float(x << 23);
  inv = __uint_as_float((254u - x) << 23);
}

// hi + lo parts of a query's element, below 2^14.  AWAY (f16 keys): hi is rounded away
// from 0, so that lo has the other sign or is 0, and an infinity of a key gives
// inf - inf or 0 x inf, no number, whichever its sign; lo, below 2^-10 then, is exact
// to 2^-22 of the element instead of 2^-23.  (The lo part of an f32 key's infinity is
// no number as it is.)
struct Parts {
  _Float16 hi, lo;
};
template <bool AWAY>
__device__ __forceinline__ Parts split_query(float x) {
  const float hi = AWAY ? __uint_as_float((__float_as_uint(x) + 0x1fffu) & 0xffffe000u) : float(_Float16(x));
  return {_Float16(hi), _Float16(x - hi)};
}

// Eight halfs of a tile's transposed values: rows (keys) of `row_bytes` bytes in
// LDS; lane i of 16 reads 8 bytes of row i / 4 and gets column i of four rows.
typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef __attribute__((address_space(3))) half8 lds_half8;
__device__ __forceinline__ half4 read_tr(lds_byte* p) {
  typedef short short4v __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p));
}

__device__ __forceinline__ bool not_zero(half8 z) {
  bool bad = false;
#pragma unroll
  for (int c = 0; c < 8; ++c) bad |= !(z[c] == _Float16(0));
  return bad;
}
// Ones where x is no number, which becomes 0 there.
__device__ __forceinline__ half8 take_odd(half8& x) {
  half8 marks;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const bool bad = !(__builtin_fabsf16(x[c]) < _Float16(INFINITY));
    marks[c] = bad ? _Float16(1) : _Float16(0);
    x[c] = bad ? _Float16(0) : x[c];
  }
  return marks;
}

}  // namespace
}  // namespace s2
