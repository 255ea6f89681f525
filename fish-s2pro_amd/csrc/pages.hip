// pages.hip -- a KV cache in pages, keys and values in 4 bits, for gfx950 (CDNA4,
// wave64): head norms, rotation and cache write of a batch's new tokens; attention
// over the requests' pages; the rows of pages made anew; a pool compacted.

#include "kv_dev.h"
#include "launch.h"
#include "lds_dma.h"
#include "pages.h"

namespace s2 {
namespace {

static_assert(S2HIP_PAGES_ERR_LENS == S2HIP_KV_ERR_LENS, "checked() reports for both");

// Where a kv head's parts of a page begin, in bytes from the part: key codes at 0,
// value codes, key scales, value scales (f16).
template <int HD>
struct Chunk {
  uint32_t shift;
  __device__ __forceinline__ uint32_t v() const { return (HD / 2) << shift; }
  __device__ __forceinline__ uint32_t ks() const { return HD << shift; }
  __device__ __forceinline__ uint32_t vs() const { return (HD + HD / 16) << shift; }
};

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// 1 / 8 of the largest of 32 numbers to 8 significant bits, at the bottom to
// multiples of 2^-24 (powers of two take and give back the rest exactly).
__device__ __forceinline__ double rounded8(double x) {
  const int e = max(int((__double_as_longlong(x) >> 52) & 2047) - 1023 - 7, -24);
  return ldexp(rint(ldexp(x, -e)), e);
}

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t v = uint64_t(__double_as_longlong(x));
  return __longlong_as_double((long long)(uint64_t(dpp_u32<CTRL>(uint32_t(v >> 32))) << 32 | dpp_u32<CTRL>(uint32_t(v))));
}

// One block per token and run of heads (blockIdx.y, every gridDim.y-th 16 or 32), 8
// elements per thread.  Norms, angles, rotation and what is rounded to 4 bits are in
// 64 bits, whose instructions cost what those of 32 bits do here: a rounding of f32 in
// front would move a code across a border now and then, and the element by a sixteenth
// of its block's range.
//   Memory bounds a turn: 8 x 250 tokens of 32 + 2 x 8 heads of 128, 78 MB, 20.4 us (3.9
// TB/s), vector units 28 % busy.  A step's token is split over blocks by runs of heads
// (up to 512 blocks; 8 x 1 tokens in 3.9 us, all of it latency).
template <int HD, bool HALF>
__global__ __launch_bounds__(256) void pg_append_kernel(PgAppendArgs a) {
  constexpr uint32_t LP = HD / 8;     // lanes per head
  constexpr uint32_t HPB = 256 / LP;  // heads per step of the block
  constexpr int PAIRS = HALF ? 8 : 4;
  __shared__ double2 turn[HD / 2];
  __shared__ __align__(16) float gains[2][HD];  // of queries, of keys
  const uint32_t tid = threadIdx.x, b = blockIdx.x / a.c.n, t = blockIdx.x % a.c.n;
  const RawRequest raw = load_request(a.c, b);
  const int32_t pos = a.positions[size_t(b) * a.c.n + t];
  const uint32_t heads = a.s.H + 2 * a.s.G, l = tid % LP, d0 = 8 * l, half = a.rope.dims / 2, h0 = blockIdx.y * HPB + tid / LP;
  const float* src = a.qkv + (size_t(b) * a.c.n + t) * heads * HD;
  // in halves: the other half's elements, 8 dims of it
  const bool turns = d0 < a.rope.dims, second = HALF && d0 >= half;
  const uint32_t o0 = HALF && turns ? (second ? d0 - half : d0 + half) : d0;
  float x[8], z[HALF ? 8 : 1];
  auto load = [&](uint32_t h) {
    const float* row = src + size_t(min(h, heads - 1)) * HD;
    *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(row + d0);
    *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(row + d0 + 4);
    if constexpr (HALF) {  // (loaded once more: exchanged between lanes they cost 5 % of a turn)
      *reinterpret_cast<float4*>(z) = *reinterpret_cast<const float4*>(row + o0);
      *reinterpret_cast<float4*>(z + 4) = *reinterpret_cast<const float4*>(row + o0 + 4);
    }
  };
  load(h0);
  const double per_token = tid < half ? a.rope.turns[tid] : 0.0;
  float4 gain4{};
  const bool brings = a.q_norm && tid < HD / 2;  // 4 of the gains each
  if (brings) gain4 = *reinterpret_cast<const float4*>((tid < HD / 4 ? a.q_norm : a.k_norm) + 4 * (tid % (HD / 4)));
  const Request r = checked(a.c, raw, tid == 0 && t == 0 && blockIdx.y == 0 ? a.s.err : nullptr);
  if (t >= r.fresh) return;
  if (pos < 0) {
    if (tid == 0 && blockIdx.y == 0) atomicOr(a.s.err, S2HIP_PAGES_ERR_POSITION);
    return;
  }
  const uint32_t slot = r.len - r.fresh + t;
  const uint32_t page = uint32_t(a.p.table[size_t(b) * a.p.width + (slot >> a.p.shift)]);
  const bool there = page < a.p.pages;
  if (!there && tid == 0 && blockIdx.y == 0) atomicOr(a.s.err, S2HIP_PAGES_ERR_PAGE);
  if (tid < HD / 2) {
    const double angle = double(pos) * per_token;
    double sn, cs;
    sincospi(2.0 * (angle - rint(angle)), &sn, &cs);
    turn[tid] = make_double2(cs * a.rope.gain, sn * a.rope.gain);
  }
  if (brings) *reinterpret_cast<float4*>(&gains[0][4 * tid]) = gain4;
  __syncthreads();
  double2 cs[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    cs[i] = turn[HALF ? (second ? d0 - half + i : d0 + i) % (HD / 2) : d0 / 2 + i];
    if (second) cs[i].y = -cs[i].y;  // the second of a pair takes the first's times sin, the first the second's times -sin
  }
  for (uint32_t h = h0; h < heads;) {  // whole rows of LP lanes take part
    const bool value = h >= a.s.H + a.s.G;
    double y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e];
    if (!value) {
      double f = 1.0;
      const float* gain = gains[h < a.s.H ? 0 : 1];
      double w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = HALF ? z[e] : 0.0f;
      if (a.q_norm) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fma(y[e], y[e], ss);
        ss += dpp_f64<DPP_QUAD_XOR1>(ss);
        ss += dpp_f64<DPP_QUAD_XOR2>(ss);
        ss += dpp_f64<DPP_ROW_HALF_MIRROR>(ss);
        if constexpr (LP == 16) ss += dpp_f64<DPP_ROW_MIRROR>(ss);
        f = 1.0 / sqrt(ss * (1.0 / HD) + double(a.s.eps));
        float gs[8], go[8];
        *reinterpret_cast<float4*>(gs) = *reinterpret_cast<const float4*>(gain + d0);
        *reinterpret_cast<float4*>(gs + 4) = *reinterpret_cast<const float4*>(gain + d0 + 4);
        if constexpr (HALF) {
          *reinterpret_cast<float4*>(go) = *reinterpret_cast<const float4*>(gain + o0);
          *reinterpret_cast<float4*>(go + 4) = *reinterpret_cast<const float4*>(gain + o0 + 4);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] *= double(gs[e]);
          if constexpr (HALF) w[e] *= double(go[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < (HALF ? 8 : 4); ++e) {
        // (dims that do not turn go past it: 0 times an infinity beside them is no number)
        if constexpr (HALF) {
          const double r = y[e] * cs[e].x - w[e] * cs[e].y;
          y[e] = (turns ? r : y[e]) * f;
        } else {
          const double p = y[2 * e], q = y[2 * e + 1], r0 = p * cs[e].x - q * cs[e].y, r1 = p * cs[e].y + q * cs[e].x;
          const bool turned = d0 + 2 * e < a.rope.dims;
          y[2 * e] = (turned ? r0 : p) * f;
          y[2 * e + 1] = (turned ? r1 : q) * f;
        }
      }
    }
    const uint32_t now = h;
    h += HPB * gridDim.y;
    load(h);
    if (now < a.s.H) {
      float* dst = a.q_out + ((size_t(b) * a.c.n + t) * a.s.H + now) * HD + d0;
      *reinterpret_cast<float4*>(dst) = make_float4(float(y[0]), float(y[1]), float(y[2]), float(y[3]));
      *reinterpret_cast<float4*>(dst + 4) = make_float4(float(y[4]), float(y[5]), float(y[6]), float(y[7]));
      continue;
    }
    // the group's ends (4 lanes), and whether all are numbers (0 x what is none)
    double most = y[0], least = y[0], zero = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e) most = fmax(most, y[e]);
      if (e) least = fmin(least, y[e]);
      zero = fma(y[e], 0.0, zero);
    }
    most = fmax(most, dpp_f64<DPP_QUAD_XOR1>(most));
    least = fmin(least, dpp_f64<DPP_QUAD_XOR1>(least));
    zero += dpp_f64<DPP_QUAD_XOR1>(zero);
    most = fmax(most, dpp_f64<DPP_QUAD_XOR2>(most));
    least = fmin(least, dpp_f64<DPP_QUAD_XOR2>(least));
    zero += dpp_f64<DPP_QUAD_XOR2>(zero);
    const double big = fmax(most, -least);
    const bool odd = !(zero == 0.0) || big >= 16384.0;
    bool negative = -least > most;  // the largest by size is
    if (__any(most == -least && most != 0.0)) {  // two are, one of either sign: the first of them
      uint32_t first = 1000;  // place in the group, doubled, + 1 of a negative one
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (fabs(y[e]) == big) first = 2 * (8 * (l % 4) + e) + (y[e] < 0.0 ? 1 : 0);
      first = min(first, dpp_u32<DPP_QUAD_XOR1>(first));
      first = min(first, dpp_u32<DPP_QUAD_XOR2>(first));
      if (most == -least) negative = first & 1u;
    }
    const double size = rounded8(big * 0.125), d = negative ? size : -size;
    const double inv = odd || size == 0.0 ? 0.0 : 1.0 / d;
    // y / d is y inv but for 2^-52 of it.  It is at most 8 2^9 / (2^9 - 1), and below 12 where d is a few times 2^-24 and rounded
    // by up to a third (a code of 8 and more is 7 then).  Beside 1.5 2^12 it is taken to a multiple of 2^-40: one that is halfway
    // between whole numbers is so again (no other quotient of a value's 24 bits by 8 comes nearer than 2^-25).  Then to a whole
    // number, ties to even, which stands in the low bits of the sum with 1.5 2^52.
    int code[8];  // less 8
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double near = fma(y[e], inv, 0x1.8p12);
      const int whole = int(uint32_t(uint64_t(__double_as_longlong(near + (0x1.8p52 - 0x1.8p12)))));
      code[e] = odd ? 0 : min(max(whole, -8), 7);
    }
    const float scale = odd ? NAN : float(d);
    const uint32_t g = value ? now - a.s.H - a.s.G : now - a.s.H, j = l / 4;
    float* held = value ? a.v_held : a.k_held;
    if (held) {
      held += ((size_t(b) * a.c.n + t) * a.s.G + g) * HD + d0;
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<float4*>(held + e) = make_float4(scale * float(code[e]), scale * float(code[e + 1]), scale * float(code[e + 2]), scale * float(code[e + 3]));
    }
    if (!there) continue;
    if (odd) atomicOr(a.s.err, S2HIP_PAGES_ERR_RANGE);
    const Chunk<HD> at{a.p.shift};
    uint8_t* part = a.p.pool + (size_t(page) * a.s.G + g) * a.p.chunk;
    const uint32_t s = slot & ((1u << a.p.shift) - 1u);
    if (!value) {
      uint32_t word = 0x88888888u;
#pragma unroll
      for (int e = 0; e < 8; ++e) word += uint32_t(code[e]) << (e / 2 * 4 + e % 2 * 16);
      *reinterpret_cast<uint32_t*>(part + ((s * 4 + l % 4) * (HD / 32) + j) * 4) = word;
      if (l % 4 == 0) *reinterpret_cast<_Float16*>(part + at.ks() + (s * (HD / 32) + j) * 2) = _Float16(scale);
    } else {
      const uint32_t quad = s / 4, one = s % 4;  // (16 u + 4 i = 4 quad)
#pragma unroll
      for (uint32_t m = 0; m < 4; ++m)
        part[at.v() + ((quad * 16 + 4 * (l % 4) + m) * (HD / 32) + j) * 4 + one] = uint8_t(0x88u + uint32_t(code[2 * m]) + (uint32_t(code[2 * m + 1]) << 4));
      if (l % 4 == 0) *reinterpret_cast<_Float16*>(part + at.vs() + ((quad * (HD / 32) + j) * 4 + one) * 2) = _Float16(scale);
    }
  }
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// As for the dense caches: scores in powers of two, a kv head's query rows packed,
// row (b n + t) rep + r, a row's softmax state (m, l, o); f16 parts of queries and
// weights, whose keys and values are f16 numbers as they are.
//   An element is d (c - 8).  Four bits c become the f16 number 16 + c by an or into
// the upper mantissa bits, and one fma with d and -24 d takes them to the element,
// exactly: -24 d has 8 + 2 significant bits, the element 8 + 3.

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ half2v as_half2(uint32_t x) { return __builtin_bit_cast(half2v, x); }
__device__ __forceinline__ half2v both(_Float16 x) { return half2v{x, x}; }

// The mask of the codes and the bits of 16, in registers: as literals they would take an and and an or apart (an
// instruction of three operands has no literal, and one scalar register).
struct Bits {
  uint32_t mask, sixteen;
};
__device__ __forceinline__ Bits code_bits() {
  Bits b{0x03c003c0u, 0x4c004c00u};
  asm("" : "+s"(b.mask));
  asm("" : "+v"(b.sixteen));
  return b;
}
// The two elements whose codes are in bits 4 F .. of a word's halves.
template <int F>
__device__ __forceinline__ half2v elements(Bits bits, uint32_t w, half2v d, half2v c) {
  const uint32_t x = F == 0 ? w << 6 : F == 1 ? w << 2 : F == 2 ? w >> 2 : w >> 6;
  return __builtin_elementwise_fma(as_half2((x & bits.mask) | bits.sixteen), d, c);
}
// A key's eight elements of a word (dims in order).
__device__ __forceinline__ half8 key8(Bits bits, uint32_t w, _Float16 d) {
  const half2v dd = both(d), c = both(d * _Float16(-24.0f));
  const half2v a = elements<0>(bits, w, dd, c), b = elements<1>(bits, w, dd, c), e = elements<2>(bits, w, dd, c), f = elements<3>(bits, w, dd, c);
  return half8{a[0], a[1], b[0], b[1], e[0], e[1], f[0], f[1]};
}
// Weights are 2^(s - m), up to 2^15: m, a whole number, follows LIFT below a row's maximum, by BEHIND at most.  So the largest
// of a row is 2^14 or more, and the lo part of a small one, of whole 2^-24, is exact to 2^-39 of it.  (Where one key weighs e^16
// times as much as any other and its value is 0, the output is the others': with a lift of 6, the maximum up to 2^8 behind, it was
// off by a thousandth.)  o is rescaled more often: lift and slack 14 1 : 11 4 : 6 8, us: 1 x 3999 262.8 : 258.7 : 257.8, 8 x 250
// over 1500 + 250 102.5 : 100.5 : 100.8, 16 x 1 over 32001 116.4 : 116.1 : 115.9.
constexpr float LIFT = 14.0f, BEHIND = 1.0f;

// The m of a maximum.  From 2^25 on f32 has every 4th whole number or fewer, and LIFT less may be 16 less: a weight of 2^16, which
// is no f16 number, so the maximum itself then.
__device__ __forceinline__ float base_of(float most) {
  const float to = floorf(most) - LIFT;
  return most - to > LIFT + BEHIND ? to + 16.0f : to;
}

// Two weights' f16 parts and what those leave of them (f16 too: 2^-22 of the weight, or 2^-25), both in one register each.
struct WeightParts {
  half2v hi, lo;
};
__device__ __forceinline__ WeightParts split_weights(float p, float q) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  WeightParts w;
  w.hi = __builtin_convertvector((float2v{p, q}), half2v);
  uint32_t lo;  // p - hi in f32, rounded once
  asm("v_fma_mixlo_f16 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(lo) : "v"(w.hi), "v"(p));
  asm("v_fma_mixhi_f16 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(lo) : "v"(w.hi), "v"(q));
  w.lo = as_half2(lo);
  return w;
}
// Four tokens' values of two dims (a byte each, dim 2 m below) as pairs of neighbours: v[x]: tokens 0 1 of dim 2 m + x,
// v[2 + x]: tokens 2 3.  d: the tokens' scales.
__device__ __forceinline__ void values8(Bits bits, uint32_t w, u32x2 d, half2v (&v)[4]) {
  w = __builtin_amdgcn_perm(w, w, 0x03010200u);  // bytes 0 2 1 3
  const half2v d0 = as_half2(d[0]), d1 = as_half2(d[1]), c0 = d0 * both(_Float16(-24.0f)), c1 = d1 * both(_Float16(-24.0f));
  v[0] = elements<0>(bits, w, d0, c0);
  v[1] = elements<1>(bits, w, d0, c0);
  v[2] = elements<2>(bits, w, d1, c1);
  v[3] = elements<3>(bits, w, d1, c1);
}
// A scale that append writes is at most 2048 by size.  One beyond that counts as no number where a row must not see it: 24 of
// it is an infinity from 2730 on, and so are its elements, whose product with a weight of 0 is no number.
constexpr uint32_t SCALE_MOST = 0x6800u;  // 2048
__device__ __forceinline__ bool odd_scale(uint32_t half) { return (half & 0x7fffu) > SCALE_MOST; }
__device__ __forceinline__ bool odd_scales(uint32_t pair) { return ((pair & 0x7fff7fffu) + 0x00010001u * (0x7fffu - SCALE_MOST)) & 0x80008000u; }
// Of pair x of scales those of no number become 0; the first of them, or a large number.
template <class Pairs>
__device__ __forceinline__ uint32_t take_odd_scales(Pairs& pairs, int x) {
  uint32_t first = 1000, pair = pairs[x];
#pragma unroll
  for (int i = 1; i >= 0; --i)
    if (odd_scale(pair >> (16 * i))) {
      pair &= ~(0xffffu << (16 * i));
      first = i;
    }
  pairs[x] = pair;
  return first;
}

// Few rows over many keys (decode steps, short turns).  A wave owns RG groups of 16
// packed rows of a kv head and a run of tiles of 32 keys; nothing is exchanged between
// waves before the end, when the block's four join their states in LDS and, with several
// blocks per row tile, leave them for the join kernel.
//   S^T = K Q^T and O^T += V^T P^T by v_mfma_f32_16x16x32_f16, so a lane holds one row
// (lane % 16).  Keys lie in memory as the first product's lanes take them (lane % 16 =
// key, 8 dims of each 32), values as the second's (lane % 16 = pair of dims, 4 tokens
// of each 16, as the weights stand in the registers): both go from memory to operands
// with no exchange.
//   Vector instructions bound it: 4 bits become f16 numbers, and a weight two of them, at one
// issue of four units (16 x 1 over 32001 slots: 105 to 116 us by the card for 450 MB, 3.9 to 4.3 TB/s, vector units 59 %
// busy, matrix units 19 %; its loads alone took 97 on the quickest).  Short runs are latency: of 10 us of 8 x 1
// over 1500 + 512, 2.5 go before the first load of a page (lengths, tables, queries), 1 in it, 1 to
// a tile (a wave alone on its unit issues every fifth cycle), 1 at the end, and 3.5 in the join.
//   The run: first the tiles that all requests of the rows have in common (the same
// pages at the head of their rows of the table, seen by all), read once for all; then
// each request's own.  Page numbers stand one per lane, 64 at a time.
constexpr int STEP_WAVES = 4;

// The tiles of `n_rows` packed rows from row0 on.  Lane j holds request b_lo + j (at most 16 requests).
struct PgRun {
  uint32_t b_lo;
  uint32_t common;    // keys that all have in common, a multiple of 32
  uint32_t tiles;     // of the requests' own keys
  Request rq;         // the lane's request
  uint32_t seg_keys;  // keys that its rows see, at most (0: it has no row)
  uint32_t seg_end;   // its last own tile + 1
};

// The first 64 page numbers of a row tile's first FEW requests, one per lane: loaded before anything is known of the requests.
constexpr int FEW = 4;
struct Pages64 {
  int32_t of[FEW];
};
__device__ __forceinline__ Pages64 load_pages(const PgAttendArgs& pa, uint32_t b_lo) {
  Pages64 p;
  const uint32_t i = min(threadIdx.x & 63u, pa.p.width - 1);
#pragma unroll
  for (int j = 0; j < FEW; ++j) p.of[j] = pa.p.table[size_t(min(b_lo + j, pa.a.c.R - 1)) * pa.p.width + i];
  return p;
}

// Sum over lanes 0 .. l of 16.
__device__ __forceinline__ uint32_t row_scan(uint32_t x) {
  x += dpp_or_0<0x111, 0xF>(x);
  x += dpp_or_0<0x112, 0xF>(x);
  x += dpp_or_0<0x114, 0xF>(x);
  x += dpp_or_0<0x118, 0xF>(x);
  return x;
}

template <int KT>
__device__ __forceinline__ PgRun pg_run(const PgAttendArgs& pa, uint32_t row0, uint32_t n_rows, RawRequest raw, const Pages64& early, uint32_t* err) {
  const KvAttendArgs& a = pa.a;
  const uint32_t lane = threadIdx.x & 63u, per = a.c.n * a.s.rep, row1 = min(row0 + n_rows, a.c.R * per);
  PgRun r{};
  r.b_lo = pa.by_rows(row0);
  const uint32_t b = r.b_lo + lane;
  if (b <= pa.by_rows(row1 - 1)) {
    r.rq = checked(a.c, raw, err);
    const uint32_t first = max(row0, b * per) - b * per, last = min(row1, (b + 1) * per) - 1 - b * per;
    if (pa.by_rep(first) < r.rq.fresh) r.seg_keys = r.rq.len - r.rq.fresh + min(pa.by_rep(last), r.rq.fresh - 1) + 1;
  }
  // what every row with a token sees, as far as the tables agree
  const uint64_t has = __ballot(r.seg_keys != 0);
  if (__popcll(has) > 1) {
    uint32_t least = r.seg_keys ? r.rq.len - r.rq.fresh + 1 : 0xffffffffu;
    least = lane_read_u32(row_reduce(least, [](uint32_t x, uint32_t y) { return min(x, y); }), 0);
    const uint32_t pages = least >> pa.p.shift;
    uint32_t same = 0;
    for (; same < pages;) {
      const uint32_t i = min(same + lane, pages - 1);  // (of the first pages, lane i's: what is behind is looked at twice or not)
      int32_t first = 0;
      bool differs = false, led = false;
      auto look = [&](int32_t page) {
        differs |= led && page != first;
        if (!led) first = page;
        led = true;
      };
      if (same == 0) {
#pragma unroll
        for (int j = 0; j < FEW; ++j)
          if ((has >> j) & 1u) look(early.of[j]);
        for (uint64_t rest = has >> FEW << FEW; rest; rest &= rest - 1)
          look(pa.p.table[size_t(r.b_lo + uint32_t(__ffsll((unsigned long long)rest)) - 1) * pa.p.width + min(lane, pa.p.width - 1)]);
        differs = differs && lane < pages;
      } else {
        for (uint64_t rest = has; rest; rest &= rest - 1)
          look(pa.p.table[size_t(r.b_lo + uint32_t(__ffsll((unsigned long long)rest)) - 1) * pa.p.width + i]);
      }
      const uint64_t out = __ballot(differs);
      if (out) {
        same += uint32_t(__ffsll((unsigned long long)out)) - 1;
        break;
      }
      same = min(same + 64, pages);
    }
    r.common = (same << pa.p.shift) / KT * KT;
  }
  r.seg_end = row_scan(r.seg_keys > r.common ? (r.seg_keys - r.common + KT - 1) / KT : 0u);
  r.tiles = lane_read_u32(r.seg_end, 15);
  return r;
}
// The request of own tile x, less b_lo: how many end before it.
__device__ __forceinline__ uint32_t owner(const PgRun& r, uint32_t x) {
  return min(15u, uint32_t(__popcll(__ballot(r.seg_end <= x) & 0xffffu)));
}

__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t x = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const uint8_t*>(uint64_t(uniform(uint32_t(x >> 32))) << 32 | uniform(uint32_t(x)));
}

// 64 page numbers of a request, one per lane.
struct PageWindow {
  uint32_t b = 0xffffffffu, first = 0;
  int32_t page = 0;
  __device__ __forceinline__ void load(const PgPool& p, uint32_t req, uint32_t i) {
    b = req;
    first = i;
    page = p.table[size_t(req) * p.width + min(i + (threadIdx.x & 63u), p.width - 1)];
  }
  __device__ __forceinline__ void begin(const Pages64& early, uint32_t b_lo, uint32_t req) {  // (where req is one of the few)
    if (req - b_lo >= uint32_t(FEW)) return;
    b = req;
#pragma unroll
    for (int j = 0; j < FEW; ++j)
      if (req - b_lo == uint32_t(j)) page = early.of[j];
  }
  __device__ __forceinline__ uint32_t get(const PgPool& p, uint32_t req, uint32_t i) {
    if (req != b || i - first >= 64u) load(p, req, i);
    return lane_read_u32(uint32_t(page), int(i - first));
  }
};

// The blocks of a kv head, `blocks` of them, and its states [kv heads][blocks][1 << shift rows] (of the tile kernel, whose
// splits are the same for all: each 16 rows' as if a block did no more).
struct PgShare {
  float* o;
  float* ml;
  uint2* ranges;  // [row tiles]: first block and number of them; NULL: each
  uint32_t tiles, blocks, each;
  Div by_each;
  uint32_t row_tiles, of_request;  // the kernel's row tiles; those of a request, where none has rows of two (0: they may)
  Div by_of;
  uint32_t shift;
};
// The row tile of block x, its first block and how many it has: one at least, and the rest by the keys in its
// requests' caches, so that no block has much more than another.
struct Share {
  uint32_t tile, first, count;
};
template <int ROWS>
__device__ __forceinline__ Share share_of(const PgAttendArgs& pa, const PgShare& sp, uint32_t x) {
  if (!sp.ranges) {
    const uint32_t tile = sp.by_each(x);
    return {tile, tile * sp.each, sp.each};
  }
  const KvAttendArgs& a = pa.a;
  const uint32_t lane = threadIdx.x & 63u;  // (at most 64 row tiles)
  uint32_t keys = 0;
  if (lane < sp.tiles)
    for (uint32_t b = sp.of_request ? sp.by_of(lane) : pa.by_rows(lane * ROWS), end = sp.of_request ? b : min(pa.by_rows((lane + 1) * ROWS - 1), a.c.R - 1); b <= end; ++b) {
      const int32_t len = a.c.lens[b];
      keys += len > 0 && len <= int32_t(a.c.cap) ? uint32_t(len) / 32 + 1 : 0u;
    }
  const uint32_t upto = wave_scan(keys), all = max(1u, lane_read_u32(upto, 63));
  const uint32_t first = lane < sp.tiles ? lane + uint32_t(uint64_t(sp.blocks - sp.tiles) * (upto - keys) / all) : sp.blocks;
  const uint32_t tile = uint32_t(__popcll(__ballot(first <= x))) - 1;  // (first goes up with the lane)
  const uint32_t begin = lane_read_u32(first, int(tile)), end = tile == 63 ? sp.blocks : lane_read_u32(first, int(tile) + 1);
  return {tile, begin, end - begin};
}

// A tile of 32 keys in halves of 16, which lie in one page or (TWO) may lie in two.
template <bool TWO>
struct PgTile {
  uint32_t req, key0, keys;      // request, first key; keys of it that are there
  uint32_t left, seg_keys;       // further tiles of the same request (or in common), and its keys
  int seg;                       // -1: in common; else request b_lo + seg
  const uint8_t* part[1 + TWO];  // the kv head's part of the page
  uint32_t slot[1 + TWO];        // the first slot there
  uint32_t gone;                 // bit h: half h lies in no page of the pool
};

template <int HD, bool TWO, int RG>
__global__ __launch_bounds__(64 * STEP_WAVES, RG == 1 ? 3 : 2) void pg_step_kernel(PgAttendArgs pa, PgShare sp) {
  constexpr int ROWS = 16 * RG, KT = 32, OT = HD / 16, GR = HD / 32;  // key tile, 16 x 16 output tiles, scales of a head
  constexpr int OP = HD + 4;                          // padded row of the joined states
  // A tile: key codes, value codes, key scales, value scales (and what the load of those leaves behind them); a wave's two, and in their place its
  // state in the end.
  constexpr uint32_t TILE = KT * HD + 1024, STAGE = 2 * TILE, K_AT = 0, V_AT = KT * HD / 2, KS_AT = KT * HD, VS_AT = KT * (HD + HD / 16);
  constexpr int LOADS = HD == 128 ? 5 : 3;
  static_assert(16 * OP * 4 <= STAGE, "a state fits");
  __shared__ __align__(16) uint8_t lds[STEP_WAVES * STAGE];
  __shared__ float ml[STEP_WAVES][ROWS][2];
  const KvAttendArgs& a = pa.a;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), r16 = lane & 15u, q4 = lane >> 4;
  const uint32_t block = pa.by_groups(blockIdx.x), g = blockIdx.x - block * a.s.G;
  const Share share = share_of<ROWS>(pa, sp, block);
  const uint32_t tile = share.tile, split = block - share.first;
  const uint32_t per = a.c.n * a.s.rep, whose = sp.by_of(tile), row0 = sp.of_request ? whose * per + (tile - whose * sp.of_request) * ROWS : tile * ROWS;
  const uint32_t n_rows = min(uint32_t(ROWS), (sp.of_request ? whose + 1 : a.c.R) * per - row0);
  const Chunk<HD> at{pa.p.shift};
  const Bits bits = code_bits();

  const RawRequest raw = load_request(a.c, min(pa.by_rows(row0) + lane, a.c.R - 1));
  const Pages64 early = load_pages(pa, pa.by_rows(row0));
  uint32_t b_row[RG], t_row[RG];
  float4 qx[RG][HD / 16];  // dims 32 (j / 2) + 8 q4 + 4 (j % 2) ..
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    const uint32_t row = row0 + min(16 * r + r16, n_rows - 1);
    b_row[r] = pa.by_rows(row);
    t_row[r] = pa.by_rep(row - b_row[r] * per);
    const uint32_t h_row = g * a.s.rep + row - (b_row[r] * a.c.n + t_row[r]) * a.s.rep;
    const size_t q_at = ((size_t(b_row[r]) * a.c.n + t_row[r]) * a.s.H + h_row) * HD;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) qx[r][j] = *reinterpret_cast<const float4*>(a.q + q_at + 32 * (j / 2) + 8 * q4 + 4 * (j % 2));
  }
  const PgRun run = pg_run<KT>(pa, row0, n_rows, raw, early, g == 0 && split == 0 && wave == 0 ? a.s.err : nullptr);
  const uint32_t b_lo = run.b_lo, lots = share.count * STEP_WAVES, lot = split * STEP_WAVES + wave;
  const uint32_t c_tiles = run.common / KT, c_lo = c_tiles * lot / lots, n_com = c_tiles * (lot + 1) / lots - c_lo;
  // (the own tiles the other way round: the waves with one more in common get one fewer)
  const uint32_t o_lo = run.tiles * (lots - 1 - lot) / lots, n_tiles = n_com + run.tiles * (lots - lot) / lots - o_lo;

  uint32_t seg = 0;
  const uint32_t lead = uint32_t(__ffsll((unsigned long long)__ballot(run.seg_keys != 0))) - 1;  // (with the others' pages in common)
  PageWindow window;
  if (n_com == 0) seg = owner(run, o_lo);
  window.begin(early, b_lo, b_lo + (n_com ? lead : seg));
  using Tile = PgTile<TWO>;
  auto turn_page = [&](Tile& w) {
    w.gone = 0;
#pragma unroll
    for (int h = 0; h < 1 + TWO; ++h) {
      const uint32_t key = w.key0 + (h && w.keys > 16 ? 16 : 0);
      const uint32_t page = window.get(pa.p, w.req, key >> pa.p.shift);
      const bool in = page < pa.p.pages;
      w.gone |= in ? 0u : TWO ? 1u << h : 3u;
      w.part[h] = pa.p.pool + (size_t(in ? page : 0u) * a.s.G + g) * pa.p.chunk;
      w.slot[h] = key & ((1u << pa.p.shift) - 1u);
    }
    if (w.gone && lane == 0) atomicOr(a.s.err, S2HIP_PAGES_ERR_PAGE);
  };
  auto where = [&](uint32_t i) {
    Tile w;
    if (i < n_com) {
      w.seg = -1;
      w.req = b_lo + lead;
      w.key0 = (c_lo + i) * KT;
      w.left = n_com - 1 - i;
      w.seg_keys = run.common;
    } else {
      const uint32_t x = o_lo + (i - n_com);
      seg = owner(run, x);
      const uint32_t begin = seg ? lane_read_u32(run.seg_end, int(seg) - 1) : 0u;
      w.seg = int(seg);
      w.req = b_lo + seg;
      w.key0 = run.common + (x - begin) * KT;
      w.left = lane_read_u32(run.seg_end, int(seg)) - 1 - x;
      w.seg_keys = lane_read_u32(run.seg_keys, int(seg));
    }
    w.keys = min(uint32_t(KT), w.seg_keys - w.key0);
    turn_page(w);
    return w;
  };
  // the tile behind w, the i-th
  auto behind = [&](const Tile& was, uint32_t i) {
    if (was.left == 0) return where(i);
    Tile w = was;
    --w.left;
    w.key0 += KT;
    w.keys = min(uint32_t(KT), w.seg_keys - w.key0);
    w.slot[0] += KT;
    if (TWO || w.slot[0] >> pa.p.shift) turn_page(w);
    return w;
  };
  // Tiles go straight to LDS, two ahead of their use: in registers one more tile would cost a fourth wave per SIMD.
  lds_byte* const stage = (lds_byte*)lds + wave * STAGE;
  const uint32_t stage_at = uint32_t(uintptr_t(stage));
  const uint32_t k_lane = r16 * (HD / 2) + q4 * 16, s_lane = (lane & 16u ? at.vs() - at.ks() : 0u) + r16 * 16;
  auto fetch = [&](const Tile& w, uint32_t slot) {
    const uint32_t to = uniform(stage_at + slot * TILE);
    if constexpr (!TWO) {
      const uint8_t* part = uniform(w.part[0]);
      const uint32_t first = uniform(w.slot[0]);
      const uint8_t *k = part + first * (HD / 2), *v = k + at.v(), *d = part + at.ks() + first * (HD / 16);
      if constexpr (HD == 128) {
        dma16(k, k_lane, to + K_AT);
        dma16(k, k_lane + 1024, to + K_AT + 1024);
        dma16(v, lane * 16, to + V_AT);
        dma16(v, lane * 16 + 1024, to + V_AT + 1024);
        dma16(d, s_lane, to + KS_AT);  // 16 lanes each: key scales, value scales, and both again behind the tile
      } else {
        dma16(k, lane * 16, to + K_AT);
        dma16(v, lane * 16, to + V_AT);
        dma16(d, (lane & 8u ? at.vs() - at.ks() : 0u) + (lane & 7u) * 16, to + KS_AT);  // 8 lanes each
      }
    } else {
      const bool second = lane >= 32;
      const uint8_t* mine = second ? w.part[TWO] : w.part[0];
      const uint32_t at_slot = second ? w.slot[TWO] : w.slot[0], l32 = lane & 31u;
      if constexpr (HD == 128) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          dma16(w.part[h] + w.slot[h] * (HD / 2), k_lane, to + K_AT + 1024 * h);
          dma16(w.part[h] + at.v() + w.slot[h] * (HD / 2), lane * 16, to + V_AT + 1024 * h);
        }
      } else {
        dma_lane<16>(mine + at_slot * (HD / 2) + l32 * 16, to + K_AT);
        dma_lane<16>(mine + at.v() + at_slot * (HD / 2) + l32 * 16, to + V_AT);
      }
      // pieces of 16 bytes: key scales of both halves, value scales of both, and all again
      constexpr uint32_t PH = HD / 16;  // of a half
      const uint32_t piece = lane % (4 * PH);
      const bool odd = (piece / PH) & 1u;
      const uint8_t* from = odd ? w.part[TWO] : w.part[0];
      dma_lane<16>(from + (piece >= 2 * PH ? at.vs() : at.ks()) + (odd ? w.slot[TWO] : w.slot[0]) * (HD / 16) + piece % PH * 16, to + KS_AT);
    }
  };
  // codes of key r16, dims 32 j + 8 q4 ..; its scales; codes of dims 32 j + 2 r16 .. of tokens 4 q4 ..; their scales
  typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
  typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
  typedef __attribute__((address_space(3))) uint32_t lds_u32;
  uint32_t kc[2][GR], ks[2][GR / 2];
  auto take_k = [&](uint32_t slot) {
    lds_byte* p = stage + slot * TILE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (HD == 128) {
        *reinterpret_cast<u32x4*>(kc[h]) = *reinterpret_cast<lds_u32x4*>(p + K_AT + 1024 * h + lane * 16);
        *reinterpret_cast<u32x2*>(ks[h]) = *reinterpret_cast<lds_u32x2*>(p + KS_AT + 128 * h + r16 * 8);
      } else {
        *reinterpret_cast<u32x2*>(kc[h]) = *reinterpret_cast<lds_u32x2*>(p + K_AT + 512 * h + r16 * 32 + q4 * 8);
        ks[h][0] = *reinterpret_cast<lds_u32*>(p + KS_AT + 64 * h + r16 * 4);
      }
    }
  };
  Tile w{}, next{};
  if (n_tiles) {
    w = where(0);
    fetch(w, 0);
  }
  if (n_tiles > 1) {
    next = behind(w, 1);
    fetch(next, 1);
  }

  // this lane's rows
  int own_limit[RG], own_seg[RG];
  half8 qh[RG][GR], ql[RG][GR];  // dims 32 j + 8 q4 + e
  float unscale[RG];
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    const int mine = int(b_row[r] - b_lo);
    const uint32_t len_row = __shfl(run.rq.len, mine & 15, 64), fresh_row = __shfl(run.rq.fresh, mine & 15, 64);
    const bool live = 16 * r + r16 < n_rows && t_row[r] < fresh_row;
    // (a row of no token may see anything: nobody reads it)
    own_limit[r] = live ? int(len_row - fresh_row + t_row[r]) : 0x7fffffff;
    own_seg[r] = live ? mine : -2;
    const float s2 = live ? a.s.scale2 : 0.0f;
    float x[HD / 16][4], big = 0.0f;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) {
      x[j][0] = live ? qx[r][j].x * s2 : 0.0f;  // (a query of no token may hold anything)
      x[j][1] = live ? qx[r][j].y * s2 : 0.0f;
      x[j][2] = live ? qx[r][j].z * s2 : 0.0f;
      x[j][3] = live ? qx[r][j].w * s2 : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(x[j][e]));
    }
    float inv;
    pow2_scale(quarter_max(big), unscale[r], inv);
#pragma unroll
    for (int j = 0; j < GR; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Parts y = split_query<false>(x[2 * j + e / 4][e % 4] * inv);
        qh[r][j][e] = y.hi;
        ql[r][j][e] = y.lo;
      }
  }

  floatx4 o[RG][OT];  // o[][2 c + h][i]: dim 32 c + 8 q4 + 2 i + h
  float m[RG], l[RG];
#pragma unroll
  for (int r = 0; r < RG; ++r) {
#pragma unroll
    for (int i = 0; i < OT; ++i) o[r][i] = floatx4{0.f, 0.f, 0.f, 0.f};
    m[r] = -INFINITY;
    l[r] = 0.0f;
  }

  for (uint32_t i = 0; i < n_tiles; ++i) {
    const uint32_t slot = i & 1u;
    if (i + 1 < n_tiles)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");  // (all but the next tile's)
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    bool mine[RG], sees = true, fits = true;
    int limit[RG];
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      mine[r] = w.seg < 0 || own_seg[r] == -2 || own_seg[r] == w.seg;
      limit[r] = w.seg < 0 || own_seg[r] == -2 ? 0x7fffffff : mine[r] ? own_limit[r] : -1;
      sees = sees && limit[r] >= int(w.key0 + KT - 1);
      fits = fits && (!mine[r] || limit[r] >= int(w.key0 + KT - 1));
    }
    const bool all_see = __all(sees) && !w.gone;  // every row, the whole tile: nothing to keep off
    bool masks = false;
    if (!all_see) {
      // A pair of scales per lane: keys' of dims .., values' of tokens 16 h + 4 i + 2 x and the next.
      constexpr uint32_t PAIRS = 16 * GR;
      lds_u32* const kp = reinterpret_cast<lds_u32*>(stage + slot * TILE + KS_AT) + lane % PAIRS;
      lds_u32* const vp = reinterpret_cast<lds_u32*>(stage + slot * TILE + VS_AT) + lane % PAIRS;
      const uint32_t quad = lane % PAIRS / (2 * GR), first_token = 4 * quad + 2 * (lane & 1u);
      uint32_t pair = *vp;
      if (w.keys < KT || w.gone) {  // scales of tokens that no row sees may hold anything: 0
        const int there = (w.gone >> (quad / 4)) & 1u ? 0 : int(w.keys) - int(first_token);
        pair &= there >= 2 ? 0xffffffffu : there == 1 ? 0xffffu : 0u;
        *vp = pair;
      }
      // Where the rows of its request see all of it and its keys are numbers, the other rows' weights are 0 by their bias.
      masks = w.gone || !__all(fits && !odd_scales(*kp));
      if (__any(odd_scales(pair))) {  // values of no number: 0 too; outputs of rows that see the first of them are no number
        const uint32_t at_token = odd_scale(pair) ? first_token : odd_scales(pair) ? first_token + 1 : 1000u;
        if (odd_scale(pair)) pair &= 0xffff0000u;
        if (odd_scale(pair >> 16)) pair &= 0xffffu;
        *vp = pair;
#pragma unroll
        for (int c = 0; c < GR; ++c) {
          const uint32_t first = wave_reduce(int(lane / 2 % GR) == c ? at_token : 1000u, [](uint32_t x, uint32_t y) { return min(x, y); });
#pragma unroll
          for (int r = 0; r < RG; ++r)
            if (first < KT && limit[r] >= int(w.key0 + first)) o[r][2 * c] = o[r][2 * c + 1] = floatx4{NAN, NAN, NAN, NAN};
        }
      }
      asm volatile("" ::: "memory");  // (what is read below in other types is what was written here)
    }
    take_k(slot);
    floatx4 s[RG][2] = {};
#pragma unroll
    for (int j = 0; j < GR; ++j) {
      half8 k8[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        k8[h] = key8(bits, kc[h][j], as_half2(ks[h][j / 2])[j % 2]);
#pragma unroll
        for (int r = 0; r < RG; ++r) s[r][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[h], ql[r][j], s[r][h], 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < RG; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) s[r][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[h], qh[r][j], s[r][h], 0, 0, 0);
    }
    if (masks) {
      asm volatile("");
#pragma unroll
      for (int r = 0; r < RG; ++r)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int key = int(w.key0 + 16u * (c / 4) + 4u * q4 + (c % 4));
          if (key > limit[r] || ((w.gone >> (c / 4)) & 1u)) s[r][c / 4][c % 4] = -INFINITY;
        }
    }
    half8 ph[RG], pl[RG];  // the lane's four tokens of each half
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      float top = fmaxf(fmaxf(s[r][0][0], s[r][0][1]), s[r][0][2]), top1 = fmaxf(fmaxf(s[r][1][0], s[r][1][1]), s[r][1][2]);
      top = fmaxf(fmaxf(top, s[r][0][3]), fmaxf(top1, s[r][1][3]));
      const float mn = mine[r] ? fmaxf(m[r], quarter_max(top) * unscale[r]) : m[r];
      const bool up = mn - m[r] > LIFT + BEHIND;
      if (__any(up)) {
        const float to = up ? base_of(mn) : m[r], f = up ? __builtin_amdgcn_exp2f(m[r] - to) : 1.0f;
#pragma unroll
        for (int c = 0; c < OT; ++c) o[r][c] *= f;
        l[r] *= f;
        m[r] = to;
      }
      // (a weight of a row that is not of the request: 2^-infinity)
      const float bias = mine[r] ? (m[r] == -INFINITY ? 0.0f : -m[r]) : -INFINITY;
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int v = 2 * (i % 2);
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r][i / 2][v], unscale[r], bias)), q = __builtin_amdgcn_exp2f(fmaf(s[r][i / 2][v + 1], unscale[r], bias));
        sum[0] += p;
        sum[1] += q;
        const WeightParts w2 = split_weights(p, q);
        ph[r][2 * i] = w2.hi[0];
        ph[r][2 * i + 1] = w2.hi[1];
        pl[r][2 * i] = w2.lo[0];
        pl[r][2 * i + 1] = w2.lo[1];
      }
      l[r] += sum[0] + sum[1];
    }
    lds_byte* const values = stage + slot * TILE;
#pragma unroll
    for (int half_c = 0; half_c < GR / 2; ++half_c) {  // two groups of 32 dims
      uint32_t vc[2][2];
      u32x2 vs[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (HD == 128)
          *reinterpret_cast<u32x2*>(vc[h]) = *reinterpret_cast<lds_u32x2*>(values + V_AT + 1024 * h + lane * 16 + 8 * half_c);
        else
          *reinterpret_cast<u32x2*>(vc[h]) = *reinterpret_cast<lds_u32x2*>(values + V_AT + 512 * h + lane * 8);
        *reinterpret_cast<u32x4*>(vs[h]) = *reinterpret_cast<lds_u32x4*>(values + VS_AT + HD * h + q4 * (HD / 4) + 16 * half_c);
      }
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const int c = 2 * half_c + cc;
        half2v v[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) values8(bits, vc[h][cc], vs[h][cc], v[h]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const half8 v8 = {v[0][x][0], v[0][x][1], v[0][2 + x][0], v[0][2 + x][1], v[1][x][0], v[1][x][1], v[1][2 + x][0], v[1][2 + x][1]};
#pragma unroll
          for (int r = 0; r < RG; ++r) {
            o[r][2 * c + x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, ph[r], o[r][2 * c + x], 0, 0, 0);
            o[r][2 * c + x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, pl[r], o[r][2 * c + x], 0, 0, 0);
          }
        }
      }
    }
    w = next;
    if (i + 2 < n_tiles) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the tile is in registers)
      next = behind(next, i + 2);
      fetch(next, slot);
    }
  }

  // the block's four states as one, 16 rows at a time
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    l[r] = quarter_sum(l[r]);
    if (q4 == 0) {
      ml[wave][16 * r + r16][0] = m[r];
      ml[wave][16 * r + r16][1] = l[r];
    }
  }
  const bool last = sp.blocks == sp.tiles;
  if (sp.ranges && g == 0 && split == 0 && tid == 0) sp.ranges[tile] = make_uint2(share.first, share.count);
  const uint32_t jr = tid / 16, d0 = tid % 16 * 4;  // a row per 16 threads
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < STEP_WAVES; ++i) M = fmaxf(M, ml[i][16 * r + r16][0]);
    const float f = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[r] - M);
    float* os = reinterpret_cast<float*>(lds + wave * STAGE) + r16 * OP;
#pragma unroll
    for (int c = 0; c < GR; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        *reinterpret_cast<floatx4*>(os + 32 * c + 8 * q4 + 4 * x) =
            floatx4{o[r][2 * c][2 * x] * f, o[r][2 * c + 1][2 * x] * f, o[r][2 * c][2 * x + 1] * f, o[r][2 * c + 1][2 * x + 1] * f};
    __syncthreads();
    float M_row = -INFINITY, L_row = 0.0f;
#pragma unroll
    for (int i = 0; i < STEP_WAVES; ++i) M_row = fmaxf(M_row, ml[i][16 * r + jr][0]);
    const float M_base = M_row == -INFINITY ? 0.0f : M_row;  // (then every l is 0, or no number)
#pragma unroll
    for (int i = 0; i < STEP_WAVES; ++i) L_row = fmaf(ml[i][16 * r + jr][1], __builtin_amdgcn_exp2f(ml[i][16 * r + jr][0] - M_base), L_row);
    const size_t part = (size_t(g) * sp.blocks + block) * ROWS + 16 * r + jr;
    const uint32_t out_row = row0 + 16 * r + jr, ob = pa.by_rows(out_row), ot = pa.by_rep(out_row - ob * per), oh = g * a.s.rep + out_row - (ob * a.c.n + ot) * a.s.rep;
    const bool out_live = 16 * r + jr < n_rows && ot < __shfl(run.rq.fresh, int(ob - b_lo) & 15, 64);
    if (!last || out_live) {
      float* dst = last ? a.out + ((size_t(ob) * a.c.n + ot) * a.s.H + oh) * HD : sp.o + part * HD;
      const float inv = last ? (M_row == -INFINITY ? NAN : 1.0f / L_row) : 1.0f;  // (it sees a key, its own)
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const float* src = reinterpret_cast<const float*>(lds) + jr * OP + d0 + 64 * c;
        floatx4 x = *reinterpret_cast<const floatx4*>(src);
#pragma unroll
        for (int i = 1; i < STEP_WAVES; ++i) x += *reinterpret_cast<const floatx4*>(src + i * (STAGE / 4));
        *reinterpret_cast<floatx4*>(dst + d0 + 64 * c) = x * inv;
      }
      if (tid % 16 == 0 && !last) {
        sp.ml[2 * part] = M_row;
        sp.ml[2 * part + 1] = L_row;
      }
    }
  }
}

// Many rows (turns, prompts).  A block of four waves owns up to 128 rows of a request and kv
// head, 32 per wave, and walks the run of tiles of 64 keys.  Each wave takes 16 of a
// tile's keys and values from 4 bits to f16, once for the block, and leaves them in
// LDS, the next tile's while this one's products run; codes are loaded another tile
// ahead.
//   Its products bound it (two for a term: hi and lo): a prompt of 3999 takes 255 to 263 us by the card,
// the products alone, at the rate that the card's power allows, 226; matrix units 48 % busy by cycles, vector units 46.
// Of 8 x 250 tokens over 1500 + 250 (100 us) 380 blocks have rows: a second one on half of the CUs.
//   v_mfma_f32_32x32x16_f16, S^T = K Q^T and O^T += V^T P^T, a lane holds one row
// (lane % 32).  Values stand transposed, a row of 64 tokens per dim, each 16 bytes the
// 8 tokens that a lane's 8 weights belong to.
constexpr int TILE_ROWS = 128;

template <int HD>
__global__ __launch_bounds__(256, 2) void pg_tile_kernel(PgAttendArgs pa, PgShare sp) {
  constexpr int KT = 64, GR = HD / 32, DS = HD / 16, DT = HD / 32;
  constexpr uint32_t RB = HD * 2, PLANE = KT * RB, BUF = 2 * PLANE;  // bytes of a key's row, of the keys (and of the values), of both
  __shared__ __align__(16) uint8_t lds[2 * BUF];
  // of tiles i, i + 1 and the one behind: bit w: the 16 keys of wave w lie in no page, bit 8: there are values of no number; a
  // group's first
  __shared__ uint32_t gone_tile[3], odd_tile[3][GR];
  const KvAttendArgs& a = pa.a;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), r32 = lane & 31u, h2 = lane >> 5, r16 = lane & 15u, q4 = lane >> 4;
  const uint32_t rest = pa.by_groups(blockIdx.x), g = blockIdx.x - rest * a.s.G;
  const uint32_t split = rest / sp.row_tiles, tile = sp.row_tiles - 1 - (rest - split * sp.row_tiles);  // later rows see more keys: they go first
  const uint32_t splits = sp.each, per = a.c.n * a.s.rep, whose = sp.by_of(tile), row0 = whose * per + (tile - whose * sp.of_request) * TILE_ROWS;
  const uint32_t rows = (whose + 1) * per, n_rows = min(uint32_t(TILE_ROWS), rows - row0);
  const Chunk<HD> at{pa.p.shift};
  const Bits bits = code_bits();

  const RawRequest raw = load_request(a.c, whose);
  PageWindow window;
  window.load(pa.p, whose, 0);
  const uint32_t my_row = row0 + wave * 32 + r32, row = min(my_row, rows - 1);
  const uint32_t t_row = pa.by_rep(row - whose * per), h_row = g * a.s.rep + row - (whose * a.c.n + t_row) * a.s.rep;
  const size_t at_row = (size_t(whose) * a.c.n + t_row) * a.s.H + h_row;
  float4 qx[DS][2];  // dims 16 ks + 8 h2 ..
#pragma unroll
  for (int ks = 0; ks < DS; ++ks)
#pragma unroll
    for (int e = 0; e < 2; ++e) qx[ks][e] = *reinterpret_cast<const float4*>(a.q + at_row * HD + 16 * ks + 8 * h2 + 4 * e);
  const Request rq = checked(a.c, raw, g == 0 && split == 0 && tid == 0 ? a.s.err : nullptr);
  const uint32_t first_token = pa.by_rep(row0 - whose * per), last_token = pa.by_rep(row0 - whose * per + n_rows - 1);
  if (first_token >= rq.fresh) return;  // no row of a token
  const uint32_t seen = uniform(rq.len - rq.fresh + min(last_token, rq.fresh - 1) + 1);  // keys that its rows see, at most
  const uint32_t all = (seen + KT - 1) / KT, lo = all * split / splits, n_tiles = all * (split + 1) / splits - lo;

  // a tile, and where the wave's 16 keys of it are
  struct Tile {
    uint32_t key0, keys;
    const uint8_t* part;
    uint32_t slot;
    bool gone;
  };
  auto where = [&](uint32_t i) {
    Tile w;
    w.key0 = (lo + i) * KT;
    w.keys = min(uint32_t(KT), seen - w.key0);
    const uint32_t key = w.key0 + (16 * wave < w.keys ? 16 * wave : 0u);
    const uint32_t page = window.get(pa.p, whose, key >> pa.p.shift);
    w.gone = page >= pa.p.pages;
    w.part = pa.p.pool + (size_t(w.gone ? 0u : page) * a.s.G + g) * pa.p.chunk;
    w.slot = key & ((1u << pa.p.shift) - 1u);
    if (w.gone && lane == 0) atomicOr(a.s.err, S2HIP_PAGES_ERR_PAGE);
    return w;
  };
  // codes of key lane / 4, dims 32 j + 8 (lane % 4) ..; its scales; codes of dims 32 j + 2 r16 .. of tokens 4 q4 ..; their scales
  uint32_t kc[GR], vc[GR], ks[GR / 2];
  u32x2 vs[GR];
  auto load = [&](const Tile& w) {
    const uint8_t *k = w.part + w.slot * (HD / 2) + lane * (HD / 8), *d = w.part + at.ks() + w.slot * (HD / 16) + lane / 4 * (HD / 16);
    const uint8_t *v = w.part + at.v() + w.slot * (HD / 2) + lane * (HD / 8), *e = w.part + at.vs() + w.slot * (HD / 16) + q4 * (HD / 4);
    if constexpr (HD == 128) {
      *reinterpret_cast<u32x4*>(kc) = *reinterpret_cast<const u32x4*>(k);
      *reinterpret_cast<u32x2*>(ks) = *reinterpret_cast<const u32x2*>(d);
      *reinterpret_cast<u32x4*>(vc) = *reinterpret_cast<const u32x4*>(v);
      *reinterpret_cast<u32x4*>(&vs[0]) = *reinterpret_cast<const u32x4*>(e);
      *reinterpret_cast<u32x4*>(&vs[2]) = *reinterpret_cast<const u32x4*>(e + 16);
    } else {
      *reinterpret_cast<u32x2*>(kc) = *reinterpret_cast<const u32x2*>(k);
      ks[0] = *reinterpret_cast<const uint32_t*>(d);
      *reinterpret_cast<u32x2*>(vc) = *reinterpret_cast<const u32x2*>(v);
      *reinterpret_cast<u32x4*>(&vs[0]) = *reinterpret_cast<const u32x4*>(e);
    }
  };
  // 16-byte piece p of key's row stands at p ^ k_swz(key), piece p of a dim's row of values at p ^ (dim / 2 % 8): 16 lanes'
  // reads of one piece (16 keys, or dims) and 16 lanes' writes (4 keys x 4 pieces; 16 pairs of dims: half as many) are apart.
  // A lane's addresses differ by an exclusive or with constants; they are worked out where they are used, for kept ones cost
  // registers.
  auto k_at = [](uint32_t key, uint32_t piece) {
    const uint32_t swz = HD == 128 ? 4 * (key & 3u) + ((key >> 2) & 3u) : 4 * ((key >> 1) & 1u) + ((key >> 2) & 3u);
    return key * RB + ((piece ^ swz) << 4);
  };
  auto v_at = [](uint32_t dim, uint32_t piece) { return PLANE + dim * (KT * 2) + ((piece ^ ((dim >> 1) & 7u)) << 4); };
  lds_byte* const lds0 = (lds_byte*)lds;
  typedef __attribute__((address_space(3))) half4 lds_half4;
  // The wave's 16 keys and values from registers to LDS, in pieces: 0 .. GR - 1 a key's words, from GR on a group of the
  // values, before which their scales are looked over.
  uint32_t k_to = 0, v_to = 0;
  auto store_begin = [&](uint32_t buf) {
    k_to = buf * BUF + k_at(16 * wave + lane / 4, lane % 4);
    v_to = buf * BUF + v_at(2 * r16, 2 * wave + (q4 & 1u)) + 8 * (q4 >> 1);
    asm volatile("" : "+v"(k_to), "+v"(v_to));
  };
  auto store_key = [&](int j) { *reinterpret_cast<lds_half8*>(lds0 + (k_to ^ (64u * j))) = key8(bits, kc[j], as_half2(ks[j / 2])[j % 2]); };
  auto store_scales = [&](const Tile& w, uint32_t flag) {
    if (w.gone || w.keys < KT) {  // scales of tokens that are not there may hold anything: 0
      asm volatile("");
      const int there = w.gone ? 0 : int(w.keys) - int(16u * wave + 4u * q4);  // of the lane's four
      const uint32_t low = there >= 2 ? 0xffffffffu : there == 1 ? 0xffffu : 0u, high = there >= 4 ? 0xffffffffu : there == 3 ? 0xffffu : 0u;
#pragma unroll
      for (int c = 0; c < GR; ++c) vs[c] = u32x2{vs[c][0] & low, vs[c][1] & high};
    }
    float z = 0.0f;  // (their squares' sum: none is beyond 2048 where it is not beyond 2048^2, and most are far below)
#pragma unroll
    for (int c = 0; c < GR; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) z = __builtin_amdgcn_fdot2(as_half2(vs[c][x]), as_half2(vs[c][x]), z, false);
    if (__any(!(z <= 0x1p22f))) {  // of no number: 0 too, and noted
#pragma unroll
      for (int c = 0; c < GR; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t first = take_odd_scales(vs[c], x) + 16 * wave + 4 * q4 + 2 * x;
          if (first < KT) atomicMin(&odd_tile[flag][c], first);
        }
      if (lane == 0) atomicOr(&gone_tile[flag], 256u);
    }
    if (w.gone && lane == 0) atomicOr(&gone_tile[flag], 1u << wave);
  };
  auto store_value = [&](int c) {
    half2v v[4];
    values8(bits, vc[c], vs[c], v);
#pragma unroll
    for (int x = 0; x < 2; ++x)  // the first or second half of a piece
      *reinterpret_cast<lds_half4*>(lds0 + (v_to + (32 * c + x) * (KT * 2))) = half4{v[x][0], v[x][1], v[2 + x][0], v[2 + x][1]};
  };
  auto store_piece = [&](int c) {
    if (c < GR)
      store_key(c);
    else
      store_value(c - GR);
  };
  auto store = [&](const Tile& w, uint32_t buf, uint32_t flag) {
    store_begin(buf);
    store_scales(w, flag);
#pragma unroll
    for (int c = 0; c < 2 * GR; ++c) {
      store_piece(c);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // this lane's row
  const bool live = my_row < rows && t_row < rq.fresh;
  const int limit = live ? int(rq.len - rq.fresh + t_row) : -1;  // the last key that it sees
  half8 qh[DS], ql[DS];  // dims 16 ks + 8 h2 + e
  float unscale;
  {
    float big = 0.0f;
#pragma unroll
    for (int c = 0; c < DS; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float4& y = qx[c][e];
        y = live ? make_float4(y.x * a.s.scale2, y.y * a.s.scale2, y.z * a.s.scale2, y.w * a.s.scale2) : make_float4(0.f, 0.f, 0.f, 0.f);
        big = fmaxf(big, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
      }
    float inv;
    pow2_scale(half_reduce(big, [](float p, float q) { return fmaxf(p, q); }), unscale, inv);
#pragma unroll
    for (int c = 0; c < DS; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float4 z = qx[c][e / 4];
        const Parts y = split_query<false>((e % 4 == 0 ? z.x : e % 4 == 1 ? z.y : e % 4 == 2 ? z.z : z.w) * inv);
        qh[c][e] = y.hi;
        ql[c][e] = y.lo;
      }
  }

  floatx16 o[DT];  // dim 32 dt + 8 (v / 4) + 4 h2 + v % 4
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = floatx16{};
  float m = -INFINITY, l = 0.0f;
  if (tid < 3 * GR) (&odd_tile[0][0])[tid] = KT;
  if (tid < 3) gone_tile[tid] = 0;
  Tile w{}, next{};
  __syncthreads();
  if (n_tiles) {
    w = where(0);
    load(w);
    store(w, 0, 0);
    if (n_tiles > 1) {
      next = where(1);
      load(next);
    }
  }
  __syncthreads();
  uint32_t flag = 0;
  for (uint32_t i = 0; i < n_tiles; ++i) {
    const uint32_t buf = i & 1u, flag1 = flag == 2 ? 0 : flag + 1, flag2 = flag1 == 2 ? 0 : flag1 + 1;
    const Tile cur = w;
    if (tid < GR) odd_tile[flag2][tid] = KT;  // (last looked at a tile ago)
    if (tid == 0) gone_tile[flag2] = 0;
    const uint32_t gone = uniform(gone_tile[flag]);  // (and bit 8)
    const bool more = i + 1 < n_tiles;
    const bool sees = __any(limit >= int(cur.key0));  // else nothing of it is for this wave's rows
    if (more && !sees) store(next, buf ^ 1u, flag1);
    uint32_t k_from = buf * BUF + k_at(r32, h2), v_from = buf * BUF + v_at(r32, h2);
    asm volatile("" : "+v"(k_from), "+v"(v_from));
    auto value8 = [&](int sub, int st, int dt) { return *reinterpret_cast<const lds_half8*>(lds0 + ((v_from ^ (64u * sub + 32u * st)) + 32 * dt * (KT * 2))); };
    floatx16 s[2] = {};
    if (sees) {
      // A step: 16 dims of all scores, and a piece of the next tile (of what the registers hold, where there is none: it
      // goes where nobody reads).  Fragments are read two steps ahead; the barriers keep the compiler from reading all of
      // them first, the groups have it put other work between the products, which take as long as eight of it each.
      store_begin(buf ^ 1u);
      if (more) store_scales(next, flag1);
      half8 k8[3][2];
      auto read = [&](int c) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) k8[c % 3][sub] = *reinterpret_cast<const lds_half8*>(lds0 + ((k_from ^ (32u * c)) + 32 * sub * RB));
      };
      if (0 < DS) read(0);
      if (1 < DS) read(1);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int c = 0; c < DS; ++c) {
        if (c + 2 < DS) read(c + 2);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[c % 3][0], qh[c], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[c % 3][1], qh[c], s[1], 0, 0, 0);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[c % 3][0], ql[c], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[c % 3][1], ql[c], s[1], 0, 0, 0);
        store_piece(c);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
          __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // vector instructions
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (more) {
      w = next;
      if (i + 2 < n_tiles) {
        next = where(i + 2);
        load(next);
      }
    }
    if (sees) {
      __builtin_amdgcn_s_setprio(0);
      const bool whole = __all(!live || limit >= int(cur.key0) + KT - 1) && !(gone & 15u);
      if (!whole) {
        asm volatile("");  // (a branch: selects for every tile would cost as much as a fifth of its other vector work)
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (int(cur.key0) + int(32u * sub + 8u * (v / 4) + 4u * h2 + (v % 4)) > limit || ((gone >> (2 * sub + v / 8)) & 1u)) s[sub][v] = -INFINITY;
      }
      float top = -INFINITY, top1 = -INFINITY;
#pragma unroll
      for (int v = 0; v < 16; v += 2) {
        top = fmaxf(fmaxf(top, s[0][v]), s[0][v + 1]);
        top1 = fmaxf(fmaxf(top1, s[1][v]), s[1][v + 1]);
      }
      top = fmaxf(top, top1) * unscale;
      const float mn = fmaxf(m, half_reduce(top, [](float p, float q) { return fmaxf(p, q); }));
      const bool up = mn - m > LIFT + BEHIND;
      if (__any(up)) {
        const float to = up ? base_of(mn) : m, f = up ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
        l *= f;
        m = to;
      }
      const float bias = m == -INFINITY ? 0.0f : -m;
      if (gone >> 8) {  // values of no number
        asm volatile("");
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint32_t first = uniform(odd_tile[flag][dt]);
          if (first < KT && limit >= int(cur.key0 + first)) o[dt] = floatx16{} + NAN;
        }
      }
      // 16 keys each: the weights' f16 parts, and the rest
      half8 ph[2][2], pl[2][2];
      float sum[2] = {0.0f, 0.0f};
      auto weigh_pair = [&](int sub, int i) {
        const int v = 2 * i, to = v % 8;
        const float p = __builtin_amdgcn_exp2f(fmaf(s[sub][v], unscale, bias)), q = __builtin_amdgcn_exp2f(fmaf(s[sub][v + 1], unscale, bias));
        sum[0] += p;
        sum[1] += q;
        const WeightParts w2 = split_weights(p, q);
        ph[sub][v / 8][to] = w2.hi[0];
        ph[sub][v / 8][to + 1] = w2.hi[1];
        pl[sub][v / 8][to] = w2.lo[0];
        pl[sub][v / 8][to + 1] = w2.lo[1];
      };
#pragma unroll
      for (int i = 0; i < 8; ++i) weigh_pair(0, i);
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        // block c: 16 keys (st = c / DT) of 32 dims; its second term comes a block later, not right behind the first.  The
        // second half's weights are worked out between the first's products.
        constexpr int BL = 2 * DT, EACH = 8 / BL;
        half8 v8[6];
        auto read = [&](int c) { v8[c % 6] = value8(sub, c / DT, c % DT); };
        if (0 < BL) read(0);
        if (1 < BL) read(1);
        if (2 < BL) read(2);
        if (3 < BL) read(3);

#pragma unroll
        for (int c = 0; c <= BL; ++c) {
          if (c + 4 < BL) read(c + 4);
          if (c < BL) o[c % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8[c % 6], ph[sub][c / DT], o[c % DT], 0, 0, 0);
          if (c >= 1) o[(c - 1) % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8[(c - 1) % 6], pl[sub][(c - 1) / DT], o[(c - 1) % DT], 0, 0, 0);
          if (sub == 0 && c < BL) {
#pragma unroll
            for (int i = 0; i < EACH; ++i) weigh_pair(1, EACH * c + i);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      l += sum[0] + sum[1];
    }
    __syncthreads();
    flag = flag1;
  }

  l = half_reduce(l, [](float p, float q) { return p + q; });
  const bool last = splits == 1;
  if (my_row >= rows || (last && !live)) return;
  const size_t part = ((size_t(g) * sp.tiles + row / 16) * splits + split) * 16 + row % 16;
  float* dst = last ? a.out + at_row * HD : sp.o + part * HD;
  const float f = last ? (m == -INFINITY ? NAN : 1.0f / l) : 1.0f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<floatx4*>(dst + 32 * dt + 8 * c + 4 * h2) =
          floatx4{o[dt][4 * c] * f, o[dt][4 * c + 1] * f, o[dt][4 * c + 2] * f, o[dt][4 * c + 3] * f};
  if (h2 == 0 && !last) {
    sp.ml[2 * part] = m;
    sp.ml[2 * part + 1] = l;
  }
}

// The blocks' states of the rows of the output joined: HD / 4 threads per row and TEAM teams of them per row, each
// with every TEAM-th state.
template <int HD, int TEAM>
__global__ __launch_bounds__(256) void pg_join_kernel(KvAttendArgs a, PgShare sp) {
  constexpr uint32_t LP = HD / 4, ROWS = 256 / LP / TEAM;
  __shared__ floatx4 os[TEAM == 1 ? 1 : TEAM][LP];
  __shared__ float ms[TEAM], ls[TEAM];
  const uint32_t tid = threadIdx.x, team = tid / LP % TEAM, d = tid % LP;
  const uint32_t at = blockIdx.x * ROWS + tid / LP / TEAM;
  const bool is_row = at < a.c.R * a.c.n * a.s.H;
  const uint32_t out = is_row ? at : 0u, bt = out / a.s.H, h = out % a.s.H, b = bt / a.c.n, t = bt % a.c.n, g = h / a.s.rep;
  const RawRequest raw = load_request(a.c, b);
  const uint32_t row_b = t * a.s.rep + h % a.s.rep, row = sp.of_request ? row_b : b * a.c.n * a.s.rep + row_b, in_tile = row & ((1u << sp.shift) - 1u);
  const uint32_t tile = (sp.of_request ? b * sp.of_request : 0u) + (row >> sp.shift);
  const uint2 range = sp.ranges ? sp.ranges[tile] : make_uint2(tile * sp.each, sp.each);
  const size_t part = ((size_t(g) * sp.blocks + range.x) << sp.shift) + in_tile;
  float M = -INFINITY, L = 0.0f;
  floatx4 x = floatx4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t s0 = team; s0 < range.y; s0 += 4 * TEAM) {
    floatx4 y[4];
    float2 ml[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t s = min(s0 + i * TEAM, range.y - 1);
      const size_t of = part + (size_t(s) << sp.shift);
      ml[i] = *reinterpret_cast<const float2*>(sp.ml + 2 * of);
      if (TEAM > 1 || s0 + i < range.y) y[i] = *reinterpret_cast<const floatx4*>(sp.o + of * HD + 4 * d);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s0 + i * TEAM >= range.y) continue;
      if (ml[i].x == -INFINITY) {  // no key (zeros), or none but of no number
        x += y[i];
        L += ml[i].y;
        continue;
      }
      const float mn = fmaxf(M, ml[i].x);
      const float f0 = M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - mn), f1 = __builtin_amdgcn_exp2f(ml[i].x - mn);
      L = L * f0 + ml[i].y * f1;
      x = x * f0 + y[i] * f1;
      M = mn;
    }
  }
  if constexpr (TEAM > 1) {
    os[team][d] = x;
    if (d == 0) {
      ms[team] = M;
      ls[team] = L;
    }
    __syncthreads();
    if (team) return;
    float all = -INFINITY;
#pragma unroll
    for (int i = 0; i < TEAM; ++i) all = fmaxf(all, ms[i]);
    x = floatx4{0.f, 0.f, 0.f, 0.f};
    L = 0.0f;
#pragma unroll
    for (int i = 0; i < TEAM; ++i) {
      const float f = ms[i] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ms[i] - all);
      x += os[i][d] * f;
      L = fmaf(ls[i], f, L);
    }
    M = all;
  }
  if (!is_row || t >= checked(a.c, raw, nullptr).fresh) return;
  *reinterpret_cast<floatx4*>(a.out + size_t(out) * HD + 4 * d) = x * (M == -INFINITY ? NAN : 1.0f / L);
}

// ---------------------------------------------------------------------------
// rows and pools
// ---------------------------------------------------------------------------
constexpr uint32_t ROWS_THREADS = 1024, MAX_ROWS = 256;

__device__ __forceinline__ int32_t load_now(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Exclusive sum over the block's threads, and the sum of all.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t& all) {
  __shared__ uint32_t waves[ROWS_THREADS / 64];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t upto = wave_scan(x);
  __syncthreads();
  if (lane == 63) waves[wave] = upto;
  __syncthreads();
  uint32_t before = 0;
  all = 0;
#pragma unroll
  for (uint32_t i = 0; i < ROWS_THREADS / 64; ++i) {
    before += i < wave ? waves[i] : 0u;
    all += waves[i];
  }
  return before + upto - x;
}

// Every thread's stores and counts so far have reached memory and are seen by all.
__device__ __forceinline__ void settled() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}
// The same, and what has been found wrong so far (the same for all: nobody goes on to find more before all have read it).
__device__ __forceinline__ uint32_t settled(const uint32_t& bad) {
  settled();
  const uint32_t x = *const_cast<const volatile uint32_t*>(&bad);
  __syncthreads();
  return x;
}

// Neighbouring counts of a pool's pages (4-byte addresses will do).
template <int N>
struct Counts {
  int32_t of[N];
};
template <int N>
__device__ __forceinline__ Counts<N> load_counts(const int32_t* from) {
  Counts<N> x;
  __builtin_memcpy(&x, from, sizeof x);
  return x;
}
template <int N>
__device__ __forceinline__ void store_counts(int32_t* to, Counts<N> x) {
  __builtin_memcpy(to, &x, sizeof x);
}
// f(p, counts from p on) for all pages, by the block's threads: of many pages four at a time, two such loads together.  (One
// block, so what is in flight is what there is of bandwidth; a turn that a small pool does not need is a jump.)
template <class F>
__device__ __forceinline__ void each_page(const int32_t* refs, uint32_t pages, F&& f) {
  constexpr uint32_t T = ROWS_THREADS;
  const uint32_t tid = threadIdx.x;
  uint32_t p0 = 0;
  for (; p0 + 8 * T <= pages; p0 += 8 * T) {
    const uint32_t p = p0 + 4 * tid;
    const Counts<4> x = load_counts<4>(refs + p), y = load_counts<4>(refs + p + 4 * T);
    f(p, x);
    f(p + 4 * T, y);
  }
  for (; p0 < pages; p0 += T)
    if (p0 + tid < pages) f(p0 + tid, load_counts<1>(refs + p0 + tid));
}
// f(p, count) where order counts: each wave has a run of pages, 64 at a time, and all its lanes take part (`rest` behind the pages).
template <class F>
__device__ __forceinline__ void by_waves(const int32_t* refs, uint32_t pages, int32_t rest, F&& f) {
  constexpr uint32_t WAVES = ROWS_THREADS / 64;
  const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), per = ((pages + WAVES - 1) / WAVES + 63) / 64 * 64;
  const uint32_t lo = min(wave * per, pages), hi = min(lo + per, pages);
  uint32_t p0 = lo;
  for (; p0 + 256 <= hi; p0 += 256) {
    int32_t x[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) x[k] = refs[p0 + 64 * k + lane];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) f(p0 + 64 * k + lane, x[k]);
  }
  for (; p0 < hi; p0 += 64) f(p0 + lane, p0 + lane < hi ? refs[p0 + lane] : rest);
}
__device__ __forceinline__ uint32_t lanes_below(uint64_t of) {
  return __builtin_amdgcn_mbcnt_hi(uint32_t(of >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(of), 0));
}
// The block's sum of what its waves have, each the same in all lanes, and that of the waves before.
__device__ __forceinline__ uint32_t wave_offsets(uint32_t x, uint32_t& all) {
  return uniform(block_scan((threadIdx.x & 63u) == 0 ? x : 0u, all));
}

// Nothing changes: arrays out become as those in.
__device__ __forceinline__ void copy_rows(const PgUpdateArgs& a) {
  const uint32_t tid = threadIdx.x;
  if (a.refs_out != a.refs)
    for (uint32_t p = tid; p < a.p.pages; p += ROWS_THREADS) a.refs_out[p] = a.refs[p];
  if (a.table_out != a.p.table)
    for (uint32_t i = tid; i < a.R * a.p.width; i += ROWS_THREADS) a.table_out[i] = a.p.table[i];
  if (a.lens_out && a.lens_out != a.lens && tid < a.R) a.lens_out[tid] = a.lens[tid];
}

__device__ __forceinline__ void copy_page(const PgUpdateArgs& a, uint32_t layer, int32_t from, int32_t to, uint32_t bytes, uint32_t i0, uint32_t step) {
  uint8_t* pool = a.p.pool + layer * a.layer_stride;
  const u32x4* src = reinterpret_cast<const u32x4*>(pool + size_t(from) * bytes);
  u32x4* dst = reinterpret_cast<u32x4*>(pool + size_t(to) * bytes);
  for (uint32_t i = i0; i < bytes / 16; i += step) dst[i] = src[i];
}

// n pages, from[i] to to[i], in every layer, by all of the grid's blocks: 16 KB a turn.
__device__ __forceinline__ void copy_pages(const PgUpdateArgs& a, const int32_t* from, const int32_t* to, uint32_t n, uint32_t bytes) {
  constexpr uint32_t TURN = 16 * ROWS_THREADS;
  const uint32_t parts = (bytes + TURN - 1) / TURN, per_layer = n * parts, all = per_layer * a.layers;
  u32x4* to_now = nullptr;  // a turn's loads before the stores of the one before
  u32x4 now{};
  for (uint32_t i = blockIdx.x; i < all; i += gridDim.x) {
    const uint32_t layer = i / per_layer, page = i % per_layer / parts, at = i % parts * TURN + threadIdx.x * 16;
    if (at >= bytes) continue;
    uint8_t* pool = a.p.pool + layer * a.layer_stride + at;
    const u32x4 next = *reinterpret_cast<const u32x4*>(pool + size_t(from[page]) * bytes);
    if (to_now) *to_now = now;
    to_now = reinterpret_cast<u32x4*>(pool + size_t(to[page]) * bytes);
    now = next;
  }
  if (to_now) *to_now = now;
}

// One block, a wave per row at a time.  References are counted apart: what every row holds is taken off, then what it will
// hold added, also where that is the same: a count that goes below 0 on the way was below the rows that hold the page, and
// two rows would each take the page for their own.  Of w rows that write to a page of r references, the
// first r - 1 write to copies: the last writes in place if no one else holds it.
//   All latency: two loads one after the other (the rows' lengths, their pages), a few turns over LDS, the stores; sixteen
// waves share four vector units, so each instruction of a turn counts (64 rows of 102 pages 13 us, 16 of 32 pages 8, of a
// pool of 7000).  FITS: counts, free pages and new rows are in LDS.  COUNTS: the counts alone, the rest in the workspace (64
// rows of 32 pages, tables of 512, in a pool of 20000: 19 us; the counts there too, 32).  Else each turn is a trip to the
// second-level cache (64 rows of 102 pages of a pool of 38400, the most for COUNTS, 20 us, of 38401 36).
//   MOVES (arrays out apart from those in): every block works it all out for itself, the first writes it down, and all of
// them copy pages: one launch (16 rows 8.5 us; in place, with a second launch that copies, 9.3, and the caller's own 2.7 for
// it).  64 rows that each copy a page in 36 layers: 31 us, 122 MB in 18 of them.
constexpr uint32_t ROWS_LDS = 150 * 1024;  // bytes: counts, free pages, rows

template <bool COUNTS, bool FITS, bool MOVES>
__global__ __launch_bounds__(ROWS_THREADS) void pg_update_kernel(PgUpdateArgs a, PgWorkspace w, uint32_t bytes) {
  extern __shared__ int32_t dyn[];
  __shared__ int32_t source[MAX_ROWS], lens[MAX_ROWS], kept[MAX_ROWS], total[MAX_ROWS], last[MAX_ROWS], before[MAX_ROWS];
  __shared__ uint32_t first[MAX_ROWS], offset[MAX_ROWS], bad;
  const bool writes = !MOVES || blockIdx.x == 0;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), width = a.p.width, page_up = (1u << a.p.shift) - 1u;
  const int64_t cap = int64_t(width) << a.p.shift;
  auto refs = [&](uint32_t p) -> int32_t* {
    if constexpr (COUNTS) return dyn + p;
    return w.refs + p;
  };
  auto list = [&](uint32_t i) -> int32_t* {
    if constexpr (FITS) return dyn + a.p.pages + i;
    return w.list + i;
  };
  auto rows = [&](uint32_t x) -> int32_t* {
    if constexpr (FITS) return dyn + 2 * a.p.pages + x;
    return w.table + x;
  };
  auto count = [&](uint32_t p) {  // now, with what others have added
    if constexpr (COUNTS) return *refs(p);
    return load_now(refs(p));
  };
  auto pages_of = [&](int32_t n) { return (uint32_t(n) + page_up) >> a.p.shift; };
  auto report = [&](uint32_t bits) { atomicOr(&bad, bits); };
  if (tid == 0) bad = 0;
  int32_t keep = 0, add = 0;
  __syncthreads();
  if (tid < a.R) {
    source[tid] = a.source ? a.source[tid] : int32_t(tid);
    lens[tid] = a.lens[tid];
    keep = a.keep ? a.keep[tid] : 0x7fffffff;
    add = a.add ? a.add[tid] : 0;
    if (!MOVES) w.moves[2 * tid] = -1;
    if (lens[tid] < 0 || lens[tid] > cap || source[tid] < -1 || source[tid] >= int32_t(a.R) || keep < 0 || add < 0) report(S2HIP_PAGES_ERR_LENS);
  }
  each_page(a.refs, a.p.pages, [&](uint32_t p, auto x) { store_counts(refs(p), x); });
  auto turn_over = [&] {
    if constexpr (FITS)
      __syncthreads();
    else
      settled();
  };
  auto stops = [&] {
    turn_over();
    const uint32_t why = *const_cast<const volatile uint32_t*>(&bad);
    __syncthreads();
    if (why && writes) copy_rows(a);
    if (why && writes && tid == 0) atomicOr(a.err, why);
    return why != 0;
  };
  if (stops()) return;
  if (tid < a.R) {
    kept[tid] = source[tid] < 0 ? 0 : min(keep, lens[source[tid]]);
    if (int64_t(kept[tid]) + add > cap) report(S2HIP_PAGES_ERR_LENS);
    total[tid] = int32_t(uint32_t(kept[tid]) + uint32_t(add));
  }
  if (stops()) return;
  // (what is the same for a row's lanes in scalar registers: the block's sixteen waves share four vector units)
  for (uint32_t b = wave; b < a.R; b += ROWS_THREADS / 64) {
    const uint32_t n_old = uniform(pages_of(lens[b])), n_base = uniform(pages_of(kept[b])), s = uniform(uint32_t(source[b]));
    const int32_t *old_row = a.p.table + size_t(b) * width, *base_row = a.p.table + size_t(s == 0xffffffffu ? 0 : s) * width;
    const bool same = s == b;
    for (uint32_t i0 = 0; i0 < max(n_old, n_base); i0 += 128) {  // two entries a lane, their loads together
      int32_t e[2], v[2];
#pragma unroll
      for (uint32_t k = 0; k < 2; ++k) {
        const uint32_t i = i0 + 64 * k + lane;
        e[k] = i < n_old ? old_row[i] : 0;
        v[k] = same ? e[k] : i < n_base ? base_row[i] : 0;
      }
#pragma unroll
      for (uint32_t k = 0; k < 2; ++k) {
        const uint32_t i = i0 + 64 * k + lane;
        const bool in = uint32_t(e[k]) < a.p.pages && uint32_t(v[k]) < a.p.pages;
        if (!in) report(S2HIP_PAGES_ERR_PAGE);
        if (COUNTS && in && i < n_old && atomicSub(refs(uint32_t(e[k])), 1) < 1) report(S2HIP_PAGES_ERR_REFS);
        if (i < n_base) *rows(b * width + i) = v[k];
      }
    }
  }
  if (stops()) return;
  if constexpr (COUNTS) {
    for (uint32_t b = wave; b < a.R; b += ROWS_THREADS / 64) {
      const uint32_t n = uniform(pages_of(kept[b]));
      for (uint32_t i0 = 0; i0 < n; i0 += 128) {
        const uint32_t i = i0 + lane;
        if (i < n) atomicAdd(refs(uint32_t(*rows(b * width + i))), 1);
        if (i + 64 < n) atomicAdd(refs(uint32_t(*rows(b * width + i + 64))), 1);
      }
    }
  } else {
    // f(page, how many) of the entries table[b][i], i below the pages of n[b] tokens: a lane takes a column of the wave's rows,
    // and those that have a page in common there, as rows that begin alike do, are one change of its count.  (One change
    // each, 64 rows with 93 pages in common made anew in a pool of 38401: 47 us, so 36.)
    auto by_columns = [&](const int32_t* table, const int32_t* n, auto&& f) {
      constexpr uint32_t WAVES = ROWS_THREADS / 64;
      uint32_t most = 0;
      for (uint32_t b = wave; b < a.R; b += WAVES) most = max(most, uniform(pages_of(n[b])));
      for (uint32_t i0 = 0; i0 < most; i0 += 64) {
        const uint32_t i = i0 + lane;
        int32_t page = -1, count = 0;
        for (uint32_t b0 = wave; b0 < a.R; b0 += 4 * WAVES) {
          int32_t e[4];
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t b = b0 + k * WAVES;
            e[k] = b < a.R && i < uniform(pages_of(n[min(b, a.R - 1)])) ? table[size_t(b) * width + i] : -1;
          }
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) {
            if (e[k] != page) {
              if (page >= 0) f(uint32_t(page), count);
              page = e[k];
              count = 0;
            }
            ++count;
          }
        }
        if (page >= 0) f(uint32_t(page), count);
      }
    };
    by_columns(a.p.table, lens, [&](uint32_t p, int32_t n) {
      if (atomicSub(refs(p), n) < n) report(S2HIP_PAGES_ERR_REFS);
    });
    if (stops()) return;
    by_columns(w.table, kept, [&](uint32_t p, int32_t n) { atomicAdd(refs(p), n); });
  }
  const bool grows = tid < a.R && add > 0 && (uint32_t(kept[tid]) & page_up) != 0;
  if (tid < a.R) last[tid] = grows ? *rows(tid * width + (uint32_t(kept[tid]) >> a.p.shift)) : -1;
  turn_over();
  for (uint32_t b = wave; b < a.R; b += ROWS_THREADS / 64) {  // earlier rows that grow into the same page
    uint32_t n = 0;
    for (uint32_t i = lane; i < (b + 63) / 64 * 64; i += 64) n += uint32_t(__popcll(__ballot(i < b && last[i] == last[b])));
    if (lane == 0) before[b] = int32_t(n);
  }
  __syncthreads();
  uint32_t needs = 0, copies = 0;
  if (tid < a.R) {
    if (grows) copies = before[tid] < count(uint32_t(last[tid])) - 1;
    first[tid] = pages_of(kept[tid]) - copies;
    needs = pages_of(total[tid]) - first[tid];
  }
  uint32_t all, found;
  const uint32_t begin = block_scan(needs, all);
  if (tid < a.R) offset[tid] = begin;
  // the free pages: each wave counts those of a run of pages, then says which they are
  if constexpr (!COUNTS) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");  // (plain loads of what atomics have changed)
  uint32_t mine = 0;
  bool below = false;
  by_waves(refs(0), a.p.pages, 1, [&](uint32_t, int32_t r) {
    mine += uint32_t(__popcll(__ballot(r == 0)));
    below |= r < 0;
  });
  if (below) report(S2HIP_PAGES_ERR_REFS);
  uint32_t rank = wave_offsets(mine, found);
  if (mine && rank < all)
    by_waves(refs(0), a.p.pages, 1, [&](uint32_t p, int32_t r) {
      const uint64_t free = __ballot(r == 0);
      const uint32_t to = rank + lanes_below(free);
      if (r == 0 && to < all) *list(to) = int32_t(p);
      rank += uint32_t(__popcll(free));
    });
  if (found < all && tid == 0) report(S2HIP_PAGES_ERR_FULL);
  if (stops()) return;
  if constexpr (MOVES) {
    uint32_t n;
    const uint32_t at = block_scan(copies, n);
    if (copies) {
      source[at] = last[tid];
      kept[at] = *list(offset[tid]);
    }
    __syncthreads();
    copy_pages(a, source, kept, n, bytes);
    if (!writes) return;
  }
  for (uint32_t i = tid; i < all; i += ROWS_THREADS) *refs(uint32_t(*list(i))) = 1;
  turn_over();
  if (tid < a.R) {
    a.lens_out[tid] = total[tid];
    if (copies) {
      if (!MOVES) {
        w.moves[2 * tid] = last[tid];
        w.moves[2 * tid + 1] = *list(offset[tid]);
      }
      atomicSub(refs(uint32_t(last[tid])), 1);
    }
  }
  for (uint32_t b = wave; b < a.R; b += ROWS_THREADS / 64) {
    const uint32_t n = uniform(pages_of(total[b])), from = uniform(first[b]), at = uniform(offset[b]);
    for (uint32_t i = lane; i < width; i += 64) a.table_out[size_t(b) * width + i] = i < from ? *rows(b * width + i) : i < n ? *list(at + i - from) : -1;
  }
  turn_over();
  if constexpr (!COUNTS) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  each_page(refs(0), a.p.pages, [&](uint32_t p, auto x) { store_counts(a.refs_out + p, x); });
}

// blockIdx.y = row, z = layer
__global__ __launch_bounds__(256) void pg_copy_kernel(PgUpdateArgs a, const int32_t* moves, uint32_t bytes) {
  const int32_t from = moves[2 * blockIdx.y];
  if (from >= 0) copy_page(a, blockIdx.z, from, moves[2 * blockIdx.y + 1], bytes, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// The pages in use, the lists of holes and movers, refs.  A short call is three trips over refs (1 layer of a few hundred
// pages 6 us), a long one memory (36 layers, 12 x 3500 tokens, half of the pages moved: 270 to 290 us, 1.36 GB: 4.7 to 5 TB/s).  MOVES (arrays out apart from those in, and few enough pages):
// every block works them out in its LDS, and all of them move pages and rewrite the table; else one block leaves the
// lists in the workspace.
template <bool MOVES>
__global__ __launch_bounds__(ROWS_THREADS) void pg_pack_kernel(PgUpdateArgs a, PgWorkspace w, uint32_t bytes) {
  extern __shared__ int32_t dyn[];  // MOVES: holes, movers, where each page goes
  __shared__ uint32_t bad;
  const bool writes = !MOVES || blockIdx.x == 0;
  const uint32_t tid = threadIdx.x, width = a.p.width, page_up = (1u << a.p.shift) - 1u, pages = a.p.pages;
  int32_t* const holes = MOVES ? dyn : w.list;
  int32_t* const movers = MOVES ? dyn + pages : w.list + pages;
  int32_t* const moved = MOVES ? dyn + 2 * pages : w.refs;
  auto pages_of = [&](int32_t n) { return (uint32_t(n) + page_up) >> a.p.shift; };
  if (tid == 0) bad = 0;
  __syncthreads();
  // each wave looks at a run of pages
  const uint32_t lane = tid & 63u;
  uint32_t mine = 0, used;
  bool below = false;
  by_waves(a.refs, pages, 0, [&](uint32_t, int32_t r) {
    mine += uint32_t(__popcll(__ballot(r > 0)));
    below |= r < 0;
  });
  if (below) atomicOr(&bad, S2HIP_PAGES_ERR_REFS);
  for (uint32_t b = tid >> 6; b < a.R; b += ROWS_THREADS / 64) {
    const int32_t len = a.lens[b];
    if (len < 0 || int64_t(len) > int64_t(width) << a.p.shift) {
      atomicOr(&bad, S2HIP_PAGES_ERR_LENS);
      continue;
    }
    for (uint32_t i = lane; i < pages_of(len); i += 64) {
      const int32_t e = a.p.table[size_t(b) * width + i];
      if (uint32_t(e) >= pages)
        atomicOr(&bad, S2HIP_PAGES_ERR_PAGE);
      else if (a.refs[e] < 1)
        atomicOr(&bad, S2HIP_PAGES_ERR_REFS);
    }
  }
  wave_offsets(mine, used);
  const uint32_t why = settled(bad);
  if (writes && tid == 0) a.used_out[0] = int32_t(used);
  if (why) {
    if (!writes) return;
    if (tid == 0) {
      w.moves[0] = 0;
      w.moves[1] = 0x7fffffff;  // no entry follows
      atomicOr(a.err, why);
    }
    if (a.refs_out != a.refs)
      for (uint32_t p = tid; p < pages; p += ROWS_THREADS) a.refs_out[p] = a.refs[p];
    if (a.moved_to)
      for (uint32_t p = tid; p < pages; p += ROWS_THREADS) a.moved_to[p] = a.refs[p] > 0 ? int32_t(p) : -1;
    if (MOVES)
      for (uint32_t i = tid; i < a.R * width; i += ROWS_THREADS) a.table_out[i] = a.p.table[i];
    return;
  }
  uint32_t here[2] = {0, 0}, n_holes, n_movers;
  by_waves(a.refs, pages, -1, [&](uint32_t p, int32_t r) {
    here[0] += uint32_t(__popcll(__ballot(p < used && r == 0)));
    here[1] += uint32_t(__popcll(__ballot(p >= used && r > 0)));
  });
  uint32_t h = wave_offsets(here[0], n_holes), m = wave_offsets(here[1], n_movers);  // (as many of one as of the other)
  if (here[0] || here[1])
    by_waves(a.refs, pages, -1, [&](uint32_t p, int32_t r) {
      const bool hole = p < used && r == 0, mover = p >= used && r > 0;
      const uint64_t hs = __ballot(hole), ms = __ballot(mover);
      if (hole) holes[h + lanes_below(hs)] = int32_t(p);
      if (mover) movers[m + lanes_below(ms)] = int32_t(p);
      h += uint32_t(__popcll(hs));
      m += uint32_t(__popcll(ms));
    });
  settled();
  for (uint32_t i = tid; i < n_movers; i += ROWS_THREADS) moved[movers[i]] = holes[i];
  if (writes && (a.refs_out != a.refs || a.moved_to))
    each_page(a.refs, pages, [&](uint32_t p, auto x) {
      auto out = x, to = x;
#pragma unroll
      for (uint32_t i = 0; i < sizeof x / 4; ++i) {
        out.of[i] = p + i < used ? x.of[i] : 0;
        to.of[i] = x.of[i] > 0 ? int32_t(p + i) : -1;
      }
      if (a.refs_out != a.refs) store_counts(a.refs_out + p, out);
      if (a.moved_to) store_counts(a.moved_to + p, to);
    });
  settled();
  if (writes)
    for (uint32_t i = tid; i < n_movers; i += ROWS_THREADS) {
      const int32_t from = movers[i], to = holes[i], r = a.refs[from];
      a.refs_out[to] = r;
      a.refs_out[from] = 0;
      if (a.moved_to) a.moved_to[from] = to;
    }
  if constexpr (MOVES) {
    for (uint32_t x = blockIdx.x * ROWS_THREADS + tid; x < a.R * width; x += gridDim.x * ROWS_THREADS) {
      const int32_t e = a.p.table[x];
      if (x % width < pages_of(a.lens[x / width])) a.table_out[x] = uint32_t(e) >= used ? moved[e] : e;
    }
    copy_pages(a, movers, holes, n_movers, bytes);
  } else if (tid == 0) {
    w.moves[0] = int32_t(n_movers);
    w.moves[1] = int32_t(used);
  }
}

// The pages in blocks' turns, and the table.
__global__ __launch_bounds__(256) void pg_move_kernel(PgUpdateArgs a, PgWorkspace w, uint32_t bytes) {
  const uint32_t n = uint32_t(w.moves[0]), used = uint32_t(w.moves[1]), page_up = (1u << a.p.shift) - 1u;
  for (uint32_t x = blockIdx.x * 256 + threadIdx.x; x < a.R * a.p.width; x += gridDim.x * 256) {
    const int32_t len = a.lens[x / a.p.width], e = a.p.table[x];
    const bool in_use = x % a.p.width < (uint32_t(len) + page_up) >> a.p.shift;
    if (used == 0x7fffffffu) {
      if (a.table_out != a.p.table) a.table_out[x] = e;
    } else if (in_use) {
      a.table_out[x] = uint32_t(e) >= used ? w.refs[e] : e;
    }
  }
  for (uint32_t i = blockIdx.x; i < n * a.layers; i += gridDim.x)
    copy_page(a, i / n, w.list[a.p.pages + i % n], w.list[i % n], bytes, threadIdx.x, 256);
}

template <class F>
hipError_t by_dim(uint32_t hd, F&& f) {
  if (hd == 64) return f(std::integral_constant<int, 64>());
  if (hd == 128) return f(std::integral_constant<int, 128>());
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_pg_append(uint32_t hd, const PgAppendArgs& a, hipStream_t s) {
  return by_dim(hd, [&](auto HD) {
    const uint32_t tokens = a.c.R * a.c.n, steps = ((a.s.H + 2 * a.s.G) * HD() + 2047) / 2048;
    const dim3 grid(tokens, min(steps, max(1u, 512 / tokens)));
    auto go = [&](auto HALF) { hipLaunchKernelGGL((pg_append_kernel<HD(), HALF()>), grid, dim3(256), 0, s, a); };
    if (a.rope.half)
      go(std::true_type());
    else
      go(std::false_type());
    return hipGetLastError();
  });
}

hipError_t launch_pg_attend(uint32_t hd, PgAttendArgs pa, const PgWorkspace& w, hipStream_t s) {
  const KvAttendArgs& a = pa.a;
  pa.by_rows = Div::by(a.c.n * a.s.rep);
  pa.by_rep = Div::by(a.s.rep);
  pa.by_groups = Div::by(a.s.G);
  PgShare sp{};
  sp.o = w.part;
  sp.ml = w.part_ml;
  const uint32_t per = a.c.n * a.s.rep, rows = a.c.R * per;
  // A row tile with rows of two requests walks both's keys, twice as long as its neighbours; tiles of one request each have
  // empty rows (the step kernel's up to a third, but where 32 rows hold the request).  Tiles of two : of one, us, heads 32 over 8
  // of 128: 8 x 500 tokens over 4000 467 : 329, 8 x 100 (400 rows) over 4000 188 : 112, over 1500 shared + 500 79 : 70; of 16
  // rows 16 x 3 (12 rows) over 4000 38 : 30.
  auto apart = [&](uint32_t n) { return (per + n - 1) / n * n <= per + per / 3; };
  // The tile kernel takes half as long for a score but 10 us more (128 rows' states).  Step : tile kernel: 1 x 1000 over 1000
  // (20 M scores) 47 : 46, 1 x 1200 over 1200 (29) 61 : 55, 2 x 100 over 4000 (26) 57 : 50, heads 64 over 8, 2 x 50 over 3000 (20) 55 :
  // 39; of 160 rows, which are two tiles, 8 x 40 over 4000 65 : 68, over 3500 shared + 500 84 : 69.  (Requests of fewer than 96
  // rows, several to a tile: 8 x 20 over 16000 118 : 167, 8 x 8 over 20000 shared + 500 77 : 66.)
  const size_t scores = size_t(a.s.G) * rows * (a.c.cap - min(a.c.n, a.c.cap) / 2);
  const bool many = per >= 96 && scores > 18000000u * size_t(128) / hd;
  // Rows of the step kernel's tiles.  32 take a key's four bits apart once for twice as many, but short runs want the waves of
  // 16.  16 : 32, us: 16 x 5 over 32001 239 : 172, 8 x 8 over 16000 64 : 58, 1 x 100 over 4000 44 : 41, 8 x 8 over 4000 29 : 31,
  // 2 x 6 over 500 10.6 : 13.0, 1 x 40 over 200 9.0 : 12.1; where 16 would have rows of two requests, 16 x 5 over 1000 28 : 20.
  const bool two = !many && per > 16 && size_t(a.s.G) * ((rows + 15) / 16) * ((a.c.cap + 31) / 32) >= (apart(16) ? 16 : 4) * 1024;
  const uint32_t tile_rows = many ? uint32_t(TILE_ROWS) : two ? 32 : 16, of_request = (per + tile_rows - 1) / tile_rows;
  if (many || apart(tile_rows) || (two && of_request == 1)) sp.of_request = of_request;
  sp.by_of = Div::by(of_request);
  sp.row_tiles = sp.of_request ? a.c.R * of_request : (rows + tile_rows - 1) / tile_rows;
  sp.tiles = many ? (rows + 15) / 16 : sp.row_tiles;
  sp.shift = two ? 5 : 4;
  const uint32_t kt = many ? 64 : 32, lots = a.s.G * sp.row_tiles;
  const uint32_t most = (a.c.cap + kt - 1) / kt * (many || sp.of_request ? 1u : min(a.c.R, (tile_rows - 1) / per + 1));  // key tiles of a row tile (one that begins inside a request may have a request more)
  // Blocks of the step kernel, by the key tiles that a wave of 256 would walk at most: short runs end sooner with fewer
  // states to join, long ones want more waves to take turns.  256 : 512 : 768 blocks, us: 8 x 1 over 1500 + 512 (4 tiles) 13 :
  // 17 : 21, 16 x 1 over 1000 (5) 17 : 18 : 21, 1 x 1 over 30000 (7) 21 : 20 : 22, 16 x 1 over 6000 (24) 44 : 35 : 34, over
  // 32001 (126) 202 : 127 : 120.
  const size_t walk = size_t(lots) * most / 1024;
  const uint32_t fill = many ? PG_TILE_BLOCKS : walk < 6 ? 256 : walk < 24 ? 512 : PG_STEP_BLOCKS;
  // (the tile kernel's: 8 key tiles each on average, or their states cost more than they save: 1 x 1000 in 1 : 2 46 : 54, 1 x 100
  // over 4000 in 4 : 8 : 16 50 : 38 : 42)
  uint32_t splits = max(1u, min(fill / lots, many ? (a.c.cap - min(a.c.n, a.c.cap) / 2) / (8 * kt) : (most + STEP_WAVES - 1) / STEP_WAVES));
  // One block, and no join, for short runs (in a graph, one : several, us: 1 x 1, table of 14 tiles 8.9 : 9.1, of 18 10.1 : 9.2;
  // heads of 64, 18 8.3 : 8.4, 26 10.1 : 8.4).
  if (!many && most <= (hd == 64 ? 24u : 16u)) splits = 1;
  const size_t parts = size_t(a.s.G) * sp.tiles << (sp.shift - 4);  // (16 rows each)
  if (splits > 1 && parts * splits > PG_STATES) return hipErrorInvalidValue;  // (lots splits is at most fill)
  sp.blocks = sp.tiles * splits;
  sp.each = splits;
  sp.by_each = Div::by(splits);
  // Shares by length where runs are long (1 of 16 over 32001, the others over 500: 30 us, equal shares 39): they take up to a
  // microsecond to work out.
  if (!many && splits > 1 && walk >= 6 && sp.tiles > 1 && sp.tiles <= 64) sp.ranges = w.ranges;
  return by_dim(hd, [&](auto HD) {
    if (many)
      hipLaunchKernelGGL(pg_tile_kernel<HD()>, dim3(lots * splits), dim3(256), 0, s, pa, sp);
    else {
      const dim3 grid(a.s.G * sp.blocks), block(64 * STEP_WAVES);
      auto step = [&](auto TWO, auto RG) { hipLaunchKernelGGL((pg_step_kernel<HD(), TWO(), RG()>), grid, block, 0, s, pa, sp); };
      auto pages = [&](auto RG) {
        if (pa.p.shift == 4)  // a tile takes two pages
          step(std::true_type(), RG);
        else
          step(std::false_type(), RG);
      };
      if (two)
        pages(std::integral_constant<int, 2>());
      else
        pages(std::integral_constant<int, 1>());
    }
    // (several teams a row : one, us: 8 x 1 over 2000 16.7 : 18.6, 16 x 1 over 8000 40.3 : 44.7, 64 x 1 over 2000 43.0 : 42.6)
    if (many) sp.of_request = 0;  // (its states go by rows alone)
    const uint32_t out_rows = a.c.R * a.c.n * a.s.H, teams = 256 / (HD() / 4);
    if (splits > 1 && out_rows <= 2048)
      hipLaunchKernelGGL((pg_join_kernel<HD(), 1024 / HD()>), dim3(out_rows), dim3(256), 0, s, a, sp);
    else if (splits > 1)
      hipLaunchKernelGGL((pg_join_kernel<HD(), 1>), dim3((out_rows + teams - 1) / teams), dim3(256), 0, s, a, sp);
    return hipGetLastError();
  });
}

// n ints from p, from q: any in common?
static bool meets(const void* p, const void* q, size_t n) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
  return x < y + 4 * n && y < x + 4 * n;
}

// Once per device, before the launches there.
hipError_t prepare_pg() {
  static std::atomic<uint64_t> devices[4];
  const void* kernels[4] = {reinterpret_cast<const void*>(pg_update_kernel<true, true, true>), reinterpret_cast<const void*>(pg_update_kernel<true, true, false>),
                            reinterpret_cast<const void*>(pg_update_kernel<true, false, false>), reinterpret_cast<const void*>(pg_pack_kernel<true>)};
  for (int i = 0; i < 4; ++i) {
    const hipError_t e = allow_lds(kernels[i], ROWS_LDS, devices[i]);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// A kernel of one block (or several that do the same) with `lds` bytes of LDS.
template <class K>
static hipError_t launch_rows(K kernel, uint32_t blocks, size_t lds, hipStream_t s, const PgUpdateArgs& a, const PgWorkspace& w, uint32_t bytes) {
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(ROWS_THREADS), lds, s, a, w, bytes);
  return hipGetLastError();
}

hipError_t launch_pg_update(const PgUpdateArgs& a, const PgWorkspace& w, uint32_t page_bytes, hipStream_t s) {
  const size_t words = size_t(a.R) * a.p.width, lds = (2 * size_t(a.p.pages) + words) * 4;
  const bool fits = lds <= ROWS_LDS, in_place = meets(a.refs, a.refs_out, a.p.pages) || meets(a.p.table, a.table_out, words) || meets(a.lens, a.lens_out, a.R);
  if (fits && !in_place) return launch_rows(pg_update_kernel<true, true, true>, 256, lds, s, a, w, page_bytes);
  const size_t counts = size_t(a.p.pages) * 4;
  const hipError_t e = fits                 ? launch_rows(pg_update_kernel<true, true, false>, 1, lds, s, a, w, page_bytes)
                       : counts <= ROWS_LDS ? launch_rows(pg_update_kernel<true, false, false>, 1, counts, s, a, w, page_bytes)
                                            : launch_rows(pg_update_kernel<false, false, false>, 1, 0, s, a, w, page_bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(pg_copy_kernel, dim3((page_bytes + 16383) / 16384, a.R, a.layers), dim3(256), 0, s, a, w.moves, page_bytes);
  return hipGetLastError();
}

hipError_t launch_pg_compact(const PgUpdateArgs& a, const PgWorkspace& w, uint32_t page_bytes, hipStream_t s) {
  const size_t words = size_t(a.R) * a.p.width, lds = 3 * size_t(a.p.pages) * 4;
  if (lds <= ROWS_LDS && !meets(a.refs, a.refs_out, a.p.pages) && !meets(a.p.table, a.table_out, words))
    return launch_rows(pg_pack_kernel<true>, 256, lds, s, a, w, page_bytes);
  const hipError_t e = launch_rows(pg_pack_kernel<false>, 1, 0, s, a, w, page_bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(pg_move_kernel, dim3(2048), dim3(256), 0, s, a, w, page_bytes);
  return hipGetLastError();
}

}  // namespace s2
