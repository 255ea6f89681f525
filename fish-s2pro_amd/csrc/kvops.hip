// kvops.hip -- KV-cache operators for gfx950 (CDNA4, wave64): head norms,
// rotation and cache write of a batch's new tokens; attention over a shared
// prefix and the requests' own caches, with or without the keys' weights;
// eviction by score.

#include <type_traits>

#include "kvops.h"
#include "lds_dma.h"
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

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// One block per token and run of heads (blockIdx.y, every gridDim.y-th 8 or 16):
// the token's hd / 2 angles once (64-bit product with the position, whole turns
// taken off in 64 bits, cos and sin of the rest in f32, turned by what its rounding
// left), then 4 elements (two
// pairs) per thread.  Memory bound: 8 requests x 250 tokens of 32 + 8 + 8 heads,
// f16 caches, read and write 71 MB in 13.3 us (5.3 TB/s); one step of 8 requests
// is all latency (3 us), so its loads start together and its heads are spread over
// blocks.
template <int HD, bool KH>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a) {
  constexpr uint32_t LP = HD / 4;       // lanes per head
  constexpr uint32_t HPB = 256 / LP;    // heads per step of the block
  __shared__ float2 turn[HD / 2];
  const uint32_t tid = threadIdx.x, b = blockIdx.x / a.c.n, t = blockIdx.x % a.c.n;
  const RawRequest raw = load_request(a.c, b);
  const int32_t pos = a.positions[size_t(b) * a.c.n + t];
  const uint32_t heads = a.s.H + 2 * a.s.G, d = 4 * (tid % LP), h0 = blockIdx.y * HPB + tid / LP;
  const float* src = a.qkv + (size_t(b) * a.c.n + t) * heads * HD;
  float4 x = *reinterpret_cast<const float4*>(src + size_t(min(h0, heads - 1)) * HD + d);
  const double freq = a.s.freq[tid % (HD / 2)];
  const Request r = checked(a.c, raw, tid == 0 && t == 0 && blockIdx.y == 0 ? a.s.err : nullptr);
  if (t >= r.fresh) return;
  const uint32_t slot = r.len - r.fresh + t;
  if (pos < 0) {
    if (tid == 0 && blockIdx.y == 0) atomicOr(a.s.err, S2HIP_KV_ERR_POSITION);
    return;
  }
  if (tid < HD / 2) {
    const double angle = double(pos) * freq * 0.15915494309189535;  // in turns
    const double rest = angle - rint(angle);
    const float part = float(rest), more = 6.2831853f * float(rest - double(part));  // (what f32 loses of the angle, in radians)
    float sn, cs;
    sincospif(2.0f * part, &sn, &cs);
    turn[tid] = make_float2(fmaf(-sn, more, cs), fmaf(cs, more, sn));
  }
  __syncthreads();
  for (uint32_t h = h0; h < heads;) {  // whole rows of 16 lanes take part
    const uint32_t next = h + HPB * gridDim.y;
    const float4 ahead = *reinterpret_cast<const float4*>(src + size_t(min(next, heads - 1)) * HD + d);
    if (h < a.s.H + a.s.G) {
      if (a.q_norm) {
        float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
        ss = row_reduce(ss, [](float p, float q) { return p + q; });
        if constexpr (LP == 32) ss += __shfl_xor(ss, 16, 64);
        const float mean = ss * (1.0f / HD) + a.s.eps, near = rsqrtf(mean), step = fmaf(-mean * near, near, 1.0f);
        const float f = step == step ? fmaf(0.5f * near, step, near) : near;  // (mean 0 or infinite)
        const float4 gain = *reinterpret_cast<const float4*>((h < a.s.H ? a.q_norm : a.k_norm) + d);
        x = make_float4(x.x * f * gain.x, x.y * f * gain.y, x.z * f * gain.z, x.w * f * gain.w);
      }
      const float2 t0 = turn[d / 2], t1 = turn[d / 2 + 1];
      x = make_float4(x.x * t0.x - x.y * t0.y, x.x * t0.y + x.y * t0.x, x.z * t1.x - x.w * t1.y, x.z * t1.y + x.w * t1.x);
    }
    if (h < a.s.H) {
      *reinterpret_cast<float4*>(a.q_out + ((size_t(b) * a.c.n + t) * a.s.H + h) * HD + d) = x;
    } else {
      const bool key = h < a.s.H + a.s.G;
      const uint32_t g = key ? h - a.s.H : h - a.s.H - a.s.G;
      Elem<KH>* dst = static_cast<Elem<KH>*>(key ? a.c.k : a.c.v) + b * a.c.req_stride + g * a.c.head_stride + slot * a.c.slot_stride + d;
      if constexpr (KH) {
        const half4 y = {_Float16(x.x), _Float16(x.y), _Float16(x.z), _Float16(x.w)};
        const float big = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
        if (big >= 65520.0f) atomicOr(a.s.err, S2HIP_KV_ERR_F16_RANGE);  // rounds to infinity
        *reinterpret_cast<half4*>(dst) = y;
      } else {
        *reinterpret_cast<float4*>(dst) = x;
      }
      if (!key && tid % LP == 0) {
        const size_t at = (size_t(b) * a.s.G + g) * a.c.cap + slot;
        if (a.scores) a.scores[at] = 0.0f;
        if (a.slot_positions) a.slot_positions[at] = pos;
      }
    }
    x = ahead;
    h = next;
  }
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// Scores are kept in powers of two (q times scale log2(e)), so that a weight is
// one exp2 of a difference.  A kv head's query rows are packed: row (b n + t)
// rep + r.  A row's softmax state is (m, l, o): weights 2^(s - m), their sum and
// their sum with the values; states over disjoint keys join by their m.

// m follows a row's maximum only when it is SLACK behind: weights stay below
// 2^SLACK and the o registers are hardly ever rescaled.  It is a whole number, so
// that taking it off and the factors between states round nothing, and each row's
// goes by the keys that the row sees alone.  f16 parts of
// weights are of 2^(s - m + F16_LIFT), up to 2^14: the lo part of a small weight is
// exact to 2^-25, 2^-31 of the largest.  The o of f32 values leave (and in
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

// The own caches that `n_rows` packed rows from row0 on attend to, in tiles of KT
// keys, each as far as the last of the rows sees.  Lane j holds request b_lo + j
// (at most 64 requests).
struct Run {
  uint32_t b_lo, tiles;
  Request rq;         // the lane's request
  uint32_t seg_keys;  // keys of it
  uint32_t seg_end;   // its last tile + 1
};
__device__ __forceinline__ RawRequest load_requests(const KvAttendArgs& a, uint32_t row0) {
  return load_request(a.c, min(row0 / (a.c.n * a.s.rep) + (threadIdx.x & 63u), a.c.R - 1));
}
template <int KT>
__device__ __forceinline__ Run run_of(const KvAttendArgs& a, uint32_t row0, uint32_t n_rows, RawRequest raw, uint32_t* err) {
  const uint32_t lane = threadIdx.x & 63u, per = a.c.n * a.s.rep, row1 = min(row0 + n_rows, a.c.R * per);
  Run r{};
  r.b_lo = row0 / per;
  const uint32_t b = r.b_lo + lane;
  if (b <= (row1 - 1) / per) {
    r.rq = checked(a.c, raw, err);
    const uint32_t first = max(row0, b * per) - b * per, last = min(row1, (b + 1) * per) - 1 - b * per;
    if (first / a.s.rep < r.rq.fresh) r.seg_keys = r.rq.len - r.rq.fresh + min(last / a.s.rep, r.rq.fresh - 1) + 1;
  }
  r.seg_end = wave_scan((r.seg_keys + KT - 1) / KT);
  r.tiles = lane_read_u32(r.seg_end, 63);
  return r;
}

// A tile of keys: where its rows are and whose they are.
template <class T>
struct Where {
  const T* k;
  const T* v;
  size_t stride;
  uint32_t key0, keys;
  int seg;  // -1: the prefix; else request b_lo + seg
};
template <class T, int KT>
__device__ __forceinline__ Where<T> prefix_tile(const KvCaches& c, uint32_t g, uint32_t i) {
  Where<T> w;
  w.seg = -1;
  w.key0 = i * KT;
  w.keys = min(uint32_t(KT), c.P - w.key0);
  w.stride = c.p_slot_stride;
  const size_t at = g * c.p_head_stride + w.key0 * w.stride;
  w.k = static_cast<const T*>(c.pk) + at;
  w.v = static_cast<const T*>(c.pv) + at;
  return w;
}
// tile i of the run; `seg` goes up with i
template <class T, int KT>
__device__ __forceinline__ Where<T> own_tile(const KvCaches& c, const Run& r, uint32_t g, uint32_t i, uint32_t& seg) {
  Where<T> w;
  while (i >= lane_read_u32(r.seg_end, int(seg))) ++seg;
  const uint32_t begin = seg ? lane_read_u32(r.seg_end, int(seg) - 1) : 0u;
  w.seg = int(seg);
  w.key0 = (i - begin) * KT;
  w.keys = min(uint32_t(KT), lane_read_u32(r.seg_keys, int(seg)) - w.key0);
  w.stride = c.slot_stride;
  const size_t at = (r.b_lo + seg) * c.req_stride + g * c.head_stride + w.key0 * w.stride;
  w.k = static_cast<const T*>(c.k) + at;
  w.v = static_cast<const T*>(c.v) + at;
  return w;
}

// Few rows over many keys (decode steps).  A wave owns 16 packed rows of a kv
// head and a run of key tiles out of the shared prefix followed by the own
// caches of the rows' requests; nothing is exchanged between waves before the
// end, when the block's four join their states in LDS and, with several blocks
// per 16 rows, leave them for kv_join_kernel.
//   Scores transposed, S^T = K Q^T, so a lane holds one row (lane % 16) and some
// of the tile's keys, and the weights are the B operand of O^T += V^T P^T as
// they stand in the registers.
//   f32 caches: v_mfma_f32_16x16x4_f32 (f32 products and sums, 16 keys a tile).
// It takes one element per lane and step, so K and V go from memory to the
// operand registers by 16-byte loads in an order of dims of our own choosing.
//   f16 caches: v_mfma_f32_16x16x32_f16, 32 keys a tile, q and the weights as
// hi + lo f16 parts (2^-22 of a row's largest q, 2^-22 of a weight; weights are
// lifted by F16_LIFT so that small ones keep their lo part); K from memory to
// registers, V through the wave's own 32 rows of LDS, read transposed.
//   What a row must not see: scores by select; where a tile that some row does
// not see in whole holds values that are no number (0 x NaN), they count as 0 in
// the product, and a second product of marks, theirs with the keys each row
// sees, says which outputs are no number.
//   Bound by latency, then by memory: 8 requests over 1500 shared and 512 own
// slots, f32, take 12.7 us, 6 of them start and end (3 to the requests' lengths
// and the first keys, 3 the joining in LDS), the rest 39 MB; 16 over 24001 + 2000,
// f16, 55 us (49 where the last-level cache still holds the keys): 200 MB from
// memory, 520 MB (9.5 TB/s) past the second-level cache, for four row tiles read
// the prefix.  Two row tiles a wave, which halve that,
// take 8 % off this call and put 10 to 60 % on shorter ones.
constexpr int STEP_WAVES = 4;

template <int HD, bool KH>
__global__ __launch_bounds__(64 * STEP_WAVES, 2) void kv_step_kernel(KvAttendArgs a, KvSplit sp, float* stat, KvScores keep) {
  using T = Elem<KH>;
  constexpr int KT = KH ? 32 : 16;
  constexpr int OT = HD / 16;                 // 16 x 16 output tiles
  constexpr int KL = HD * sizeof(T) / 64;     // 16-byte loads of a key row per lane
  constexpr int OP = HD + 4;                  // padded row of the joined states
  constexpr float LIFT = KH ? F16_LIFT : 0.0f;
  constexpr uint32_t VB = KT * HD * 2;        // bytes of a wave's value tile in LDS
  constexpr uint32_t JOIN = STEP_WAVES * 16 * OP * 4;
  constexpr uint32_t LDS = KH && STEP_WAVES * VB > JOIN ? STEP_WAVES * VB : JOIN;
  __shared__ __align__(16) uint8_t lds[LDS];
  __shared__ float ml[STEP_WAVES][16][2];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), r16 = lane & 15u, q4 = lane >> 4;
  const uint32_t g = blockIdx.x % a.s.G, rest = blockIdx.x / a.s.G, tile = rest % sp.tiles, split = rest / sp.tiles;
  const uint32_t per = a.c.n * a.s.rep, rows = a.c.R * per;

  // what needs nothing first: the requests, the row's query, the wave's first tile of the prefix
  const RawRequest raw = load_requests(a, tile * 16);
  const uint32_t row = min(tile * 16 + r16, rows - 1), b_row = row / per, t_row = row / a.s.rep % a.c.n, h_row = g * a.s.rep + row % a.s.rep;
  const size_t q_at = ((size_t(b_row) * a.c.n + t_row) * a.s.H + h_row) * HD;
  float4 qx[HD / 16];  // f32: dims 16 j + 4 q4 ..; f16: dims 32 (j / 2) + 8 q4 + 4 (j % 2) ..
#pragma unroll
  for (int j = 0; j < HD / 16; ++j)
    qx[j] = *reinterpret_cast<const float4*>(a.q + q_at + (KH ? 32 * (j / 2) + 8 * q4 + 4 * (j % 2) : 16 * j + 4 * q4));
  const uint32_t lots = sp.splits * STEP_WAVES, lot = split * STEP_WAVES + wave;
  const uint32_t p_tiles = (a.c.P + KT - 1) / KT;
  const uint32_t p_lo = p_tiles * lot / lots, n_pre = p_tiles * (lot + 1) / lots - p_lo;
  // f32: K key r16, dims 16 j + 4 q4 ..; V key 4 q4 + i, dims 64 hh + 4 r16 ..
  // f16: K key 16 kt + r16, dims 32 j + 8 q4 ..; V 16-byte pieces lane + 64 i of the tile
  u32x4 kr[KH ? 2 : 1][KL], vr[KH ? HD / 16 : 4][KH ? 1 : HD / 64];
  // (offsets in 32 bits from a uniform base: 64-bit products per row took a quarter of a tile's vector cycles)
  auto load_k = [&](const Where<T>& w) {
    const uint8_t* base = reinterpret_cast<const uint8_t*>(w.k);
    const uint32_t stride = uint32_t(w.stride) * sizeof(T);
#pragma unroll
    for (int kt = 0; kt < (KH ? 2 : 1); ++kt) {
      const uint32_t off = min(16u * kt + r16, w.keys - 1) * stride + 16 * q4;
#pragma unroll
      for (int j = 0; j < KL; ++j) kr[kt][j] = *reinterpret_cast<const u32x4*>(base + (off + 64 * j));
    }
  };
  auto load_v = [&](const Where<T>& w) {
    const uint8_t* base = reinterpret_cast<const uint8_t*>(w.v);
    const uint32_t stride = uint32_t(w.stride) * sizeof(T);
    if constexpr (KH) {
      constexpr uint32_t PR = HD / 8;  // pieces per row
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        const uint32_t p = lane + 64 * i;
        vr[i][0] = *reinterpret_cast<const u32x4*>(base + (min(p / PR, w.keys - 1) * stride + (p % PR) * 16));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t off = min(4 * q4 + i, w.keys - 1) * stride + 16 * r16;
#pragma unroll
        for (int hh = 0; hh < HD / 64; ++hh) vr[i][hh] = *reinterpret_cast<const u32x4*>(base + (off + 256 * hh));
      }
    }
  };

  // (Loads stand on one path wherever they can: behind a branch the compiler waits for all that may be in flight.
  // Where there is nothing to load, a row that is there anyway is read again.)
  Where<T> w{static_cast<const T*>(a.c.k) + g * a.c.head_stride, static_cast<const T*>(a.c.v) + g * a.c.head_stride, 0, 0, 1, -1};
  if (n_pre) w = prefix_tile<T, KT>(a.c, g, p_lo);
  load_k(w);
  load_v(w);
  const Run run = run_of<KT>(a, tile * 16, 16, raw, g == 0 && split == 0 && wave == 0 ? a.s.err : nullptr);
  const uint32_t b_lo = run.b_lo;
  // (the own tiles the other way round: the waves with one more of the prefix get one fewer)
  const uint32_t o_lo = run.tiles * (lots - 1 - lot) / lots, n_tiles = n_pre + run.tiles * (lots - lot) / lots - o_lo;
  uint32_t seg = 0;
  if (n_pre == 0 && n_tiles) {
    w = own_tile<T, KT>(a.c, run, g, o_lo, seg);
    load_k(w);
    load_v(w);
  }

  // this lane's row
  const uint32_t len_row = __shfl(run.rq.len, int(b_row - b_lo) & 15, 64), fresh_row = __shfl(run.rq.fresh, int(b_row - b_lo) & 15, 64);
  const bool live = tile * 16 + r16 < rows && t_row < fresh_row;
  const int own_limit = live ? int(len_row - fresh_row + t_row) : -1;
  float qf[KH ? 1 : HD / 4];                                       // f32: dims 16 j + 4 q4 + c
  half8 qh[KH ? HD / 32 : 1], ql[KH ? HD / 32 : 1];                // f16: dims 32 j + 8 q4 + e
  float unscale = 1.0f;
  {
    const float s2 = live ? a.s.scale2 : 0.0f;
    float x[HD / 16][4], big = 0.0f;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) {
      x[j][0] = live ? qx[j].x * s2 : 0.0f;  // (a query of no token may hold anything)
      x[j][1] = live ? qx[j].y * s2 : 0.0f;
      x[j][2] = live ? qx[j].z * s2 : 0.0f;
      x[j][3] = live ? qx[j].w * s2 : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(x[j][e]));
    }
    if constexpr (!KH) {
#pragma unroll
      for (int j = 0; j < HD / 4; ++j) qf[j] = x[j / 4][j % 4];
    } else {
      float inv;
      pow2_scale(quarter_max(big), unscale, inv);
#pragma unroll
      for (int j = 0; j < HD / 32; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Parts y = split_query<true>(x[2 * j + e / 4][e % 4] * inv);
          qh[j][e] = y.hi;
          ql[j][e] = y.lo;
        }
    }
  }

  // f32: o[4 hh + c][j]: dim 64 hh + 16 q4 + 4 j + c; f16: o[dt][j]: dim 16 dt + 4 q4 + j
  floatx4 o[OT];
#pragma unroll
  for (int i = 0; i < OT; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.0f;
  lds_byte* v_lds = (lds_byte*)lds + (KH ? wave * VB : 0u);
  // 16-byte piece p of row `key` stands at piece p ^ swz(key): the 16 rows that a transposed read takes 32 bytes
  // of then lie in distinct banks
  auto swz = [](uint32_t key) { return HD == 128 ? 2 * (key & 7u) : 2 * ((key >> 1) & 3u); };

  for (uint32_t i = 0; i < n_tiles; ++i) {
    const bool more = i + 1 < n_tiles;
    Where<T> next = w;
    next.stride = 0;
    if (more) next = i + 1 < n_pre ? prefix_tile<T, KT>(a.c, g, p_lo + i + 1) : own_tile<T, KT>(a.c, run, g, o_lo + (i + 1 - n_pre), seg);
    constexpr int NS = KH ? 8 : 4;  // scores per lane
    float s[NS];
    if constexpr (KH) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        floatx4 hi = floatx4{0.f, 0.f, 0.f, 0.f}, lo = hi;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          const half8 k8 = __builtin_bit_cast(half8, kr[kt][j]);
          hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qh[j], hi, 0, 0, 0);
          lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[j], lo, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) s[4 * kt + c] = (hi[c] + lo[c]) * unscale;
      }
    } else {
      floatx4 x = floatx4{0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
      for (int j = 0; j < HD / 16; ++j) {
        const floatx4 k4 = __builtin_bit_cast(floatx4, kr[0][j]);
        x = __builtin_amdgcn_mfma_f32_16x16x4f32(k4[0], qf[4 * j], x, 0, 0, 0);
        y = __builtin_amdgcn_mfma_f32_16x16x4f32(k4[1], qf[4 * j + 1], y, 0, 0, 0);
        x = __builtin_amdgcn_mfma_f32_16x16x4f32(k4[2], qf[4 * j + 2], x, 0, 0, 0);
        y = __builtin_amdgcn_mfma_f32_16x16x4f32(k4[3], qf[4 * j + 3], y, 0, 0, 0);
      }
      float z = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[c] = x[c] + y[c];
        z = fmaf(s[c], 0.0f, z);
      }
      if (__any(!(z == 0.0f))) {  // keys that hold an infinity make theirs no number, whichever its sign (not so a sum beyond f32)
        float big = 0.0f;
#pragma unroll
        for (int j = 0; j < KL; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(__uint_as_float(kr[0][j][e])));
        big = quarter_max(big);  // of key r16
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (__shfl(big, int(4 * q4) + c, 64) == INFINITY) s[c] = NAN;
      }
    }
    if constexpr (KH) {  // the values go to LDS, their registers take the next tile's
      constexpr uint32_t PR = HD / 8;
      asm volatile("" ::: "memory");
#pragma unroll
      for (int p = 0; p < HD / 16; ++p) {
        const uint32_t x = lane + 64 * p, key = x / PR, piece = x % PR;
        *reinterpret_cast<u32x4*>(lds + wave * VB + key * (HD * 2) + (piece ^ swz(key)) * 16) = vr[p][0];
      }
    }
    load_k(next);
    const int limit = w.seg < 0 ? int(a.c.P) - 1 : int(b_row - b_lo) == w.seg ? own_limit : -1;
    // rows that see the whole tile: nothing to mask
    const bool whole = __all(limit >= int(w.key0 + KT - 1));
    if (!whole) {
#pragma unroll
      for (int c = 0; c < NS; ++c) {
        const int key = int(w.key0 + 16u * (c / 4) + 4u * q4 + (c % 4));
        if (key > limit) s[c] = -INFINITY;
      }
    }
    if (keep.own && (w.seg >= 0 || keep.prefix)) {
      float* dst = w.seg < 0 ? keep.prefix + (size_t(g) * a.c.P + w.key0) * rows + row
                             : keep.own + ((size_t(b_row) * a.s.G + g) * a.c.cap + w.key0) * per + (row - b_row * per);
      const uint32_t step = w.seg < 0 ? rows : per;
#pragma unroll
      for (int c = 0; c < NS; ++c) {
        const uint32_t key = 16u * (c / 4) + 4u * q4 + (c % 4);
        if (live && int(w.key0 + key) <= limit) dst[key * step] = s[c];
      }
    }
    float top = s[0];
#pragma unroll
    for (int c = 1; c < NS; ++c) top = fmaxf(top, s[c]);
    const float mn = fmaxf(m, quarter_max(top));
    const bool up = mn > m + SLACK;
    if (__any(up)) {
      const float to = up ? floorf(mn) : m, f = up ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
#pragma unroll
      for (int c = 0; c < OT; ++c) o[c] *= f;
      l *= f;
      m = to;
    }
    const float base = (m == -INFINITY ? 0.0f : m) - LIFT;
#pragma unroll
    for (int c = 0; c < NS; ++c) {
      s[c] = __builtin_amdgcn_exp2f(s[c] - base);
      l += s[c];
      if constexpr (!KH) s[c] *= F32_DOWN;
    }
    bool odd = false;  // a value that is no number, and rows that must not see it
    if constexpr (KH) {
      half8 ph, pl;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float hi = __uint_as_float(__float_as_uint(s[c]) & 0xffffe000u);  // the upper 11 bits, and the rest
        ph[c] = _Float16(hi);
        pl[c] = _Float16(s[c] - hi);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      half8 v8[OT];
#pragma unroll
      for (int dt = 0; dt < OT; ++dt) {
        half4 part[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const uint32_t key = 16 * kt + 4 * q4 + r16 / 4, byte = 32 * dt + 8 * (r16 & 3u);
          part[kt] = read_tr(v_lds + key * (HD * 2) + (((byte >> 4) ^ swz(key)) << 4) + (byte & 15u));
        }
        v8[dt] = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
      }
      if (!whole && w.seg >= 0) {
        half8 z = half8{};
#pragma unroll
        for (int dt = 0; dt < OT; ++dt) z = __builtin_elementwise_fma(v8[dt], half8{}, z);
        odd = __any(not_zero(z));
      }
      if (odd) {
        half8 seen;
#pragma unroll
        for (int c = 0; c < 8; ++c) seen[c] = int(w.key0 + 16u * (c / 4) + 4u * q4 + (c % 4)) <= limit ? _Float16(1) : _Float16(0);
#pragma unroll
        for (int dt = 0; dt < OT; ++dt) {
          const half8 marks = take_odd(v8[dt]);
          const floatx4 hits = __builtin_amdgcn_mfma_f32_16x16x32_f16(marks, seen, floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
          for (int c = 0; c < 4; ++c) o[dt][c] = hits[c] > 0.0f ? NAN : o[dt][c];
        }
      }
#pragma unroll
      for (int dt = 0; dt < OT; ++dt) {
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8[dt], ph, o[dt], 0, 0, 0);
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8[dt], pl, o[dt], 0, 0, 0);
      }
    } else {
      if (!whole && w.seg >= 0) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int hh = 0; hh < HD / 64; ++hh) {
            const floatx4 v4 = __builtin_bit_cast(floatx4, vr[i][hh]);
#pragma unroll
            for (int c = 0; c < 4; ++c) z = fmaf(v4[c], 0.0f, z);
          }
        odd = __any(!(z == 0.0f));
      }
      if (odd) {
#pragma unroll
        for (int hh = 0; hh < HD / 64; ++hh)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            floatx4 hits = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool bad = !(fabsf(__uint_as_float(vr[i][hh][c])) < INFINITY);
              if (bad) vr[i][hh][c] = 0;
              hits = __builtin_amdgcn_mfma_f32_16x16x4f32(bad ? 1.0f : 0.0f, int(w.key0 + 4 * q4 + i) <= limit ? 1.0f : 0.0f, hits, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) o[4 * hh + c][j] = hits[j] > 0.0f ? NAN : o[4 * hh + c][j];
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int hh = 0; hh < HD / 64; ++hh) {
          const floatx4 v4 = __builtin_bit_cast(floatx4, vr[i][hh]);
#pragma unroll
          for (int c = 0; c < 4; ++c) o[4 * hh + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v4[c], s[i], o[4 * hh + c], 0, 0, 0);
        }
    }
    load_v(next);
    w = next;
  }

  // the block's four states as one
  l = quarter_sum(l);
  if (q4 == 0) {
    ml[wave][r16][0] = m;
    ml[wave][r16][1] = l;
  }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int i = 0; i < STEP_WAVES; ++i) M = fmaxf(M, ml[i][r16][0]);
  const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
  float* os = reinterpret_cast<float*>(lds) + (wave * 16 + r16) * OP;
#pragma unroll
  for (int c = 0; c < OT; ++c) {
    if constexpr (KH) {
      *reinterpret_cast<floatx4*>(os + 16 * c + 4 * q4) = o[c] * f;
    } else {
      const int hh = c / 4, j = c % 4;
      *reinterpret_cast<floatx4*>(os + 64 * hh + 16 * q4 + 4 * j) =
          floatx4{o[4 * hh][j] * f, o[4 * hh + 1][j] * f, o[4 * hh + 2][j] * f, o[4 * hh + 3][j] * f};
    }
  }
  __syncthreads();
  const uint32_t jr = tid / 16, d0 = tid % 16 * 4;  // a row per 16 threads
  const uint32_t out_row = tile * 16 + jr;
  float M_row = -INFINITY, L_row = 0.0f;
#pragma unroll
  for (int i = 0; i < STEP_WAVES; ++i) M_row = fmaxf(M_row, ml[i][jr][0]);
  const float M_base = M_row == -INFINITY ? 0.0f : M_row;  // (then every l is 0, or no number)
#pragma unroll
  for (int i = 0; i < STEP_WAVES; ++i) L_row = fmaf(ml[i][jr][1], __builtin_amdgcn_exp2f(ml[i][jr][0] - M_base), L_row);
  const size_t part = ((size_t(g) * sp.tiles + tile) * sp.splits + split) * 16 + jr;
  const bool last = sp.splits == 1;
  const uint32_t ob = out_row / per, ot = out_row / a.s.rep % a.c.n, oh = g * a.s.rep + out_row % a.s.rep;
  const bool out_live = out_row < rows && ot < __shfl(run.rq.fresh, int(ob - b_lo) & 15, 64);
  if (last && !out_live) return;
  float* dst = last ? a.out + ((size_t(ob) * a.c.n + ot) * a.s.H + oh) * HD : sp.o + part * HD;
  const float inv = last ? (M_row == -INFINITY ? NAN : (KH ? 1.0f : F32_UP) / L_row) : 1.0f;  // (it sees a key, its own)
#pragma unroll
  for (int c = 0; c < HD / 64; ++c) {
    const float* src = reinterpret_cast<const float*>(lds) + jr * OP + d0 + 64 * c;
    floatx4 x = *reinterpret_cast<const floatx4*>(src);
#pragma unroll
    for (int i = 1; i < STEP_WAVES; ++i) x += *reinterpret_cast<const floatx4*>(src + i * 16 * OP);
    *reinterpret_cast<floatx4*>(dst + d0 + 64 * c) = x * inv;
  }
  if (tid % 16 == 0) {
    float* st = last ? stat + 2 * ((size_t(ob) * a.c.n + ot) * a.s.H + oh) : sp.ml + 2 * part;
    if (!last || stat) {
      st[0] = M_row - LIFT;
      st[1] = L_row;
    }
  }
}

// Many rows (turns, prompts).  A block of four waves owns 128 packed rows of a
// kv head, 32 per wave, and walks the run of key tiles (64 keys of f16, 32 of
// f32) that they share through LDS, the next tile's loads in flight meanwhile.
//   v_mfma_f32_32x32x16_f16 with S^T = K Q^T and O^T += V^T P^T as above: a lane
// holds one row (lane % 32).  q and the weights are hi + lo f16 parts, f16
// caches as they are: two products each.
//   f32 caches: keys and values are split into hi + lo f16 parts as they are
// staged, each key's and each value's row scaled by a power of two of its own:
// three products, 2^-22 of each term, or 2^-39 of the largest of its row.  A row
// of o is in units of the largest value row that it has seen, so a term far below
// is exact to 2^-39 of that.  No scale is shared with what a row does not see (one
// for 8 keys, or for the rows of a wave, would let a later token's large value
// take the low bits off the earlier ones').  (The f32 matrix instructions do a
// sixteenth of the f16 ones' work per cycle.)
//   8 requests x 250 tokens over 1500 + 250 slots, f16, take 104 us (0.85 PFLOP/s of
// hi + lo products), the matrix units busy for 34 % of it and the vector ones for
// 26 %: a wave's products and its softmax follow one another, and the two blocks of a
// CU do not fill each other's gaps.  2048 tokens over 6000, 430 us (1.1 PFLOP/s), keep
// the matrix units busy for 61 % at the 1.66 GHz that the clock falls to; a library's
// f16 product of 8192^3 reaches 1.2 to 1.3.  f32, 3 x 37 over 1001 + 131: 27 us, of
// which a tile of 32 keys takes 2.2, a third of it products: blocks are too few to
// hide the splitting.  A prompt of 1500 tokens, f32: 104 us, 34 % vector and 23 %
// matrix cycles.
constexpr int TILE_ROWS = 128;
constexpr float NO_STATE = -1.0f;  // in the place of l: no state here
constexpr int NO_UNIT = -1000;     // of a row that has seen no value

template <int HD, bool KH>
__global__ __launch_bounds__(256, 2) void kv_tile_kernel(KvAttendArgs a, KvSplit sp, float* stat) {
  using T = Elem<KH>;
  constexpr int KT = KH ? 64 : 32, NSUB = KT / 32;
  constexpr int DS = HD / 16, DT = HD / 32;
  constexpr uint32_t RB = HD * 2, PLANE = KT * RB;        // bytes of a row and of a plane of a tile in LDS
  constexpr uint32_t BUF = (KH ? 2 : 4) * PLANE;          // K, V, or K hi, K lo, V hi, V lo
  constexpr int LD = KT * HD * sizeof(T) / 16 / 256;      // 16-byte loads per thread of a tile's keys
  constexpr uint32_t PR = HD * sizeof(T) / 16;            // 16-byte pieces of a row in memory
  constexpr float LIFT = F16_LIFT;
  __shared__ __align__(16) uint8_t lds[2 * BUF];
  __shared__ __align__(16) float k_scale[2][32];  // f32: [buffer][key], powers of two
  __shared__ __align__(16) int v_exp[2][32];      // f32: the values' scales, by their exponents
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), r32 = lane & 31u, h2 = lane >> 5;
  const uint32_t g = blockIdx.x % a.s.G, rest = blockIdx.x / a.s.G;
  const uint32_t blocks = (a.c.R * a.c.n * a.s.rep + TILE_ROWS - 1) / TILE_ROWS;
  const uint32_t tile = blocks - 1 - rest % blocks, split = rest / blocks;  // later rows see more keys: they go first
  const uint32_t per = a.c.n * a.s.rep, rows = a.c.R * per;
  // what needs nothing first: the requests, the row's query and, where it is known, the first tile of the prefix
  const RawRequest raw = load_requests(a, tile * TILE_ROWS);
  const uint32_t at = tile * TILE_ROWS + wave * 32 + r32, row = min(at, rows - 1);
  const uint32_t b_row = row / per, t_row = row / a.s.rep % a.c.n, h_row = g * a.s.rep + row % a.s.rep;
  const size_t at_row = (size_t(b_row) * a.c.n + t_row) * a.s.H + h_row;
  float4 qx[DS][2];  // dims 16 ks + 8 h2 ..
#pragma unroll
  for (int ks = 0; ks < DS; ++ks)
#pragma unroll
    for (int e = 0; e < 2; ++e) qx[ks][e] = *reinterpret_cast<const float4*>(a.q + at_row * HD + 16 * ks + 8 * h2 + 4 * e);

  // f32: eight threads per key, 128 bytes of the row per load, in an order that keeps the writes to LDS of neighbouring
  // keys in distinct banks
  u32x4 kr[KH ? 1 : LD], vr[KH ? 1 : LD];
  const uint32_t key_f32 = 8 * wave + lane / 8;
  auto piece_of = [&](int which, int i) {
    uint32_t turn = HD == 128 ? (which ? 0u : key_f32 & 3u) : (which ? key_f32 : key_f32 ^ (key_f32 >> 1)) & 1u;
    if (HD == 128 && !which) asm volatile("" : "+v"(turn));  // (worked out where it is used: addresses kept for the loop cost registers)
    return lane % 8 + 8 * (uint32_t(i) ^ turn);
  };
  // 16-byte piece p of row `key` stands at p ^ swz(key): keys' fragment reads take one piece of 8 rows in a row,
  // transposed value reads 64 bytes of 4 rows
  auto k_at = [](uint32_t key, uint32_t piece) { return key * RB + ((piece ^ (key & 7u)) << 4); };
  auto v_at = [](uint32_t key, uint32_t piece) { return key * RB + ((piece ^ (HD == 128 ? 4 * (key & 3u) : 4 * ((key >> 1) & 1u))) << 4); };
  // f16: straight to LDS, a KiB per wave and load, each lane bringing the piece that belongs where its 16 bytes go;
  // f32: to registers, and to LDS once the other tile is done with
  const uint32_t lds0 = uint32_t(uintptr_t((lds_byte*)lds));
  auto load = [&](const Where<T>& w, uint32_t buf) {
    const uint8_t *k = reinterpret_cast<const uint8_t*>(w.k), *v = reinterpret_cast<const uint8_t*>(w.v);
    const uint32_t stride = uint32_t(w.stride) * sizeof(T);
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const uint32_t x = (wave * LD + i) * 1024 + lane * 16, key = x / RB, off = min(key, w.keys - 1) * stride;
      dma16(k, off + (k_at(key, x / 16 % PR) & (RB - 1)), lds0 + buf * BUF + (wave * LD + i) * 1024);
      dma16(v, off + (v_at(key, x / 16 % PR) & (RB - 1)), lds0 + buf * BUF + PLANE + (wave * LD + i) * 1024);
    }
  };
  auto load_f32 = [&](const Where<T>& w, const T* from, int which, u32x4* r) {
    const uint8_t* src = reinterpret_cast<const uint8_t*>(from);
    const uint32_t off = min(key_f32, w.keys - 1) * (uint32_t(w.stride) * uint32_t(sizeof(T)));
#pragma unroll
    for (int i = 0; i < LD; ++i) r[i] = *reinterpret_cast<const u32x4*>(src + (off + piece_of(which, i) * 16));
  };
  auto store_f32 = [&](uint32_t buf, int which, const u32x4* r) {
    uint8_t* base = lds + buf * BUF;
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const floatx4 x = __builtin_bit_cast(floatx4, r[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(x[e]));
    }
    if (__any(!(big < INFINITY))) {  // the largest number, then
      big = 0.0f;
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        const floatx4 x = __builtin_bit_cast(floatx4, r[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.0f);
      }
    }
    big = fmaxf(big, dpp_f32<DPP_QUAD_XOR1>(big));
    big = fmaxf(big, dpp_f32<DPP_QUAD_XOR2>(big));
    big = fmaxf(big, dpp_f32<DPP_ROW_HALF_MIRROR>(big));
    float scale, inv;
    if (which)
      pow2_scale<-85>(big, scale, inv);
    else
      pow2_scale(big, scale, inv);
    if (lane % 8 == 0) {
      if (which)
        v_exp[buf][key_f32] = int(__float_as_uint(scale) >> 23) - 127;
      else
        k_scale[buf][key_f32] = scale;
    }
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const floatx4 x = __builtin_bit_cast(floatx4, r[i]) * inv;
      const half4 hi = __builtin_convertvector(x, half4);
      const half4 lo = __builtin_convertvector(x - __builtin_convertvector(hi, floatx4), half4);
      const uint32_t p = piece_of(which, i), off = (which ? v_at(key_f32, p / 2) : k_at(key_f32, p / 2)) + 8 * (p % 2);
      *reinterpret_cast<half4*>(base + 2 * which * PLANE + off) = hi;
      *reinterpret_cast<half4*>(base + (2 * which + 1) * PLANE + off) = lo;
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto load_first = [&](const Where<T>& w) {
    if constexpr (KH) {
      load(w, 0);
    } else {
      load_f32(w, w.k, 0, kr);
      load_f32(w, w.v, 1, vr);
    }
  };

  // The splits of a row tile share its prefix and its own tiles apart, the own ones the other way round; with
  // sp.least there are only as many splits as it has that many tiles, and they share the run as a whole.
  const bool whole_run = sp.least != 0;
  const uint32_t p_all = (a.c.P + KT - 1) / KT;
  uint32_t p_lo = whole_run ? 0u : p_all * split / sp.splits, n_pre = whole_run ? (split ? 0u : p_all) : p_all * (split + 1) / sp.splits - p_lo;
  const bool early = n_pre != 0;
  if (early) load_first(prefix_tile<T, KT>(a.c, g, p_lo));
  const Run run = run_of<KT>(a, tile * TILE_ROWS, TILE_ROWS, raw, g == 0 && split == 0 && wave == 0 ? a.s.err : nullptr);
  uint32_t splits = sp.splits, o_lo = run.tiles * (splits - 1 - split) / splits, n_tiles = n_pre + run.tiles * (splits - split) / splits - o_lo;
  if (whole_run) {
    const uint32_t total = p_all + run.tiles;
    splits = min(splits, (total + sp.least - 1) / sp.least);
    const uint32_t lo = total * split / splits, hi = total * (split + 1) / splits;
    p_lo = min(lo, p_all);
    n_pre = min(hi, p_all) - p_lo;
    o_lo = max(lo, p_all) - p_all;
    n_tiles = hi - lo;
    if (sp.splits > 1 && run.tiles && (split >= splits || splits == 1)) {  // no state here: say so in its place
      const uint32_t r = tile * TILE_ROWS + tid;
      if (tid < TILE_ROWS && r < rows) sp.ml[2 * (((size_t(g) * sp.tiles + r / 16) * sp.splits + split) * 16 + r % 16) + 1] = NO_STATE;
    }
  }
  if (run.tiles == 0 || split >= splits) {  // no row of a token, or no share of them
    if constexpr (KH) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (loads to LDS end before the block does)
    return;
  }

  // this lane's row
  const uint32_t len_row = __shfl(run.rq.len, int(b_row - run.b_lo) & 63, 64), fresh_row = __shfl(run.rq.fresh, int(b_row - run.b_lo) & 63, 64);
  const bool live = at < rows && t_row < fresh_row;
  const uint32_t own_rows = live ? (b_row - run.b_lo) << 16 | (len_row - fresh_row + t_row) : 0u;  // segment, last slot seen
  half8 qh[DS], ql[DS];  // dims 16 ks + 8 h2 + e
  float unscale;
  {
    float big = 0.0f;
#pragma unroll
    for (int ks = 0; ks < DS; ++ks)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float4& y = qx[ks][e];
        y = live ? make_float4(y.x * a.s.scale2, y.y * a.s.scale2, y.z * a.s.scale2, y.w * a.s.scale2) : make_float4(0.f, 0.f, 0.f, 0.f);
        big = fmaxf(big, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
      }
    float inv;
    pow2_scale(half_reduce(big, [](float p, float q) { return fmaxf(p, q); }), unscale, inv);
#pragma unroll
    for (int ks = 0; ks < DS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float4 z = qx[ks][e / 4];
        const Parts y = split_query<KH>((e % 4 == 0 ? z.x : e % 4 == 1 ? z.y : e % 4 == 2 ? z.z : z.w) * inv);
        qh[ks][e] = y.hi;
        ql[ks][e] = y.lo;
      }
  }

  floatx16 o[DT];  // dim 32 dt + 8 (v / 4) + 4 h2 + v % 4
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = floatx16{};
  float m = -INFINITY, l = 0.0f;
  int unit = NO_UNIT;  // f32: the row's o is in units of 2^unit
  uint32_t seg = 0;
  auto where = [&](uint32_t i) { return i < n_pre ? prefix_tile<T, KT>(a.c, g, p_lo + i) : own_tile<T, KT>(a.c, run, g, o_lo + (i - n_pre), seg); };
  Where<T> w{};
  if (n_tiles) {
    w = where(0);
    if (!early) load_first(w);
    if constexpr (KH) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
      store_f32(0, 0, kr);
      store_f32(0, 1, vr);
    }
  }
  __syncthreads();
  for (uint32_t i = 0; i < n_tiles; ++i) {
    const uint32_t buf = i & 1u;
    const bool more = i + 1 < n_tiles;
    const Where<T> next = more ? where(i + 1) : w;
    if constexpr (KH) {
      if (more) load(next, buf ^ 1u);
    } else {
      if (more) {
        load_f32(next, next.k, 0, kr);
        load_f32(next, next.v, 1, vr);
      }
    }
    const int limit = !live ? -1 : w.seg < 0 ? int(a.c.P) - 1 : uint32_t(w.seg) == own_rows >> 16 ? int(own_rows & 0xffffu) : -1;
    if (__any(limit >= int(w.key0))) {  // else nothing of it is for this wave's rows
      // fragment addresses: the swizzle changes with the low bits of ks and with dt, the rest are constants
      lds_byte *kp[4], *vp[DT];
#pragma unroll
      for (int c = 0; c < 4; ++c) kp[c] = (lds_byte*)lds + (buf * BUF + k_at(r32, 2 * c + h2));
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint32_t i16 = lane & 15u, byte = 64 * dt + 32 * ((lane >> 4) & 1u) + 8 * (i16 & 3u);
        vp[dt] = (lds_byte*)lds + (buf * BUF + v_at(4 * h2 + i16 / 4, byte >> 4) + (byte & 15u));
      }
      // plane 0: the keys or their hi parts, 1: the lo parts; 32 keys from 32 sub
      auto key8 = [&](int plane, int sub, int ks) {
        return *reinterpret_cast<const lds_half8*>(kp[ks % 4] + (plane * PLANE + 32 * sub * RB + ks / 4 * 128));
      };
      // 16 keys of 32 dims, transposed; plane as above
      auto value8 = [&](int plane, int sub, int dt, int st) {
        half4 y[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) y[u] = read_tr(vp[dt] + ((KH ? 1 : 2 + plane) * PLANE + (32 * sub + 16 * st + 8 * u) * RB));
        return __builtin_shufflevector(y[0], y[1], 0, 1, 2, 3, 4, 5, 6, 7);
      };
      // f16: products that follow one another go to different accumulators, for one that waits for its own leaves
      // the matrix unit idle.  Fragments are read two ahead (f32, short of registers: one); the barriers keep the
      // compiler from reading all of them first.
      floatx16 s[NSUB] = {};
      {
        constexpr int AHEAD = KH ? 2 : 1;
        half8 k8[3][2];
        floatx16 s_lo = {};
        auto read = [&](int ks) {
          k8[ks % 3][0] = key8(0, 0, ks);
          k8[ks % 3][1] = KH ? key8(0, 1, ks) : key8(1, 0, ks);
        };
#pragma unroll
        for (int ks = 0; ks < AHEAD; ++ks) read(ks);
#pragma unroll
        for (int ks = 0; ks < DS; ++ks) {
          if (ks + AHEAD < DS) read(ks + AHEAD);
          const half8 x = k8[ks % 3][0], y = k8[ks % 3][1];
          if constexpr (KH) {
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qh[ks], s[0], 0, 0, 0);
            s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, qh[ks], s[1], 0, 0, 0);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ql[ks], s[0], 0, 0, 0);
            s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, ql[ks], s[1], 0, 0, 0);
          } else {
            floatx16 &p = ks % 2 ? s_lo : s[0], &q = ks % 2 ? s[0] : s_lo;
            p = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qh[ks], p, 0, 0, 0);
            q = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, qh[ks], q, 0, 0, 0);
            p = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ql[ks], p, 0, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!KH) {  // (the scales with the query's own, all powers of two)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const floatx4 ks = *reinterpret_cast<const floatx4*>(&k_scale[buf][8 * c + 4 * h2]) * unscale;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0][4 * c + e] = (s[0][4 * c + e] + s_lo[4 * c + e]) * ks[e];
          }
        }
      }
      const bool whole = __all(limit >= int(w.key0) + KT - 1);
      if (!whole) {
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (int(w.key0) + int(32u * sub + 8u * (v / 4) + 4u * h2 + (v % 4)) > limit) s[sub][v] = -INFINITY;
      }
      float top = -INFINITY;
      if constexpr (KH) {
        float top1 = -INFINITY;
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
          top = fmaxf(fmaxf(top, s[0][v]), s[0][v + 1]);
          top1 = fmaxf(fmaxf(top1, s[NSUB - 1][v]), s[NSUB - 1][v + 1]);
        }
        top = fmaxf(top, top1) * unscale;
      } else {
#pragma unroll
        for (int v = 0; v < 16; v += 2) top = fmaxf(fmaxf(top, s[0][v]), s[0][v + 1]);
      }
      const float mn = fmaxf(m, half_reduce(top, [](float p, float q) { return fmaxf(p, q); }));
      const bool up = mn > m + SLACK;
      if (__any(up)) {
        const float to = up ? floorf(mn) : m, f = up ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
        l *= f;
        m = to;
      }
      const float bias = LIFT - (m == -INFINITY ? 0.0f : m);
      if constexpr (!KH) {
        int most = NO_UNIT;
        if (whole) {  // a key per lane
          most = int(wave_reduce(uint32_t(v_exp[buf][r32]), [](uint32_t p, uint32_t q) { return uint32_t(max(int(p), int(q))); }));
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const intx4 ve = *reinterpret_cast<const intx4*>(&v_exp[buf][8 * c + 4 * h2]);
#pragma unroll
            for (int e = 0; e < 4; ++e) most = max(most, int(w.key0) + int(8u * c + 4u * h2 + e) <= limit ? ve[e] : NO_UNIT);
          }
          const auto both = __builtin_amdgcn_permlane32_swap(uint32_t(most), uint32_t(most), false, false);
          most = max(int(both[0]), int(both[1]));
        }
        most = max(most, unit);
        if (__any(most > unit)) {
          const float f = __builtin_amdgcn_ldexpf(1.0f, unit - most);
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d] *= f;
          unit = most;
        }
        asm volatile("" ::: "memory");  // (the exponents are read again, not kept)
      }
      int odd = 0;  // a value that is no number, and rows that must not see it
      if (!whole && w.seg >= 0) {
        half8 z = half8{};
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int st = 0; st < 2; ++st) z = __builtin_elementwise_fma(value8(0, sub, dt, st), half8{}, z);
          __builtin_amdgcn_sched_barrier(0);
        }
        odd = __any(not_zero(z));
      }
#pragma unroll
      for (int sub = 0; sub < NSUB; ++sub) {
        half8 ph[2], pl[2];  // 16 keys each: the weights' upper 11 bits, and the rest
        float sum[2] = {0.0f, 0.0f};
        intx4 ve;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          if (!KH && v % 4 == 0) ve = *reinterpret_cast<const intx4*>(&v_exp[KH ? 0 : buf][8 * (v / 4) + 4 * h2]);
          float p = __builtin_amdgcn_exp2f(KH ? fmaf(s[sub][v], unscale, bias) : s[sub][v] + bias);
          sum[v % 2] += p;
          s[sub][v] = p;
          if constexpr (!KH) p = __builtin_amdgcn_ldexpf(p, ve[v % 4] - unit);  // (0 of a key that the row does not see)
          const float hi = __uint_as_float(__float_as_uint(p) & 0xffffe000u);
          ph[v / 8][v % 8] = _Float16(hi);
          pl[v / 8][v % 8] = _Float16(p - hi);
        }
        l += sum[0] + sum[1];
        if constexpr (!KH) asm volatile("" : "+v"(l));  // (here, or the sums hold all the weights' registers to the end)
        int slow = __builtin_amdgcn_readfirstlane(odd);
        if (slow) {  // key by key, for the rows that see it
          const float per_unit = KH ? 1.0f : __builtin_amdgcn_ldexpf(1.0f, -unit);
          for (int key = 0; key < 32 && 32 * sub + key < int(w.keys); ++key) {
            float p = 0.0f;
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const float x = __shfl(s[sub][v], ((key >> 2) & 1) * 32 + int(r32), 64);
              if ((v / 4) * 8 + v % 4 == (key & ~4)) p = x * per_unit;
            }
            const bool sees = int(w.key0) + 32 * sub + key <= limit;
            const T* value = w.v + size_t(32 * sub + key) * w.stride + 4 * h2;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
              for (int v = 0; v < 16; ++v) {
                const float x = fmaf(p, float(value[32 * dt + 8 * (v / 4) + v % 4]), o[dt][v]);
                o[dt][v] = sees ? x : o[dt][v];
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
        asm volatile("" : "+s"(slow));  // (one branch after the other: as two sides of one they would hold two sets of o)
        if (!slow) {
          // block c: 16 keys (st = c / DT) of 32 dims; its second and third terms come a block and two later, not right
          // behind the one before
          constexpr int BL = 2 * DT, AHEAD = KH ? 2 : 1, TERMS = KH ? 2 : 3;
          half8 v8[4], u8[KH ? 1 : 4];
          auto read = [&](int c) {
            v8[c % 4] = value8(0, sub, c % DT, c / DT);
            if constexpr (!KH) u8[c % 4] = value8(1, sub, c % DT, c / DT);
          };
#pragma unroll
          for (int c = 0; c < AHEAD; ++c) read(c);
#pragma unroll
          for (int c = 0; c < BL + TERMS - 1; ++c) {
            if (c + AHEAD < BL) read(c + AHEAD);
            if (c < BL) o[c % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8[c % 4], ph[c / DT], o[c % DT], 0, 0, 0);
            if (c >= 1 && c <= BL) {
              const int b = c - 1;
              o[b % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8[b % 4], pl[b / DT], o[b % DT], 0, 0, 0);
            }
            if constexpr (!KH) {
              if (c >= 2) {
                const int b = c - 2;
                o[b % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u8[b % 4], ph[b / DT], o[b % DT], 0, 0, 0);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
    if (more) {
      if constexpr (KH) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      } else {
        store_f32(buf ^ 1u, 0, kr);
        store_f32(buf ^ 1u, 1, vr);
      }
    }
    __syncthreads();
    w = next;
  }

  l = half_reduce(l, [](float p, float q) { return p + q; });
  const bool last = splits == 1;
  if (at >= rows || (last && !live)) return;
  const size_t part = ((size_t(g) * sp.tiles + row / 16) * sp.splits + split) * 16 + row % 16;
  float* dst = last ? a.out + at_row * HD : sp.o + part * HD;
  const float f = (last ? (m == -INFINITY ? NAN : 1.0f / l) : KH ? 1.0f : F32_DOWN) * (KH ? 1.0f : __builtin_amdgcn_ldexpf(1.0f, unit));
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<floatx4*>(dst + 32 * dt + 8 * c + 4 * h2) =
          floatx4{o[dt][4 * c] * f, o[dt][4 * c + 1] * f, o[dt][4 * c + 2] * f, o[dt][4 * c + 3] * f};
  if (h2 == 0 && (!last || stat)) {
    float* st = last ? stat + 2 * at_row : sp.ml + 2 * part;
    st[0] = m - LIFT;
    st[1] = l;
  }
}

// The splits' states of the rows of the output joined: HD / 4 threads per row and
// TEAM teams of them per row, each with every TEAM-th split.  A team loads its
// states before it looks at their m, and before it knows that the row is one.
template <int HD, int TEAM>
__device__ __forceinline__ void join_rows(const KvAttendArgs& a, const KvSplit& sp, float* stat) {
  constexpr uint32_t LP = HD / 4, ROWS = 256 / LP / TEAM;
  __shared__ floatx4 os[TEAM == 1 ? 1 : TEAM][LP];
  __shared__ float ms[TEAM], ls[TEAM];
  const uint32_t tid = threadIdx.x, team = tid / LP % TEAM, d = tid % LP;
  const uint32_t at = blockIdx.x * ROWS + tid / LP / TEAM;
  const bool is_row = at < a.c.R * a.c.n * a.s.H;
  const uint32_t out = is_row ? at : 0u, bt = out / a.s.H, h = out % a.s.H, b = bt / a.c.n, t = bt % a.c.n, g = h / a.s.rep;
  const RawRequest raw = load_request(a.c, b);
  const uint32_t row = bt * a.s.rep + h % a.s.rep, tile = row / 16;
  const size_t part = (size_t(g) * sp.tiles + tile) * sp.splits * 16 + row % 16;  // + 16 split
  bool done = false;  // the row has its output
  if (TEAM == 1) {    // many rows: the state's bytes count, not the wait for its m and l
    const float2 ml = *reinterpret_cast<const float2*>(sp.ml + 2 * part);
    if (ml.y == NO_STATE) return;
  }
  float M = -INFINITY, L = 0.0f;
  floatx4 x = floatx4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t s0 = team; s0 < sp.splits; s0 += 4 * TEAM) {
    floatx4 y[4];
    float2 ml[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t s = min(s0 + i * TEAM, sp.splits - 1);
      ml[i] = *reinterpret_cast<const float2*>(sp.ml + 2 * (part + 16 * s));
      if (TEAM > 1 || s0 + i < sp.splits) y[i] = *reinterpret_cast<const floatx4*>(sp.o + (part + 16 * s) * HD + 4 * d);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s0 + i * TEAM >= sp.splits) continue;
      if (ml[i].y == NO_STATE) {
        done |= s0 + i * TEAM == 0;
        continue;
      }
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
  if (done || !is_row || t >= checked(a.c, raw, nullptr).fresh) return;
  *reinterpret_cast<floatx4*>(a.out + size_t(out) * HD + 4 * d) = x * (M == -INFINITY ? NAN : sp.up / L);
  if (stat && d == 0) {
    stat[2 * size_t(out)] = M;
    stat[2 * size_t(out) + 1] = L;
  }
}

template <int HD, int TEAM>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttendArgs a, KvSplit sp, float* stat) {
  join_rows<HD, TEAM>(a, sp, stat);
}

// ---------------------------------------------------------------------------
// weights
// ---------------------------------------------------------------------------
// A key's weights summed over the rows that see it, from the rows' final (m, l):
// the scores once more, transposed as above, with the keys in registers for the
// whole kernel (a wave's 64 of f16, 32 of f32) and the rows passing by in LDS,
// 32 at a time as hi + lo parts that the block splits.  A lane adds up its row's
// weights per key; the 32 rows of a wave's lanes are summed at the end, so every
// sum has one order.  blockIdx.z = request, or R for the prefix with the rows of
// all requests; with several row splits the sums go to the workspace and
// kv_weights_join_kernel adds them.
//   A prompt of 1500 tokens, f16: 38 us, 0.57 PFLOP/s of hi + lo products; vector
// instructions (a step splits 32 rows and takes 64 exponentials a lane pair) take
// as many cycles as the products.
struct RowSteps {
  uint32_t base, begin, end, steps;
};
// The rows that a block of keys from k0 looks at: packed (b n + t) rep + r, or t rep + r of the request from the
// first that sees key k0.
__device__ __forceinline__ RowSteps row_steps(const KvAttendArgs& a, Request rq, bool prefix, uint32_t k0) {
  RowSteps r;
  r.base = prefix ? 0u : rq.len - rq.fresh;
  r.end = prefix ? a.c.R * a.c.n * a.s.rep : rq.fresh * a.s.rep;
  r.begin = !prefix && k0 > r.base ? min(r.end, (k0 - r.base) * a.s.rep) / 32 * 32 : 0u;
  r.steps = (r.end - r.begin + 31) / 32;
  return r;
}

template <int HD, bool KH>
__global__ __launch_bounds__(256, 2) void kv_weigh_kernel(KvAttendArgs a, const float* stat, float* part, uint32_t chunk) {
  using T = Elem<KH>;
  constexpr int KW = KH ? 2 : 1;           // 32-key tiles per wave
  constexpr int DS = HD / 16;
  constexpr uint32_t KB = 128 * KW;        // keys per block
  constexpr uint32_t RB = HD * 2, PLANE = 32 * RB;
  __shared__ __align__(16) uint8_t lds[2][2 * PLANE];
  __shared__ float4 info[2][32];           // a row's unscale, m, 1 / l (0: no row), last slot seen
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), r32 = lane & 31u, h2 = lane >> 5;
  const uint32_t g = blockIdx.x % a.s.G, split = blockIdx.y, z = blockIdx.z;
  const bool prefix = z == a.c.R;
  Request rq{a.c.P, 0};
  if (!prefix) rq = request_of(a.c, z, nullptr);
  const uint32_t n_keys = rq.len;
  for (uint32_t kb = blockIdx.x / a.s.G; kb * KB < n_keys; kb += gridDim.x / a.s.G) {
    const uint32_t k0 = kb * KB;
    const RowSteps rs = row_steps(a, rq, prefix, k0);
    const uint32_t base = rs.base, row_begin = rs.begin, row_end = rs.end;
    const uint32_t s_lo = split * chunk, s_hi = min(s_lo + chunk, rs.steps);
    if (s_lo >= s_hi && split) return;  // later keys are seen by fewer rows

    // the wave's keys: key 32 kw + r32, dims 16 ks + 8 h2 + e
    const uint32_t key0 = k0 + wave * 32 * KW;
    half8 kh[KW][DS], kl[KH ? 1 : KW][DS];
    float key_scale[KH ? 1 : 16];  // f32: a power of two of each key's own (one for several would let a later key take the low bits off earlier ones)
#pragma unroll
    for (int kw = 0; kw < KW; ++kw) {
      const size_t stride = prefix ? a.c.p_slot_stride : a.c.slot_stride;
      const T* row = (prefix ? static_cast<const T*>(a.c.pk) + g * a.c.p_head_stride
                             : static_cast<const T*>(a.c.k) + z * a.c.req_stride + g * a.c.head_stride) +
                     min(key0 + 32 * kw + r32, n_keys - 1) * stride + 8 * h2;
      if constexpr (KH) {
#pragma unroll
        for (int ks = 0; ks < DS; ++ks) kh[kw][ks] = *reinterpret_cast<const half8*>(row + 16 * ks);
      } else {
        float x[DS][8], big = 0.0f;
#pragma unroll
        for (int ks = 0; ks < DS; ++ks)
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const floatx4 y = *reinterpret_cast<const floatx4*>(row + 16 * ks + e);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              x[ks][e + c] = y[c];
              big = fmaxf(big, fabsf(y[c]) < INFINITY ? fabsf(y[c]) : 0.0f);
            }
          }
        big = half_reduce(big, [](float p, float q) { return fmaxf(p, q); });
        float r, inv;
        pow2_scale(big, r, inv);
#pragma unroll
        for (int v = 0; v < 16; ++v) key_scale[v] = __shfl(r, 8 * (v / 4) + 4 * int(h2) + v % 4, 64);
#pragma unroll
        for (int ks = 0; ks < DS; ++ks)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = x[ks][e] * inv;
            kh[kw][ks][e] = _Float16(y);
            kl[kw][ks][e] = _Float16(y - float(kh[kw][ks][e]));
          }
      }
    }

    // staging: 8 threads per row, HD / 8 dims each; nothing is looked at before it goes to LDS, a step later
    constexpr int SD = HD / 8;
    float4 qr[SD / 4];
    float2 q_ml;
    RawRequest q_rq{0, 0};
    uint32_t q_t = 0;
    bool q_row = false;
    const uint32_t srow = tid / 8, sd = tid % 8 * 4;  // dims sd + 32 i ..: 128 bytes of a row per load
    // the row of the next load: token (of the request, or b n + t) and head, counted on by 32 rows a step
    uint32_t at_row = row_begin + s_lo * 32 + srow, token = at_row / a.s.rep, head = at_row % a.s.rep;
    const uint32_t tokens_on = 32 / a.s.rep, heads_on = 32 % a.s.rep, tokens = row_end / a.s.rep;
    auto load = [&]() {
      q_row = at_row < row_end;
      q_t = min(token, tokens - 1);
      const size_t at = (prefix ? size_t(q_t) : size_t(z) * a.c.n + q_t) * a.s.H + g * a.s.rep + head;
      if (prefix) {
        const uint32_t b = a.c.n == 1 ? q_t : q_t / a.c.n;
        q_rq = load_request(a.c, b);
        q_t -= b * a.c.n;
      }
#pragma unroll
      for (int i = 0; i < SD / 4; ++i) qr[i] = *reinterpret_cast<const float4*>(a.q + at * HD + sd + 32 * i);
      q_ml = *reinterpret_cast<const float2*>(stat + 2 * at);
      at_row += 32;
      token += tokens_on;
      head += heads_on;
      if (head >= a.s.rep) {
        head -= a.s.rep;
        ++token;
      }
    };
    auto k_at = [](uint32_t key, uint32_t piece) { return key * RB + ((piece ^ (key & 7u)) << 4); };
    auto store = [&](uint32_t buf) {
      const bool live = q_row && (!prefix || q_t < checked(a.c, q_rq, nullptr).fresh);
      float4 qi = make_float4(0.0f, live ? q_ml.x : 0.0f, live ? __builtin_amdgcn_rcpf(q_ml.y) : 0.0f, __int_as_float(!live ? -1 : prefix ? 0x7fffffff : int(base + q_t)));
      float big = 0.0f;
#pragma unroll
      for (int i = 0; i < SD / 4; ++i) {
        if (!live) qr[i] = make_float4(0.f, 0.f, 0.f, 0.f);  // a row of no token may hold anything
        qr[i] = make_float4(qr[i].x * a.s.scale2, qr[i].y * a.s.scale2, qr[i].z * a.s.scale2, qr[i].w * a.s.scale2);
        big = fmaxf(big, fmaxf(fmaxf(fabsf(qr[i].x), fabsf(qr[i].y)), fmaxf(fabsf(qr[i].z), fabsf(qr[i].w))));
      }
      big = fmaxf(big, dpp_f32<DPP_QUAD_XOR1>(big));
      big = fmaxf(big, dpp_f32<DPP_QUAD_XOR2>(big));
      big = fmaxf(big, dpp_f32<DPP_ROW_HALF_MIRROR>(big));
      float inv;
      pow2_scale(big, qi.x, inv);
      if (tid % 8 == 0) info[buf][srow] = qi;
#pragma unroll
      for (int i = 0; i < SD / 4; ++i) {
        const float x[4] = {qr[i].x, qr[i].y, qr[i].z, qr[i].w};
        half4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          hi[e] = _Float16(x[e] * inv);
          lo[e] = _Float16(x[e] * inv - float(hi[e]));
        }
        const uint32_t d = sd + 32 * i, off = k_at(srow, d / 8) + d % 8 * 2;
        *reinterpret_cast<half4*>(&lds[buf][off]) = hi;
        *reinterpret_cast<half4*>(&lds[buf][PLANE + off]) = lo;
      }
    };

    float sum[KW][16];
#pragma unroll
    for (int kw = 0; kw < KW; ++kw)
#pragma unroll
      for (int v = 0; v < 16; ++v) sum[kw][v] = 0.0f;
    if constexpr (KH) {  // (waited for here; in the loop that would be for the rows in flight too)
#pragma unroll
      for (int kw = 0; kw < KW; ++kw)
#pragma unroll
        for (int ks = 0; ks < DS; ++ks) asm volatile("" : "+v"(kh[kw][ks]));
    }
    // Rows are loaded two steps ahead, and split for the next step while this one's products run.
    if (s_lo < s_hi) {
      load();
      store(0);
      if (s_lo + 1 < s_hi) load();
    }
    __syncthreads();
    for (uint32_t st = s_lo; st < s_hi; ++st) {
      const uint32_t buf = (st - s_lo) & 1u;
      float4 me = info[buf][r32];
      const int limit = __float_as_int(me.w);
      floatx16 s[KW];
#pragma unroll
      for (int kw = 0; kw < KW; ++kw) s[kw] = floatx16{};
      half8 q8[3][2];  // read two ahead
      auto read = [&](int ks) {
        const uint32_t off = k_at(r32, 2 * ks + h2);
#pragma unroll
        for (int p = 0; p < 2; ++p) q8[ks % 3][p] = *reinterpret_cast<const half8*>(&lds[buf][p * PLANE + off]);
      };
      read(0);
      read(1);
#pragma unroll
      for (int ks = 0; ks < DS; ++ks) {
        if (ks + 2 < DS) read(ks + 2);
        const half8 qh = q8[ks % 3][0], ql = q8[ks % 3][1];
#pragma unroll
        for (int kw = 0; kw < KW; ++kw) s[kw] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[kw][ks], qh, s[kw], 0, 0, 0);
#pragma unroll
        for (int kw = 0; kw < KW; ++kw) s[kw] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[kw][ks], ql, s[kw], 0, 0, 0);
        if constexpr (!KH) s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl[0][ks], qh, s[0], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (st + 1 < s_hi) {
        store(buf ^ 1u);
        if (st + 2 < s_hi) load();
      }
      if (!__all(limit >= int(key0) + 32 * KW - 1)) {
        const bool lost = !(me.y - me.y == 0.0f) || !(me.z - me.z == 0.0f);  // a row of no number: that of the keys it sees alone
#pragma unroll
        for (int kw = 0; kw < KW; ++kw)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const bool sees = int(key0) + int(32u * kw + 8u * (v / 4) + 4u * h2 + (v % 4)) <= limit;
            if (lost && sees) sum[kw][v] = NAN;
            if (lost || !sees) s[kw][v] = -INFINITY;
          }
        if (lost) me.y = me.z = 0.0f;
      }
#pragma unroll
      for (int kw = 0; kw < KW; ++kw)
#pragma unroll
        for (int v = 0; v < 16; ++v)  // (a factor of 0 would make the -infinity of a key that is not seen NaN)
          sum[kw][v] = fmaf(__builtin_amdgcn_exp2f(fmaf(s[kw][v], KH ? me.x : fmaxf(me.x * key_scale[v], 0x1p-126f), -me.y)), me.z, sum[kw][v]);
      __syncthreads();
    }
#pragma unroll
    for (int kw = 0; kw < KW; ++kw) {
      float mine = 0.0f;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        float x = row_reduce(sum[kw][v], [](float p, float q) { return p + q; });
        const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(y[0]) + __uint_as_float(y[1]);
        if (r32 == uint32_t(v)) mine = x;
      }
      const uint32_t key = key0 + 32 * kw + 8 * (r32 / 4) + 4 * h2 + r32 % 4;
      if (r32 >= 16 || key >= n_keys) continue;
      const size_t own = (size_t(z) * a.s.G + g) * a.c.cap + key;
      if (gridDim.y > 1) {
        const size_t all = size_t(a.s.G) * (size_t(a.c.R) * a.c.cap + a.c.P);
        part[split * all + (prefix ? size_t(a.c.R) * a.s.G * a.c.cap + size_t(g) * a.c.P + key : own)] = mine;
      } else if (prefix) {
        const size_t at = size_t(g) * a.pw_stride + key;
        a.pw_out[at] = (a.pw_in ? a.pw_in[at] : 0.0f) + mine;
      } else {
        a.w_out[own] = (a.w_in ? a.w_in[own] : 0.0f) + mine;
      }
    }
  }
}

// Weights of a step whose scores kv_step_kernel kept (own [b][g][slot][row of the
// request], prefix [g][key][row]): the last block of rows' joins and these in one
// launch.  A block works out its rows' (m, l) from the splits itself, the more
// lanes a row the fewer rows, then sums a key's weights per thread, or, of many
// rows, per 16 lanes.  Against the scores computed once more, the whole call, us:
// 8 requests of 1500 slots, f32, 23 : 40; 4 of 20000, f16, 70 : 95; 8 x 14 tokens
// of 8 heads over 2 after 666 positions 15 : 23, 12 x 4 of 32 over 8 after 2900
// 33 : 45, 1 x 139 18 : 23, 7 x 67 21 : 28; with shared positions 8 x 62 (1984 rows)
// over 11 27 : 34, 4 x 100 of 8 over 2 (1600) over 1500 36 : 38, 1 x 400 over 6000 82 : 80.
// Heads of 64, whose products are half as long, lose by it from about 1000 rows over
// shared positions on (4 x 100 over 1500 32 : 28): the rule goes by rows alone.
constexpr uint32_t KEPT_ROWS = 2048;     // of a request and, for the prefix, of all, at most
constexpr uint32_t KEPT_TEAM_ROWS = 32;  // from here on 16 lanes a key: 3 x 3 tokens of 14 heads over 2 after 2800 positions, 17 : 23 us a call
struct KvKeptGrid {
  uint32_t joins, prefix, own;     // blocks: of joins, per kv head of the prefix, per cache (a cache's walk over its keys)
  uint32_t prefix_keys, own_keys;  // per block
};
// Keys per block of `rows` rows, of `keys` keys over all caches and heads: one per thread, or 16 lanes; of many rows
// enough blocks that a block's walk is short (8 x 14 tokens of 8 heads over 2 after 666 positions 30 : 15 us a call).
inline uint32_t kept_keys(uint32_t rows, size_t keys) {
  if (rows < KEPT_TEAM_ROWS) return 256;
  return uint32_t(min(size_t(128), max(size_t(16), (keys / 512 + 15) / 16 * 16)));
}
template <int HD>
__global__ __launch_bounds__(256) void kv_join_weights_kernel(KvAttendArgs a, KvSplit sp, const float* stat, KvScores keep, KvKeptGrid grid) {
  if (blockIdx.x < grid.joins) return join_rows<HD, 1024 / HD>(a, sp, nullptr);
  __shared__ float2 ml[KEPT_ROWS];
  const uint32_t tid = threadIdx.x, i = blockIdx.x - grid.joins;
  const bool prefix = i < grid.prefix * a.s.G;
  const uint32_t j = prefix ? i : i - grid.prefix * a.s.G, blocks = prefix ? grid.prefix : grid.own;
  const uint32_t kb0 = j % blocks, g = j / blocks % a.s.G, z = j / blocks / a.s.G;
  const uint32_t per = a.c.n * a.s.rep, n_rows = prefix ? a.c.R * per : per, keys = prefix ? grid.prefix_keys : grid.own_keys;
  Request rq{a.c.P, a.c.n};
  if (!prefix) rq = request_of(a.c, z, nullptr);
  if (kb0 * keys >= rq.len) return;
  auto states = [&](auto LN) {
    constexpr uint32_t L = LN();  // lanes per row
    for (uint32_t r0 = 0; r0 < n_rows; r0 += 256 / L) {
      const uint32_t r = r0 + tid / L, row = min(prefix ? r : z * per + r, a.c.R * per - 1);
      float M = -INFINITY, S = 0.0f;
      if (sp.splits == 1) {
        const size_t at = size_t(row / a.s.rep) * a.s.H + g * a.s.rep + row % a.s.rep;
        M = stat[2 * at];
        S = stat[2 * at + 1];
      } else {
        const float* src = sp.ml + 2 * ((size_t(g) * sp.tiles + row / 16) * sp.splits * 16 + row % 16);
#pragma unroll 4
        for (uint32_t s = tid % L; s < sp.splits; s += L) {
          const float2 x = *reinterpret_cast<const float2*>(src + 32 * s);
          const float mn = fmaxf(M, x.x), base = mn == -INFINITY ? 0.0f : mn;
          S = S * __builtin_amdgcn_exp2f(M - base) + x.y * __builtin_amdgcn_exp2f(x.x - base);
          M = mn;
        }
        if constexpr (L > 1) {
          auto reduce = [](float x, auto op) {
            x = op(x, dpp_f32<DPP_QUAD_XOR1>(x));
            x = op(x, dpp_f32<DPP_QUAD_XOR2>(x));
            if constexpr (L == 16) {
              x = op(x, dpp_f32<DPP_ROW_HALF_MIRROR>(x));
              x = op(x, dpp_f32<DPP_ROW_MIRROR>(x));
            }
            return x;
          };
          const float all = reduce(M, [](float p, float q) { return fmaxf(p, q); });
          S = reduce(S * __builtin_amdgcn_exp2f(M - (all == -INFINITY ? 0.0f : all)), [](float p, float q) { return p + q; });
          M = all;
        }
      }
      // rows of no token give nothing
      const uint32_t b = row / per, t = row / a.s.rep % a.c.n;
      const bool live = r < n_rows && t < (prefix ? request_of(a.c, b, nullptr).fresh : rq.fresh);
      if (tid % L == 0 && r < n_rows) ml[r] = live ? make_float2(M, 1.0f / S) : make_float2(0.0f, 0.0f);
    }
  };
  if (n_rows <= 16)
    states(std::integral_constant<uint32_t, 16>());
  else if (n_rows <= 64)
    states(std::integral_constant<uint32_t, 4>());
  else
    states(std::integral_constant<uint32_t, 1>());
  __syncthreads();
  const uint32_t base = prefix ? 0xffffffffu : rq.len - rq.fresh;
  const float* in = prefix ? a.pw_in : a.w_in;
  float* out = prefix ? a.pw_out : a.w_out;
  auto sums = [&](auto LN) {
    constexpr uint32_t L = LN(), U = L == 1 ? 4 : 8;  // lanes per key, loads in flight
    const uint32_t lane = tid % L;
    for (uint32_t kb = kb0; kb * keys < rq.len; kb += blocks) {
      for (uint32_t c = 0; c < keys; c += 256 / L) {
        const uint32_t key = kb * keys + c + tid / L;
        if (key >= rq.len) break;  // (a key's lanes as one)
        const float* src = prefix ? keep.prefix + (size_t(g) * a.c.P + key) * n_rows : keep.own + ((size_t(z) * a.s.G + g) * a.c.cap + key) * per;
        const size_t at = prefix ? size_t(g) * a.pw_stride + key : (size_t(z) * a.s.G + g) * a.c.cap + key;
        const float before = in ? in[at] : 0.0f;
        const uint32_t first = key <= base ? 0u : (key - base) * a.s.rep;  // earlier rows do not see the key
        float w = 0.0f;
        for (uint32_t r0 = first; r0 < n_rows; r0 += U * L) {
          float y[U];
#pragma unroll
          for (uint32_t u = 0; u < U; ++u) y[u] = src[min(r0 + u * L + lane, n_rows - 1)];
#pragma unroll
          for (uint32_t u = 0; u < U; ++u) {
            const uint32_t r = r0 + u * L + lane;
            const float2 x = ml[min(r, n_rows - 1)];
            const float p = __builtin_amdgcn_exp2f(y[u] - x.x) * x.y;
            w += r < n_rows && x.y != 0.0f ? p : 0.0f;  // (a row of no token left no score)
          }
        }
        if constexpr (L == 16) w = row_reduce(w, [](float p, float q) { return p + q; });
        if (lane == 0) out[at] = before + w;
      }
    }
  };
  if (n_rows >= KEPT_TEAM_ROWS)
    sums(std::integral_constant<uint32_t, 16>());
  else
    sums(std::integral_constant<uint32_t, 1>());
}

// The chunks' sums, in order, and the weights so far.  KB: keys per block of kv_weigh_kernel.
__global__ __launch_bounds__(256) void kv_weights_join_kernel(KvAttendArgs a, const float* part, uint32_t chunk, uint32_t kb) {
  const uint32_t g = blockIdx.y, z = blockIdx.z;
  const bool prefix = z == a.c.R;
  Request rq{a.c.P, 0};
  if (!prefix) rq = request_of(a.c, z, nullptr);
  const size_t all = size_t(a.s.G) * (size_t(a.c.R) * a.c.cap + a.c.P);
  const float* in = prefix ? a.pw_in : a.w_in;
  float* out = prefix ? a.pw_out : a.w_out;
  for (uint32_t key = blockIdx.x * 256 + threadIdx.x; key < rq.len; key += gridDim.x * 256) {
    const uint32_t chunks = max(1u, (row_steps(a, rq, prefix, key / kb * kb).steps + chunk - 1) / chunk);
    const size_t own = (size_t(z) * a.s.G + g) * a.c.cap + key, at = prefix ? size_t(g) * a.pw_stride + key : own;
    const float* src = part + (prefix ? size_t(a.c.R) * a.s.G * a.c.cap + size_t(g) * a.c.P + key : own);
    const float before = in ? in[at] : 0.0f;
    float x = 0.0f;
    for (uint32_t i = 0; i < chunks; i += 8) {  // eight loads in flight
      float y[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) y[j] = src[min(i + j, chunks - 1) * all];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) x += i + j < chunks ? y[j] : 0.0f;
    }
    out[at] = before + x;
  }
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
// Order-preserving bits of a score: NaN as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t score_bits(float x) {
  if (!(x == x)) x = -INFINITY;
  const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the block's threads in thread order; total for all.
template <int THREADS>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* sh, uint32_t& total) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t x = wave_scan(v);
  __syncthreads();
  if (lane == 63) sh[wave] = x;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 64; ++w) {
    const uint32_t y = sh[w];
    if (w < wave) before += y;
    total += y;
  }
  return before + x - v;
}

// Rows lo .. hi - 1 of a list (to | from << 16) of cache sg, by `threads` threads; four loads of K and V each in flight.
__device__ __forceinline__ void move_rows(const KvEvictArgs& a, uint32_t sg, const uint32_t* list, uint32_t lo, uint32_t hi, uint32_t tid,
                                          uint32_t threads, uint32_t pieces) {
  const uint32_t g = sg % a.s.G, lb = sg / a.s.G, l = lb / a.c.R, b = lb % a.c.R;
  const uint32_t shift = 31 - __clz(pieces);
  const size_t base = (l * a.layer_stride + b * a.c.req_stride + g * a.c.head_stride) * a.elem;
  uint8_t *k = static_cast<uint8_t*>(a.c.k) + base, *v = static_cast<uint8_t*>(a.c.v) + base;
  const uint32_t first = lo << shift, last = hi << shift;
  for (uint32_t i0 = first + tid; i0 < last; i0 += 4 * threads) {
    u32x4 x[4], y[4];
    size_t to[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t i = min(i0 + c * threads, last - 1), mv = list[i >> shift], d = (i & (pieces - 1)) * 16;
      const size_t from = size_t(mv >> 16) * a.c.slot_stride * a.elem + d;
      to[c] = size_t(mv & 0xffffu) * a.c.slot_stride * a.elem + d;
      x[c] = *reinterpret_cast<const u32x4*>(k + from);
      y[c] = *reinterpret_cast<const u32x4*>(v + from);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (i0 + c * threads < last) {
        *reinterpret_cast<u32x4*>(k + to[c]) = x[c];
        *reinterpret_cast<u32x4*>(v + to[c]) = y[c];
      }
  }
}

// Eviction: blockIdx.x = (layer, request, kv head); thread t holds
// slots I t .. I t + I - 1.
//   The k-th largest score among the slots that compete (the safe ones all stay,
// the others compete for the rest) by digits of 8 bits from the top, until all
// scores that share them stay; of the slots that equal it in all four the lowest
// stay.  Then the freed slots below m and the kept ones from m on are counted off
// in slot order: the x-th of one takes the x-th of the other.
//   MOVE: the block then moves the rows, its part blockIdx.y of them, 16 bytes a
// thread; every part finds the same list (the scores are not written before all
// have read them: in place, there is one part).  A cache's list takes about 10 us
// of waiting for LDS and barriers, its rows the memory's time, so with two caches
// or more per CU one hides the other, and with fewer the parts share the rows
// without a second launch.  Otherwise the list goes to the workspace for
// kv_move_kernel.
//   Bound by memory: 36 layers x 4 requests x 8 heads of 1999 slots cut to 777, f16,
// 487 MB in 113 us (4.3 TB/s); 8 x 8 of 2560 to 1024, f32, 74 MB in 19 us, half of
// them the list.
struct KvMove {
  uint32_t max_moves, pieces;  // pieces: 16-byte pieces of a row
  uint32_t* moves;
  uint32_t* counts;
  bool lens;  // MOVE: write lens_out
};
template <int THREADS, int I, bool MOVE>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(KvEvictArgs a, KvMove mv) {
  constexpr int HIST = 4;  // copies of the digit counts, by lane, for many scores share a digit
  __shared__ uint32_t sh[THREADS / 64], hist[HIST][256], pick[3];
  __shared__ int32_t top[THREADS / 64];
  __shared__ uint32_t list[THREADS * I / 2];  // to | from << 16
  const uint32_t tid = threadIdx.x, sg = blockIdx.x, g = sg % a.s.G, lb = sg / a.s.G, b = lb % a.c.R;
  const uint32_t lane = tid & 63u, wave = tid >> 6;
  const int32_t in_use = a.c.lens[b];
  const size_t base = size_t(sg) * a.c.cap;
  float sc[I];
  int32_t pos[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {  // (slots not in use are loaded and left)
    const size_t at = base + min(tid * I + i, a.c.cap - 1);
    sc[i] = a.scores[at];
    pos[i] = a.positions[at];
  }
  const bool ok = in_use >= 0 && in_use <= int32_t(a.c.cap);
  const uint32_t n = ok ? uint32_t(in_use) : 0u, m = min(n, a.keep);
  const bool writes = !MOVE || blockIdx.y == 0;
  if (tid == 0 && writes) {
    if (!ok && lb == b && g == 0) atomicOr(a.s.err, S2HIP_KV_ERR_LENS);
    if (!MOVE) mv.counts[2 * blockIdx.x + 1] = ok ? m : 0xffffffffu;
    if (MOVE && mv.lens && ok && lb == b && g == 0) a.lens_out[b] = int32_t(m);
  }
  if (n <= a.keep) {  // nothing to cut
    if (!MOVE && tid == 0) mv.counts[2 * blockIdx.x] = 0;
    if (writes) {
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const uint32_t s = tid * I + i;
        if (s < n) {
          a.scores_out[base + s] = sc[i];
          a.positions_out[base + s] = pos[i];
        }
      }
    }
    return;
  }
  uint32_t bits[I];
  int32_t newest = INT32_MIN;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    bits[i] = score_bits(sc[i]);
    if (tid * I + i < n) newest = max(newest, pos[i]);
  }
  newest = int32_t(wave_reduce(uint32_t(newest) ^ 0x80000000u, [](uint32_t p, uint32_t q) { return max(p, q); }) ^ 0x80000000u);
  if (lane == 0) top[wave] = newest;
  for (uint32_t i = tid; i < HIST * 256; i += THREADS) hist[0][i] = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 64; ++w) newest = max(newest, top[w]);
  uint32_t safe = 0, n_safe = 0;  // bit i: slot i of the thread
#pragma unroll
  for (int i = 0; i < I; ++i)
    if (tid * I + i < n && (int64_t(pos[i]) > int64_t(newest) - int64_t(a.recent) || int64_t(pos[i]) < int64_t(a.sinks))) safe |= 1u << i;
  block_scan<THREADS>(__popc(safe), sh, n_safe);
  // who competes for how many places (positions given twice, or many sinks, can make more safe slots than there is room)
  const bool room = n_safe <= m;
  uint32_t want = room ? m - n_safe : m;
  uint32_t compete = 0;
#pragma unroll
  for (int i = 0; i < I; ++i)
    if (tid * I + i < n && (((safe >> i) & 1u) == 0) == room) compete |= 1u << i;
  uint32_t prefix = 0, kept = room ? safe : 0u;
  if (want) {
    int shift = 24;
    bool all = false;  // every score of the last digit stays: the rest of its bits decides nothing
#pragma unroll 1
    for (; shift >= 0 && !all; shift -= 8) {  // (the counts are zero here)
#pragma unroll
      for (int i = 0; i < I; ++i)
        if (((compete >> i) & 1u) && (shift == 24 || (bits[i] >> (shift + 8)) == prefix))
          atomicAdd(&hist[lane % HIST][(bits[i] >> shift) & 255u], 1u);
      __syncthreads();
      if (tid < 64) {  // digits from the top: lane l holds 255 - 4 l .. 252 - 4 l
        uint32_t c[4], x = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[j] = 0;
#pragma unroll
          for (int h = 0; h < HIST; ++h) {
            c[j] += hist[h][255 - 4 * lane - j];
            hist[h][255 - 4 * lane - j] = 0;
          }
          x += c[j];
        }
        uint32_t above = wave_scan(x) - x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (above < want && above + c[j] >= want) {
            pick[0] = 255 - 4 * lane - j;
            pick[1] = want - above;
            pick[2] = c[j];
          }
          above += c[j];
        }
      }
      __syncthreads();
      prefix = (prefix << 8) | pick[0];
      want = pick[1];
      all = pick[2] == want;
    }
    shift += 8;
    uint32_t equal = 0;
#pragma unroll
    for (int i = 0; i < I; ++i)
      if ((compete >> i) & 1u) {
        if ((bits[i] >> shift) > prefix) kept |= 1u << i;
        if ((bits[i] >> shift) == prefix) equal |= 1u << i;
      }
    if (all) {
      kept |= equal;
    } else {
      uint32_t dummy, rank = block_scan<THREADS>(__popc(equal), sh, dummy);
#pragma unroll
      for (int i = 0; i < I; ++i)
        if ((equal >> i) & 1u)
          if (rank++ < want) kept |= 1u << i;
    }
  }
  // slots of the thread below m; the rest of them
  const uint32_t low = tid * I >= m ? 0u : m - tid * I >= 32 ? 0xffffffffu : (1u << (m - tid * I)) - 1u;
  const uint32_t used = tid * I >= n ? 0u : n - tid * I >= uint32_t(I) ? uint32_t((uint64_t(1) << I) - 1u) : (1u << (n - tid * I)) - 1u;
  const uint32_t holes = used & low & ~kept, movers = used & ~low & kept;
  uint32_t both;
  const uint32_t ranks = block_scan<THREADS>(__popc(holes) | __popc(movers) << 16, sh, both);  // (at most 16384 of each, as many of one as of the other)
  const uint32_t n_movers = both >> 16;
  uint32_t hr = ranks & 0xffffu, mr = ranks >> 16;
  uint16_t* half = reinterpret_cast<uint16_t*>(list);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    if ((holes >> i) & 1u) half[2 * hr++] = uint16_t(tid * I + i);
    if ((movers >> i) & 1u) half[2 * mr++ + 1] = uint16_t(tid * I + i);
  }
  __syncthreads();
  if (writes) {  // scores and positions go from the threads that hold them
    mr = ranks >> 16;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const bool moves = (movers >> i) & 1u, stays = ((used & low & kept) >> i) & 1u;
      const uint32_t to = moves ? half[2 * mr++] : tid * I + i;
      if (moves || stays) {
        a.scores_out[base + to] = sc[i];
        a.positions_out[base + to] = pos[i];
      }
    }
  }
  if constexpr (!MOVE) {
    if (tid == 0) mv.counts[2 * blockIdx.x] = n_movers;
    for (uint32_t i = tid; i < n_movers; i += THREADS) mv.moves[size_t(blockIdx.x) * mv.max_moves + i] = list[i];
  } else {
    move_rows(a, sg, list, n_movers * blockIdx.y / gridDim.y, n_movers * (blockIdx.y + 1) / gridDim.y, tid, THREADS, mv.pieces);
  }
}

// blockIdx.y = (layer, request, kv head).
__global__ __launch_bounds__(256) void kv_move_kernel(KvEvictArgs a, KvMove mv) {
  const uint32_t sg = blockIdx.y, g = sg % a.s.G, lb = sg / a.s.G, b = lb % a.c.R;
  const uint32_t n_moves = mv.counts[2 * blockIdx.y], left = mv.counts[2 * blockIdx.y + 1];
  if (blockIdx.x == 0 && threadIdx.x == 0 && lb == b && g == 0 && left != 0xffffffffu) a.lens_out[b] = int32_t(left);
  move_rows(a, sg, mv.moves + size_t(blockIdx.y) * mv.max_moves, n_moves * blockIdx.x / gridDim.x, n_moves * (blockIdx.x + 1) / gridDim.x,
            threadIdx.x, 256, mv.pieces);
}

// lens_out in place of lens, once nothing reads them.
__global__ __launch_bounds__(256) void kv_lens_kernel(KvEvictArgs a) {
  const uint32_t b = threadIdx.x;
  if (b >= a.c.R) return;
  const int32_t len = a.c.lens[b];
  if (len >= 0 && len <= int32_t(a.c.cap)) a.lens_out[b] = min(len, int32_t(a.keep));
}

__global__ void kv_take_errors_kernel(uint32_t* err, uint32_t* taken) { *taken = atomicExch(err, 0u); }

// f(std::integral_constant<int, HD>, std::bool_constant<KH>)
template <class F>
hipError_t by_shape(uint32_t hd, bool f16, F&& f) {
  using std::integral_constant;
  if (hd == 64) return f16 ? f(integral_constant<int, 64>(), std::true_type()) : f(integral_constant<int, 64>(), std::false_type());
  if (hd == 128) return f16 ? f(integral_constant<int, 128>(), std::true_type()) : f(integral_constant<int, 128>(), std::false_type());
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_kv_append(uint32_t hd, bool f16, const KvAppendArgs& a, hipStream_t s) {
  return by_shape(hd, f16, [&](auto HD, auto KH) {
    const uint32_t tokens = a.c.R * a.c.n, steps = (a.s.H + 2 * a.s.G + 1024 / HD() - 1) / (1024 / HD());
    hipLaunchKernelGGL((kv_append_kernel<HD(), KH()>), dim3(tokens, min(steps, max(1u, 512 / tokens))), dim3(256), 0, s, a);
    return hipGetLastError();
  });
}

hipError_t launch_kv_attend(uint32_t hd, bool f16, const KvAttendArgs& a, const KvWorkspace& w, hipStream_t s) {
  KvSplit sp{};
  sp.o = w.part;
  sp.ml = w.part_ml;
  sp.up = f16 ? 1.0f : F32_UP;
  const uint32_t rows = a.c.R * a.c.n * a.s.rep;
  sp.tiles = (rows + 15) / 16;
  // The scores of few enough rows can be kept, where there is room for them.
  const size_t own_scores = size_t(rows) * a.s.G * a.c.cap, prefix_scores = a.pw_out ? size_t(rows) * a.s.G * a.c.P : 0;
  const bool may_keep = a.w_out && own_scores + prefix_scores <= w.cap_weights && a.c.n * a.s.rep <= KEPT_ROWS && (!a.pw_out || rows <= KEPT_ROWS);
  // Which kernel: by the scores to compute, over all heads and at most (capacities, of the turn's own slots half; lengths
  // are on the device), for the step kernel starts and ends quicker and the tile kernel multiplies quicker; heads of 64
  // count half.  Both with their join, us, step : tile, 32 heads over 8: f16 2 requests x 211 tokens over 110 + 452 slots
  // (6M scores) 21 : 29, 5 x 35 over 1500 + 78 (6.6M) 34 : 33, 4 x 64 over 1500 (13M) 37 : 39, 2 x 517 over 146 + 624 (17M)
  // 52 : 43; f32 8 x 12 over 728 + 235 (3M) 22 : 33, 3 x 37 over 1001 + 768 (6M) 34 : 34, 2 x 445 over 10 + 616 (11M) 62 : 48.
  // Kept scores save the tile kernel's weights their products: f16 8 x 145 over 488 own slots (15M) 62 : 67, 8 x 174 (17M) 51 :
  // 57, 4 x 142 of 24 over 1151 + 367 (20M) 80 : 66; f32 3 x 129 (3M) 24 : 44, 8 x 97 (8M) 34 : 46, 2 x 104 over 1500 + 239 (11M)
  // 87 : 72.  A request of fewer than 32 rows would leave most of a tile's waves idle in its own cache.
  const size_t scores = size_t(a.s.G) * rows * (a.c.P + a.c.cap - min(a.c.n, a.c.cap) / 2);
  const bool many = a.c.n * a.s.rep >= 32 && scores * hd > (may_keep ? f16 ? 14000000u : 8000000u : f16 ? 10000000u : 4200000u) * size_t(128);
  const uint32_t lots = a.s.G * (many ? (rows + TILE_ROWS - 1) / TILE_ROWS : sp.tiles), kt = many ? (f16 ? 64 : 32) : (f16 ? 32 : 16);
  // key tiles of a row tile, at most
  const uint32_t most = (a.c.P + kt - 1) / kt + (a.c.cap + kt - 1) / kt * (many ? 1u : min(a.c.R, 15 / (a.c.n * a.s.rep) + 1));
  // Step kernel: a block per CU, for more blocks' states cost the join more than they save (8 requests over 1500 + 512
  // slots, f32: 256 blocks 14.6 us, 512 16.8; 4 over 20000 with weights, f16: 70 : 75), but two where one each would leave
  // a third of the CUs idle (2 x 150 tokens of 8 heads over 2, 150 row tiles: 26.6 : 21.8).  Tile kernel: two.
  const uint32_t fill = many || (lots > 128 && lots <= 170) ? 512 : 256;
  sp.splits = max(1u, min(fill / lots, many ? max(1u, most / 2) : (most + STEP_WAVES - 1) / STEP_WAVES));
  // Up to six tiles a wave (twelve of heads of 64) cost less than a second launch, which weights have anyhow: 6 requests x
  // 3 tokens, 300 slots, f16 (24 tiles) 6.8 : 10.3 us, 3 x 22 over 207, f32 (21) 10.9 : 13.4, 7 x 2 over 307 (29) 13.6 :
  // 10.3; of heads of 64, 6 x 13 over 432, f16 (26) 6.8 : 9.1, 7 x 1 over 500 (32) 7.6 : 9.2, 2 x 4 over 1000 (53) 13.1 : 9.9.
  if (!many && most <= (a.w_out ? 20u : 24u * 128 / hd)) sp.splits = 1;
  if (many && lots > 256 && lots <= 448) {
    // More than a block per CU and less than two: row tiles of many keys in two, so that no CU has the two longest.
    // A prompt of 1500 tokens (376 row tiles) 80 : 69 us with the join, f32 153 : 105; from 448 on the join costs what it saves.
    sp.splits = 2;
    sp.least = 768 / kt;
  }
  if (size_t(a.s.G) * sp.tiles * sp.splits > w.cap_parts) sp.splits = uint32_t(max(size_t(1), w.cap_parts / (a.s.G * sp.tiles)));
  float* stat = a.w_out ? w.stat : nullptr;
  KvScores keep{};
  if (may_keep && !many) {
    keep.own = w.weights;
    keep.prefix = a.pw_out ? w.weights + own_scores : nullptr;
  }
  return by_shape(hd, f16, [&](auto HD, auto KH) {
    if (many)
      hipLaunchKernelGGL((kv_tile_kernel<HD(), KH()>), dim3(lots * sp.splits), dim3(256), 0, s, a, sp, stat);
    else
      hipLaunchKernelGGL((kv_step_kernel<HD(), KH()>), dim3(lots * sp.splits), dim3(64 * STEP_WAVES), 0, s, a, sp, stat, keep);
    const uint32_t out_rows = a.c.R * a.c.n * a.s.H, teams = 256 / (HD() / 4);
    const uint32_t z = a.c.R + (a.pw_out ? 1 : 0), keys = a.pw_out ? max(a.c.P, a.c.cap) : a.c.cap;
    if (keep.own) {
      KvKeptGrid grid{};
      grid.joins = sp.splits > 1 ? out_rows : 0;
      grid.own_keys = kept_keys(a.c.n * a.s.rep, size_t(a.c.cap) * a.c.R * a.s.G);
      grid.own = min(128u, (a.c.cap + grid.own_keys - 1) / grid.own_keys);
      grid.prefix_keys = kept_keys(rows, size_t(a.c.P) * a.s.G);
      if (a.pw_out) grid.prefix = (a.c.P + grid.prefix_keys - 1) / grid.prefix_keys;
      hipLaunchKernelGGL((kv_join_weights_kernel<HD()>), dim3(grid.joins + a.s.G * (grid.prefix + grid.own * a.c.R)), dim3(256), 0, s, a, sp, stat, keep, grid);
      return hipGetLastError();
    }
    if (sp.splits > 1 && out_rows <= 2048)
      hipLaunchKernelGGL((kv_join_kernel<HD(), 1024 / HD()>), dim3(out_rows), dim3(256), 0, s, a, sp, stat);
    else if (sp.splits > 1)
      hipLaunchKernelGGL((kv_join_kernel<HD(), 1>), dim3((out_rows + teams - 1) / teams), dim3(256), 0, s, a, sp, stat);
    if (a.w_out) {
      const uint32_t kb = KH() ? 256 : 128;
      // Steps of 32 rows.  Lengths are on the device: chunks are made for a cache of no more than the turn, whose key block i
      // is seen from its row i kb rep on (longer ones have more key blocks, so the chunks are many enough), and blocks walk
      // over the keys, so that slots not in use cost no blocks.  A block costs its start (keys, and f32 ones split) and 1.3
      // us a step, the join 64 chunks with ease.  Chunks of 2 : 3 : 5 : 8 : 13 steps, the whole call, 32 heads over 8, us:
      // f16 1 request x 1500 tokens (5184 steps) 132 : 121 : 113 : 112 : 102, 1 x 126 over 1500 (896) 42 : 43 : 46 : 48 : 56;
      // f32 5 x 243 (1840) 85 : 77 : 75 : 69 : 77, 2 x 157 over 32 (704) 34 : 35 : 37 : 39 : 44.
      const uint32_t own_steps = (a.c.n * a.s.rep + 31) / 32, all_steps = a.pw_out ? (rows + 31) / 32 : own_steps;
      const size_t own_blocks = (min(a.c.n, a.c.cap) + kb - 1) / kb, p_blocks = a.pw_out ? (a.c.P + kb - 1) / kb : 0;
      const size_t work = a.s.G * (a.c.R * (own_blocks * own_steps - own_blocks * (own_blocks - 1) / 2 * (kb * a.s.rep / 32)) + p_blocks * all_steps);
      const size_t all = size_t(a.s.G) * (size_t(a.c.R) * a.c.cap + a.c.P);
      const uint32_t room = uint32_t(max(size_t(1), min(size_t(all_steps), w.cap_weights / all)));  // chunks that fit the workspace
      const size_t blocks = !KH() && HD() == 128 ? 256 : 430;
      const uint32_t chunk = max(max(uint32_t(min(size_t(all_steps), max(size_t(2), (work + blocks - 1) / blocks))), (all_steps + 63) / 64), (all_steps + room - 1) / room);
      const uint32_t chunks = (all_steps + chunk - 1) / chunk;
      hipLaunchKernelGGL((kv_weigh_kernel<HD(), KH()>), dim3(min(16u, (keys + kb - 1) / kb) * a.s.G, chunks, z), dim3(256), 0, s, a, w.stat, w.weights, chunk);
      if (chunks > 1)
        hipLaunchKernelGGL(kv_weights_join_kernel, dim3(min(16u, (keys + 255) / 256), a.s.G, z), dim3(256), 0, s, a, w.weights, chunk, kb);
    }
    return hipGetLastError();
  });
}

template <bool MOVE>
static void select_launch(const KvEvictArgs& a, const KvMove& mv, dim3 grid, hipStream_t s) {
  if (a.c.cap <= 2048)
    hipLaunchKernelGGL((kv_select_kernel<256, 8, MOVE>), grid, dim3(256), 0, s, a, mv);
  else if (a.c.cap <= 4096)
    hipLaunchKernelGGL((kv_select_kernel<512, 8, MOVE>), grid, dim3(512), 0, s, a, mv);
  else if (a.c.cap <= 16384)
    hipLaunchKernelGGL((kv_select_kernel<1024, 16, MOVE>), grid, dim3(1024), 0, s, a, mv);
  else
    hipLaunchKernelGGL((kv_select_kernel<1024, 32, MOVE>), grid, dim3(1024), 0, s, a, mv);
}

hipError_t launch_kv_evict(const KvEvictArgs& a, const KvWorkspace& w, uint32_t hd, hipStream_t s) {
  auto meet = [](const void* p, const void* q, size_t n) {  // n words from p, from q
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    return x < y + 4 * n && y < x + 4 * n;
  };
  const uint32_t seqs = a.layers * a.c.R * a.s.G;
  const size_t words = size_t(seqs) * a.c.cap;
  const bool in_place = meet(a.scores, a.scores_out, words) || meet(a.positions, a.positions_out, words);
  const bool lens_in_place = meet(a.c.lens, a.lens_out, a.c.R);
  KvMove mv{};
  mv.max_moves = a.keep < a.c.cap ? min(a.keep, a.c.cap - a.keep) : 0u;
  mv.pieces = hd * a.elem / 16;
  mv.moves = w.moves;
  mv.counts = w.counts;
  if (seqs >= KV_LISTS || (!in_place && !lens_in_place)) {
    mv.lens = !lens_in_place;
    const uint32_t parts = in_place ? 1u : min((KV_LISTS + seqs - 1) / seqs, max(1u, mv.max_moves / 16));
    select_launch<true>(a, mv, dim3(seqs, parts), s);
    if (lens_in_place) hipLaunchKernelGGL(kv_lens_kernel, dim3(1), dim3(256), 0, s, a);
    return hipGetLastError();
  }
  select_launch<false>(a, mv, dim3(seqs), s);  // (fewer than KV_LISTS caches)
  hipLaunchKernelGGL(kv_move_kernel, dim3(max(1u, min(64u, mv.max_moves * mv.pieces / 256)), seqs), dim3(256), 0, s, a, mv);
  return hipGetLastError();
}

hipError_t launch_kv_take_errors(uint32_t* err, uint32_t* taken, hipStream_t s) {
  hipLaunchKernelGGL(kv_take_errors_kernel, dim3(1), dim3(1), 0, s, err, taken);
  return hipGetLastError();
}

}  // namespace s2
