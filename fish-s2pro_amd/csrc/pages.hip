// pages.hip -- a KV cache in pages, keys and values in 4 bits, for gfx950 (CDNA4,
// wave64): head norms, rotation and cache write of a batch's new tokens; attention
// over the requests' pages; the rows of pages made anew; a pool compacted.

#include "kv_dev.h"
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

// One block per token and run of heads (blockIdx.y, every gridDim.y-th 16 or 32), 8
// elements per thread.  Norms, angles, rotation and what is rounded to 4 bits are in
// 64 bits: a rounding of f32 in front would move a code across a border now and then,
// and the value by a sixteenth of its block's range.
template <int HD>
__global__ __launch_bounds__(256) void pg_append_kernel(PgAppendArgs a) {
  constexpr uint32_t LP = HD / 8;     // lanes per head
  constexpr uint32_t HPB = 256 / LP;  // heads per step of the block
  __shared__ double2 turn[HD / 2];
  const uint32_t tid = threadIdx.x, b = blockIdx.x / a.c.n, t = blockIdx.x % a.c.n;
  const Request r = request_of(a.c, b, tid == 0 && t == 0 && blockIdx.y == 0 ? a.s.err : nullptr);
  if (t >= r.fresh) return;
  const int32_t pos = a.positions[size_t(b) * a.c.n + t];
  if (pos < 0) {
    if (tid == 0 && blockIdx.y == 0) atomicOr(a.s.err, S2HIP_PAGES_ERR_POSITION);
    return;
  }
  const uint32_t slot = r.len - r.fresh + t, half = a.rope.dims / 2;
  const uint32_t page = uint32_t(a.p.table[size_t(b) * a.p.width + (slot >> a.p.shift)]);
  const bool there = page < a.p.pages;
  if (!there && tid == 0 && blockIdx.y == 0) atomicOr(a.s.err, S2HIP_PAGES_ERR_PAGE);
  if (tid < half) {
    const double angle = double(pos) * a.rope.turns[tid];
    double sn, cs;
    sincospi(2.0 * (angle - rint(angle)), &sn, &cs);
    turn[tid] = make_double2(cs * a.rope.gain, sn * a.rope.gain);
  }
  __syncthreads();
  const uint32_t heads = a.s.H + 2 * a.s.G, l = tid % LP, d0 = 8 * l;
  const float* src = a.qkv + (size_t(b) * a.c.n + t) * heads * HD;
  for (uint32_t h = blockIdx.y * HPB + tid / LP; h < heads; h += HPB * gridDim.y) {  // whole rows of LP lanes take part
    const float* row = src + size_t(h) * HD;
    double x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = row[d0 + e];
    const bool value = h >= a.s.H + a.s.G;
    if (!value) {
      double f = 1.0;
      const float* gain = h < a.s.H ? a.q_norm : a.k_norm;
      if (gain) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fma(x[e], x[e], ss);
#pragma unroll
        for (uint32_t m = 1; m < LP; m *= 2) ss += __shfl_xor(ss, int(m), 64);
        f = 1.0 / sqrt(ss * (1.0 / HD) + double(a.s.eps));
      }
      auto normed = [&](uint32_t d) { return gain ? double(row[d]) * f * double(gain[d]) : double(row[d]); };
      double y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t d = d0 + e;
        y[e] = normed(d);
        if (d < a.rope.dims) {
          const uint32_t i = a.rope.half ? (d < half ? d : d - half) : d / 2;
          const bool second = a.rope.half ? d >= half : d % 2;
          const double other = normed(a.rope.half ? (second ? d - half : d + half) : d ^ 1u);
          const double2 cs = turn[i];
          y[e] = second ? other * cs.y + y[e] * cs.x : y[e] * cs.x - other * cs.y;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = y[e];
    }
    if (h < a.s.H) {
      float* dst = a.q_out + ((size_t(b) * a.c.n + t) * a.s.H + h) * HD + d0;
      *reinterpret_cast<float4*>(dst) = make_float4(float(x[0]), float(x[1]), float(x[2]), float(x[3]));
      *reinterpret_cast<float4*>(dst + 4) = make_float4(float(x[4]), float(x[5]), float(x[6]), float(x[7]));
      continue;
    }
    // the group's largest by size (4 lanes), the first of equals
    double big = 0.0;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      big = fmax(big, fabs(x[e]));
      odd |= !(fabs(x[e]) < 65408.0);
    }
    big = fmax(big, __shfl_xor(big, 1, 64));
    big = fmax(big, __shfl_xor(big, 2, 64));
    int first = 1 << 20;  // place in the group, doubled, + 1 of a negative one
#pragma unroll
    for (int e = 7; e >= 0; --e)
      if (fabs(x[e]) == big) first = 2 * int(8 * (l % 4) + e) + (x[e] < 0.0 ? 1 : 0);
    int any = odd;
#pragma unroll
    for (int m = 1; m < 4; m *= 2) {
      first = min(first, __shfl_xor(first, m, 64));
      any |= __shfl_xor(any, m, 64);
    }
    odd = any != 0;
    double d = rounded8(big * 0.125);
    if (!(first & 1)) d = -d;
    uint32_t code[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) code[e] = odd || d == 0.0 ? 8u : uint32_t(int(fmin(fmax(rint(x[e] / d), -8.0), 7.0)) + 8);
    const float scale = odd ? NAN : float(d);
    const uint32_t g = value ? h - a.s.H - a.s.G : h - a.s.H, j = l / 4;
    float* held = value ? a.v_held : a.k_held;
    if (held) {
      held += ((size_t(b) * a.c.n + t) * a.s.G + g) * HD + d0;
#pragma unroll
      for (int e = 0; e < 8; ++e) held[e] = scale * float(int(code[e]) - 8);
    }
    if (!there) continue;
    if (odd) atomicOr(a.s.err, S2HIP_PAGES_ERR_RANGE);
    const Chunk<HD> at{a.p.shift};
    uint8_t* part = a.p.pool + (size_t(page) * a.s.G + g) * a.p.chunk;
    const uint32_t s = slot & ((1u << a.p.shift) - 1u);
    if (!value) {
      uint32_t word = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) word |= code[e] << (e / 2 * 4 + e % 2 * 16);
      *reinterpret_cast<uint32_t*>(part + ((s * 4 + l % 4) * (HD / 32) + j) * 4) = word;
      if (l % 4 == 0) *reinterpret_cast<_Float16*>(part + at.ks() + (s * (HD / 32) + j) * 2) = _Float16(scale);
    } else {
      const uint32_t quad = s / 4, one = s % 4;  // (16 u + 4 i = 4 quad)
#pragma unroll
      for (uint32_t m = 0; m < 4; ++m)
        part[at.v() + ((quad * 16 + 4 * (l % 4) + m) * (HD / 32) + j) * 4 + one] = uint8_t(code[2 * m] | code[2 * m + 1] << 4);
      if (l % 4 == 0) *reinterpret_cast<_Float16*>(part + at.vs() + ((quad * (HD / 32) + j) * 4 + one) * 2) = _Float16(scale);
    }
  }
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// A wave per query row: 64 keys at a time, one per lane, then their values, two
// elements per lane.
template <int HD>
__global__ __launch_bounds__(64) void pg_attend_kernel(PgAttendArgs pa) {
  const KvAttendArgs& a = pa.a;
  __shared__ float qs[HD], ps[64];
  const uint32_t lane = threadIdx.x, h = blockIdx.x % a.s.H, bt = blockIdx.x / a.s.H, b = bt / a.c.n, t = bt % a.c.n, g = h / a.s.rep;
  const Request r = request_of(a.c, b, lane == 0 ? a.s.err : nullptr);
  if (t >= r.fresh) return;
  for (uint32_t d = lane; d < HD; d += 64) qs[d] = a.q[size_t(blockIdx.x) * HD + d] * a.s.scale2;
  __syncthreads();
  const Chunk<HD> at{pa.p.shift};
  const uint32_t keys = r.len - r.fresh + t + 1, mask = (1u << pa.p.shift) - 1u;
  auto page_of = [&](uint32_t key) { return uint32_t(pa.p.table[size_t(b) * pa.p.width + (key >> pa.p.shift)]); };
  float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
  for (uint32_t k0 = 0; k0 < keys; k0 += 64) {
    const uint32_t key = k0 + lane;
    float s = -INFINITY;
    if (key < keys) {
      const uint32_t page = page_of(key), slot = key & mask;
      if (page < pa.p.pages) {
        const uint8_t* part = pa.p.pool + (size_t(page) * a.s.G + g) * pa.p.chunk;
        s = 0.0f;
        for (uint32_t j = 0; j < HD / 32; ++j) {
          const float d = float(*reinterpret_cast<const _Float16*>(part + at.ks() + (slot * (HD / 32) + j) * 2));
          for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(part + ((slot * 4 + i) * (HD / 32) + j) * 4);
            for (int e = 0; e < 8; ++e) s = fmaf(d * float(int((word >> (e / 2 * 4 + e % 2 * 16)) & 15u) - 8), qs[32 * j + 8 * i + e], s);
          }
        }
      } else {
        atomicOr(a.s.err, S2HIP_PAGES_ERR_PAGE);
      }
    }
    const float mn = fmaxf(m, wave_max(s));
    const float base = mn == -INFINITY ? 0.0f : mn, f = __builtin_amdgcn_exp2f((m == -INFINITY ? base : m) - base);
    const float p = __builtin_amdgcn_exp2f(s - base);
    l = l * f + wave_sum(p);
    m = mn;
    ps[lane] = p;
    __syncthreads();
    o[0] *= f;
    o[1] *= f;
    for (uint32_t k = k0; k < min(keys, k0 + 64) && lane < HD / 2; ++k) {
      const uint32_t page = page_of(k), slot = k & mask;
      if (page >= pa.p.pages) continue;
      const uint8_t* part = pa.p.pool + (size_t(page) * a.s.G + g) * pa.p.chunk;
      const uint32_t quad = slot / 4, one = slot % 4, j = lane / 16;
      const uint32_t c = part[at.v() + ((quad * 16 + lane % 16) * (HD / 32) + j) * 4 + one];
      const float d = float(*reinterpret_cast<const _Float16*>(part + at.vs() + ((quad * (HD / 32) + j) * 4 + one) * 2));
      o[0] = fmaf(ps[k - k0], d * float(int(c & 15u) - 8), o[0]);
      o[1] = fmaf(ps[k - k0], d * float(int(c >> 4) - 8), o[1]);
    }
    __syncthreads();
  }
  const float inv = m == -INFINITY ? NAN : 1.0f / l;
  if (lane < HD / 2) *reinterpret_cast<float2*>(a.out + size_t(blockIdx.x) * HD + 2 * lane) = make_float2(o[0] * inv, o[1] * inv);
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

// Nothing changes: arrays out become as those in.
__device__ __forceinline__ void copy_rows(const PgUpdateArgs& a) {
  const uint32_t tid = threadIdx.x;
  if (a.refs_out != a.refs)
    for (uint32_t p = tid; p < a.p.pages; p += ROWS_THREADS) a.refs_out[p] = a.refs[p];
  if (a.table_out != a.p.table)
    for (uint32_t i = tid; i < a.R * a.p.width; i += ROWS_THREADS) a.table_out[i] = a.p.table[i];
  if (a.lens_out && a.lens_out != a.lens && tid < a.R) a.lens_out[tid] = a.lens[tid];
}

// One block.  References are counted in the workspace: what rows let go of is taken
// off, what they take added; the rest of a row that stays its own is not looked at
// twice.  Of w rows that write to a page of r references, the first r - 1 write to
// copies: the last writes in place if no one else holds it.
__global__ __launch_bounds__(ROWS_THREADS) void pg_update_kernel(PgUpdateArgs a, PgWorkspace w) {
  __shared__ int32_t source[MAX_ROWS], lens[MAX_ROWS], kept[MAX_ROWS], total[MAX_ROWS], last[MAX_ROWS];
  __shared__ uint32_t first[MAX_ROWS], offset[MAX_ROWS], bad;
  const uint32_t tid = threadIdx.x, width = a.p.width, page_up = (1u << a.p.shift) - 1u;
  const int64_t cap = int64_t(width) << a.p.shift;
  auto pages_of = [&](int32_t n) { return (uint32_t(n) + page_up) >> a.p.shift; };
  auto report = [&](uint32_t bits) { atomicOr(&bad, bits); };
  if (tid == 0) bad = 0;
  __syncthreads();
  int32_t keep = 0, add = 0;
  if (tid < a.R) {
    source[tid] = a.source ? a.source[tid] : int32_t(tid);
    lens[tid] = a.lens[tid];
    keep = a.keep ? a.keep[tid] : 0x7fffffff;
    add = a.add ? a.add[tid] : 0;
    w.moves[2 * tid] = -1;
    if (lens[tid] < 0 || lens[tid] > cap || source[tid] < -1 || source[tid] >= int32_t(a.R) || keep < 0 || add < 0) report(S2HIP_PAGES_ERR_LENS);
  }
  for (uint32_t p = tid; p < a.p.pages; p += ROWS_THREADS) w.refs[p] = a.refs[p];
  auto stops = [&] {
    const uint32_t why = settled(bad);
    if (why) copy_rows(a);
    if (why && tid == 0) atomicOr(a.err, why);
    return why != 0;
  };
  if (stops()) return;
  if (tid < a.R) {
    kept[tid] = source[tid] < 0 ? 0 : min(keep, lens[source[tid]]);
    if (int64_t(kept[tid]) + add > cap) report(S2HIP_PAGES_ERR_LENS);
    total[tid] = int32_t(uint32_t(kept[tid]) + uint32_t(add));
  }
  if (stops()) return;
  for (uint32_t x = tid; x < a.R * width; x += ROWS_THREADS) {
    const uint32_t b = x / width, i = x % width;
    const int32_t s = source[b];
    const bool old = i < pages_of(lens[b]), base = i < pages_of(kept[b]);
    const int32_t e = old ? a.p.table[x] : -1, v = !base ? -1 : s == int32_t(b) ? e : a.p.table[size_t(s) * width + i];
    const bool e_in = uint32_t(e) < a.p.pages, v_in = uint32_t(v) < a.p.pages;
    if ((old && !e_in) || (base && !v_in)) report(S2HIP_PAGES_ERR_PAGE);
    if (s != int32_t(b) || !base) {
      if (old && e_in) atomicSub(&w.refs[e], 1);
      if (base && v_in) atomicAdd(&w.refs[v], 1);
    }
    w.table[x] = v;
  }
  if (stops()) return;
  for (uint32_t x = tid; x < a.R * width; x += ROWS_THREADS) {
    const uint32_t b = x / width, i = x % width;
    if (i < pages_of(kept[b]) && load_now(&w.refs[w.table[x]]) < 1) report(S2HIP_PAGES_ERR_REFS);
    if (i < pages_of(lens[b]) && load_now(&w.refs[a.p.table[x]]) < 0) report(S2HIP_PAGES_ERR_REFS);
  }
  const bool grows = tid < a.R && add > 0 && (uint32_t(kept[tid]) & page_up) != 0;
  if (tid < a.R) last[tid] = grows ? w.table[size_t(tid) * width + (uint32_t(kept[tid]) >> a.p.shift)] : -1;
  __syncthreads();
  uint32_t needs = 0, copies = 0;
  if (tid < a.R) {
    if (grows) {
      int32_t before = 0;
      for (uint32_t b = 0; b < tid; ++b) before += last[b] == last[tid];
      copies = before < load_now(&w.refs[last[tid]]) - 1;
    }
    first[tid] = pages_of(kept[tid]) - copies;
    needs = pages_of(total[tid]) - first[tid];
  }
  uint32_t all, found = 0;
  const uint32_t begin = block_scan(needs, all);
  if (tid < a.R) offset[tid] = begin;
  for (uint32_t p0 = 0; p0 < a.p.pages && found < all; p0 += ROWS_THREADS) {
    const bool free = p0 + tid < a.p.pages && load_now(&w.refs[p0 + tid]) == 0;
    uint32_t more;
    const uint32_t rank = found + block_scan(free, more);
    if (free && rank < all) w.list[rank] = int32_t(p0 + tid);
    found += more;
  }
  if (found < all && tid == 0) report(S2HIP_PAGES_ERR_FULL);
  if (stops()) return;
  for (uint32_t p = tid; p < a.p.pages; p += ROWS_THREADS) a.refs_out[p] = load_now(&w.refs[p]);
  settled();
  for (uint32_t x = tid; x < a.R * width; x += ROWS_THREADS) {
    const uint32_t b = x / width, i = x % width;
    int32_t v = w.table[x];
    if (i >= first[b] && i < pages_of(total[b])) {
      v = w.list[offset[b] + i - first[b]];
      a.refs_out[v] = 1;
    }
    a.table_out[x] = v;
  }
  if (tid < a.R) {
    a.lens_out[tid] = total[tid];
    if (copies) {
      w.moves[2 * tid] = last[tid];
      w.moves[2 * tid + 1] = w.list[offset[tid]];
      atomicSub(&a.refs_out[last[tid]], 1);
    }
  }
}

__device__ __forceinline__ void copy_page(const PgUpdateArgs& a, uint32_t layer, int32_t from, int32_t to, uint32_t bytes, uint32_t i0, uint32_t step) {
  uint8_t* pool = a.p.pool + layer * a.layer_stride;
  const u32x4* src = reinterpret_cast<const u32x4*>(pool + size_t(from) * bytes);
  u32x4* dst = reinterpret_cast<u32x4*>(pool + size_t(to) * bytes);
  for (uint32_t i = i0; i < bytes / 16; i += step) dst[i] = src[i];
}

// blockIdx.y = row, z = layer
__global__ __launch_bounds__(256) void pg_copy_kernel(PgUpdateArgs a, const int32_t* moves, uint32_t bytes) {
  const int32_t from = moves[2 * blockIdx.y];
  if (from >= 0) copy_page(a, blockIdx.z, from, moves[2 * blockIdx.y + 1], bytes, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// One block: the pages in use, the lists of holes and movers, refs.
__global__ __launch_bounds__(ROWS_THREADS) void pg_pack_kernel(PgUpdateArgs a, PgWorkspace w) {
  __shared__ uint32_t bad;
  const uint32_t tid = threadIdx.x, width = a.p.width, page_up = (1u << a.p.shift) - 1u;
  if (tid == 0) bad = 0;
  __syncthreads();
  uint32_t mine = 0, used;
  for (uint32_t p = tid; p < a.p.pages; p += ROWS_THREADS) {
    const int32_t r = a.refs[p];
    mine += r > 0;
    if (r < 0) atomicOr(&bad, S2HIP_PAGES_ERR_REFS);
  }
  for (uint32_t x = tid; x < a.R * width; x += ROWS_THREADS) {
    const int32_t len = a.lens[x / width];
    if (len < 0 || int64_t(len) > int64_t(width) << a.p.shift) {
      atomicOr(&bad, S2HIP_PAGES_ERR_LENS);
    } else if (x % width < (uint32_t(len) + page_up) >> a.p.shift) {
      const int32_t e = a.p.table[x];
      if (uint32_t(e) >= a.p.pages)
        atomicOr(&bad, S2HIP_PAGES_ERR_PAGE);
      else if (a.refs[e] < 1)
        atomicOr(&bad, S2HIP_PAGES_ERR_REFS);
    }
  }
  block_scan(mine, used);
  const uint32_t why = settled(bad);
  if (tid == 0) a.used_out[0] = int32_t(used);
  if (why) {
    if (tid == 0) {
      w.moves[0] = 0;
      w.moves[1] = 0x7fffffff;  // no entry follows
      atomicOr(a.err, why);
    }
    if (a.refs_out != a.refs)
      for (uint32_t p = tid; p < a.p.pages; p += ROWS_THREADS) a.refs_out[p] = a.refs[p];
    if (a.moved_to)
      for (uint32_t p = tid; p < a.p.pages; p += ROWS_THREADS) a.moved_to[p] = a.refs[p] > 0 ? int32_t(p) : -1;
    return;
  }
  uint32_t holes = 0, movers = 0;
  for (uint32_t p0 = 0; p0 < a.p.pages; p0 += ROWS_THREADS) {
    const uint32_t p = p0 + tid;
    const int32_t r = p < a.p.pages ? a.refs[p] : 0;
    const bool hole = p < used && r == 0, mover = p >= used && r > 0;
    uint32_t all;
    const uint32_t rank = block_scan(uint32_t(hole) | uint32_t(mover) << 16, all);
    if (hole) w.list[holes + (rank & 0xffffu)] = int32_t(p);
    if (mover) w.list[a.p.pages + movers + (rank >> 16)] = int32_t(p);
    holes += all & 0xffffu;
    movers += all >> 16;
  }
  settled();
  for (uint32_t p = tid; p < a.p.pages; p += ROWS_THREADS) {
    const int32_t r = a.refs[p];
    if (a.refs_out != a.refs) a.refs_out[p] = p < used ? r : 0;
    if (a.moved_to) a.moved_to[p] = r > 0 ? int32_t(p) : -1;
  }
  settled();
  for (uint32_t i = tid; i < movers; i += ROWS_THREADS) {
    const int32_t from = w.list[a.p.pages + i], to = w.list[i], r = a.refs[from];
    a.refs_out[to] = r;
    a.refs_out[from] = 0;
    w.refs[from] = to;
    if (a.moved_to) a.moved_to[from] = to;
  }
  if (tid == 0) {
    w.moves[0] = int32_t(movers);
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
    const uint32_t tokens = a.c.R * a.c.n, steps = (a.s.H + 2 * a.s.G + 2048 / HD() - 1) / (2048 / HD());
    hipLaunchKernelGGL(pg_append_kernel<HD()>, dim3(tokens, min(steps, max(1u, 512 / tokens))), dim3(256), 0, s, a);
    return hipGetLastError();
  });
}

hipError_t launch_pg_attend(uint32_t hd, const PgAttendArgs& a, const PgWorkspace&, hipStream_t s) {
  return by_dim(hd, [&](auto HD) {
    hipLaunchKernelGGL(pg_attend_kernel<HD()>, dim3(a.a.c.R * a.a.c.n * a.a.s.H), dim3(64), 0, s, a);
    return hipGetLastError();
  });
}

hipError_t launch_pg_update(const PgUpdateArgs& a, const PgWorkspace& w, uint32_t page_bytes, hipStream_t s) {
  hipLaunchKernelGGL(pg_update_kernel, dim3(1), dim3(ROWS_THREADS), 0, s, a, w);
  hipLaunchKernelGGL(pg_copy_kernel, dim3((page_bytes + 16383) / 16384, a.R, a.layers), dim3(256), 0, s, a, w.moves, page_bytes);
  return hipGetLastError();
}

hipError_t launch_pg_compact(const PgUpdateArgs& a, const PgWorkspace& w, uint32_t page_bytes, hipStream_t s) {
  hipLaunchKernelGGL(pg_pack_kernel, dim3(1), dim3(ROWS_THREADS), 0, s, a, w);
  hipLaunchKernelGGL(pg_move_kernel, dim3(2048), dim3(256), 0, s, a, w, page_bytes);
  return hipGetLastError();
}

}  // namespace s2
