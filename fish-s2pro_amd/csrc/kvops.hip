// kvops.hip -- KV-cache operators for gfx950 (CDNA4, wave64): head norms,
// rotation and cache write of a batch's new tokens; attention over a shared
// prefix and the requests' own caches, with or without the keys' weights;
// eviction by score.

#include <type_traits>

#include "kvops.h"
#include "s2hip.h"
#include "wave.h"

namespace s2 {
namespace {

// Slots in use and new tokens of request b; a request out of range has none.
struct Request {
  uint32_t len, fresh;
};
__device__ __forceinline__ Request request_of(const KvCaches& c, uint32_t b, uint32_t* err) {
  const int32_t len = c.lens[b];
  const int32_t fresh = c.new_lens ? c.new_lens[b] : len == 0 ? 0 : int32_t(c.n);
  const bool ok = len >= 0 && len <= int32_t(c.cap) && fresh >= 0 && fresh <= int32_t(c.n) && fresh <= len;
  if (!ok && err) atomicOr(err, S2HIP_KV_ERR_LENS);
  return ok ? Request{uint32_t(len), uint32_t(fresh)} : Request{0u, 0u};
}

template <bool KH>
using Elem = std::conditional_t<KH, _Float16, float>;

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// One block per token: the token's hd / 2 angles once (64-bit product with the
// position, whole turns taken off in 64 bits, cos and sin of the rest in f32),
// then 4 elements (two pairs) per thread.
template <int HD, bool KH>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a) {
  constexpr uint32_t LP = HD / 4;       // lanes per head
  constexpr uint32_t HPB = 256 / LP;    // heads per step of the block
  __shared__ float2 turn[HD / 2];
  const uint32_t tid = threadIdx.x, b = blockIdx.x / a.c.n, t = blockIdx.x % a.c.n;
  const Request r = request_of(a.c, b, tid == 0 && t == 0 ? a.s.err : nullptr);
  if (t >= r.fresh) return;
  const uint32_t slot = r.len - r.fresh + t;
  const int32_t pos = a.positions[size_t(b) * a.c.n + t];
  if (pos < 0) {
    if (tid == 0) atomicOr(a.s.err, S2HIP_KV_ERR_POSITION);
    return;
  }
  if (tid < HD / 2) {
    const double angle = double(pos) * a.s.freq[tid] * 0.15915494309189535;  // in turns
    const float rest = float(angle - rint(angle));
    float sn, cs;
    sincospif(2.0f * rest, &sn, &cs);
    turn[tid] = make_float2(cs, sn);
  }
  __syncthreads();
  const uint32_t heads = a.s.H + 2 * a.s.G, d = 4 * (tid % LP);
  const float* src = a.qkv + (size_t(b) * a.c.n + t) * heads * HD;
  for (uint32_t h = tid / LP; h < heads; h += HPB) {  // whole rows of 16 lanes take part
    float4 x = *reinterpret_cast<const float4*>(src + size_t(h) * HD + d);
    if (h < a.s.H + a.s.G) {
      if (a.q_norm) {
        float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
        ss = row_reduce(ss, [](float p, float q) { return p + q; });
        if constexpr (LP == 32) ss += __shfl_xor(ss, 16, 64);
        const float f = rsqrtf(ss * (1.0f / HD) + a.s.eps);
        const float4 gain = *reinterpret_cast<const float4*>((h < a.s.H ? a.q_norm : a.k_norm) + d);
        x = make_float4(x.x * f * gain.x, x.y * f * gain.y, x.z * f * gain.z, x.w * f * gain.w);
      }
      const float2 t0 = turn[d / 2], t1 = turn[d / 2 + 1];
      x = make_float4(x.x * t0.x - x.y * t0.y, x.x * t0.y + x.y * t0.x, x.z * t1.x - x.w * t1.y, x.z * t1.y + x.w * t1.x);
    }
    if (h < a.s.H) {
      *reinterpret_cast<float4*>(a.q_out + ((size_t(b) * a.c.n + t) * a.s.H + h) * HD + d) = x;
      continue;
    }
    const bool key = h < a.s.H + a.s.G;
    const uint32_t g = key ? h - a.s.H : h - a.s.H - a.s.G;
    Elem<KH>* dst = static_cast<Elem<KH>*>(key ? a.c.k : a.c.v) + b * a.c.req_stride + g * a.c.head_stride + slot * a.c.slot_stride + d;
    if constexpr (KH) {
      typedef _Float16 half4 __attribute__((ext_vector_type(4)));
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
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
template <int HD, class T>
__device__ __forceinline__ float dot_row(const T* row, const float* q) {
  float s = 0.0f;
  for (int d = 0; d < HD; ++d) s = fmaf(float(row[d]), q[d], s);
  return s;
}

__device__ __forceinline__ float block_max(float v, float* sh) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}
__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// One block per (token, query head): chunks of 256 keys, one per thread, with
// the running maximum and sum of the softmax; then a dimension per thread.
template <int HD, bool KH>
__global__ __launch_bounds__(256) void kv_attend_row_kernel(KvAttendArgs a, float* stat) {
  using T = Elem<KH>;
  constexpr uint32_t PARTS = 256 / HD;
  __shared__ float qs[HD], ps[256], sh[4], os[256];
  const uint32_t tid = threadIdx.x, h = blockIdx.x % a.s.H, bt = blockIdx.x / a.s.H, b = bt / a.c.n, t = bt % a.c.n;
  const uint32_t g = h / a.s.rep;
  const Request r = request_of(a.c, b, tid == 0 && t == 0 && h == 0 ? a.s.err : nullptr);
  if (t >= r.fresh) return;
  const uint32_t own = r.len - r.fresh + t + 1, total = a.c.P + own;
  if (tid < HD) qs[tid] = a.q[size_t(blockIdx.x) * HD + tid];
  __syncthreads();
  const T* pk = static_cast<const T*>(a.c.pk) + g * a.c.p_head_stride;
  const T* pv = static_cast<const T*>(a.c.pv) + g * a.c.p_head_stride;
  const T* k = static_cast<const T*>(a.c.k) + b * a.c.req_stride + g * a.c.head_stride;
  const T* v = static_cast<const T*>(a.c.v) + b * a.c.req_stride + g * a.c.head_stride;
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  const uint32_t d = tid % HD, part = tid / HD;
  for (uint32_t k0 = 0; k0 < total; k0 += 256) {
    const uint32_t i = k0 + tid, nk = min(256u, total - k0);
    float s = -INFINITY;
    if (i < total)
      s = a.s.scale * dot_row<HD>(i < a.c.P ? pk + i * a.c.p_slot_stride : k + (i - a.c.P) * a.c.slot_stride, qs);
    const float mn = fmaxf(m, block_max(s, sh));
    const float p = i < total && mn != -INFINITY ? expf(s - mn) : 0.0f;
    const float corr = m == -INFINITY ? 0.0f : expf(m - mn);
    l = l * corr + block_sum(p, sh);
    o *= corr;
    m = mn;
    ps[tid] = p;
    __syncthreads();
    for (uint32_t j = part; j < nk; j += PARTS) {
      const uint32_t key = k0 + j;
      const T* row = key < a.c.P ? pv + key * a.c.p_slot_stride : v + (key - a.c.P) * a.c.slot_stride;
      o = fmaf(ps[j], float(row[d]), o);
    }
    __syncthreads();
  }
  os[tid] = o;
  __syncthreads();
  if (tid < HD) {
    float sum = 0.0f;
    for (uint32_t j = 0; j < PARTS; ++j) sum += os[tid + HD * j];
    a.out[size_t(blockIdx.x) * HD + tid] = sum / l;
  }
  if (stat && tid == 0) {
    stat[2 * size_t(blockIdx.x)] = m;
    stat[2 * size_t(blockIdx.x) + 1] = l;
  }
}

// A key per thread: its weight in every row that sees it.  blockIdx.z = request,
// or R for the prefix.
template <int HD, bool KH>
__global__ __launch_bounds__(256) void kv_weigh_row_kernel(KvAttendArgs a, const float* stat) {
  using T = Elem<KH>;
  __shared__ float qs[HD], ml[2];
  const uint32_t tid = threadIdx.x, g = blockIdx.y, z = blockIdx.z, i = blockIdx.x * 256 + tid;
  const bool prefix = z == a.c.R;
  const uint32_t b0 = prefix ? 0 : z, b1 = prefix ? a.c.R : z + 1;
  const uint32_t n_keys = prefix ? a.c.P : request_of(a.c, z, nullptr).len;
  if (blockIdx.x * 256 >= n_keys) return;
  const T* row = prefix ? static_cast<const T*>(a.c.pk) + g * a.c.p_head_stride + min(i, n_keys - 1) * a.c.p_slot_stride
                        : static_cast<const T*>(a.c.k) + z * a.c.req_stride + g * a.c.head_stride + min(i, n_keys - 1) * a.c.slot_stride;
  float w = 0.0f;
  for (uint32_t b = b0; b < b1; ++b) {
    const Request r = request_of(a.c, b, nullptr);
    for (uint32_t t = 0; t < r.fresh; ++t)
      for (uint32_t h = g * a.s.rep; h < (g + 1) * a.s.rep; ++h) {
        const size_t at = (size_t(b) * a.c.n + t) * a.s.H + h;
        __syncthreads();
        if (tid < HD) qs[tid] = a.q[at * HD + tid];
        if (tid < 2) ml[tid] = stat[2 * at + tid];
        __syncthreads();
        if (prefix || i <= r.len - r.fresh + t) w += expf(a.s.scale * dot_row<HD>(row, qs) - ml[0]) / ml[1];
      }
  }
  if (i >= n_keys) return;
  const size_t at = prefix ? size_t(g) * a.pw_stride + i : (size_t(z) * a.s.G + g) * a.c.cap + i;
  const float* in = prefix ? a.pw_in : a.w_in;
  (prefix ? a.pw_out : a.w_out)[at] = (in ? in[at] : 0.0f) + w;
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

// Exclusive sum over the block's 1024 threads in thread order; total for all.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* sh, uint32_t& total) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  uint32_t x = v;
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(x, d, 64);
    if (lane >= uint32_t(d)) x += y;
  }
  __syncthreads();
  if (lane == 63) sh[wave] = x;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
  for (uint32_t w = 0; w < 16; ++w) {
    if (w < wave) before += sh[w];
    total += sh[w];
  }
  return before + x - v;
}

// One block per (layer, request, kv head): thread t holds slots I t .. I t + I - 1.
// The k-th largest score among the slots that compete (the safe ones all stay,
// the others compete for the rest) by four digits of 8 bits from the top; of the
// slots that equal it the lowest stay.  Then the freed slots below m and the
// kept ones from m on are counted off in slot order: the x-th of one takes the
// x-th of the other.
template <int I>
__global__ __launch_bounds__(1024) void kv_select_kernel(KvEvictArgs a, uint32_t seq0, uint32_t max_moves, uint32_t* moves, uint32_t* counts) {
  __shared__ uint32_t sh[16], hist[256], pick[2];
  __shared__ int32_t top[16];
  const uint32_t tid = threadIdx.x, sg = seq0 + blockIdx.x, g = sg % a.s.G, lb = sg / a.s.G, b = lb % a.c.R;
  const uint32_t lane = tid & 63u, wave = tid >> 6;
  const int32_t in_use = a.c.lens[b];
  const bool ok = in_use >= 0 && in_use <= int32_t(a.c.cap);
  if (!ok && tid == 0 && lb == b && g == 0) atomicOr(a.s.err, S2HIP_KV_ERR_LENS);
  const uint32_t n = ok ? uint32_t(in_use) : 0u, m = min(n, a.keep);
  if (tid == 0) counts[2 * blockIdx.x + 1] = ok ? m : 0xffffffffu;
  const size_t base = size_t(sg) * a.c.cap;
  float sc[I];
  int32_t pos[I];
  uint32_t bits[I];
  int32_t newest = INT32_MIN;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const uint32_t s = tid * I + i;
    sc[i] = s < n ? a.scores[base + s] : 0.0f;
    pos[i] = s < n ? a.positions[base + s] : INT32_MIN;
    bits[i] = score_bits(sc[i]);
    newest = max(newest, pos[i]);
  }
  if (n <= a.keep) {  // nothing to cut
    if (tid == 0) counts[2 * blockIdx.x] = 0;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint32_t s = tid * I + i;
      if (s < n) {
        a.scores_out[base + s] = sc[i];
        a.positions_out[base + s] = pos[i];
      }
    }
    return;
  }
  for (int d = 32; d >= 1; d >>= 1) newest = max(newest, __shfl_xor(newest, d, 64));
  if (lane == 0) top[wave] = newest;
  __syncthreads();
  for (uint32_t w = 0; w < 16; ++w) newest = max(newest, top[w]);
  uint32_t safe = 0, n_safe = 0;  // bit i: slot i of the thread
#pragma unroll
  for (int i = 0; i < I; ++i)
    if (tid * I + i < n && (int64_t(pos[i]) > int64_t(newest) - int64_t(a.recent) || int64_t(pos[i]) < int64_t(a.sinks))) safe |= 1u << i;
  block_scan(__popc(safe), sh, n_safe);
  // who competes for how many places (positions given twice can make more safe slots than there is room)
  const bool room = n_safe <= m;
  uint32_t want = room ? m - n_safe : m;
  uint32_t compete = 0;
#pragma unroll
  for (int i = 0; i < I; ++i)
    if (tid * I + i < n && (((safe >> i) & 1u) == 0) == room) compete |= 1u << i;
  uint32_t prefix = 0, kept = room ? safe : 0u;
  if (want) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < I; ++i)
        if (((compete >> i) & 1u) && (shift == 24 || (bits[i] >> (shift + 8)) == prefix)) atomicAdd(&hist[(bits[i] >> shift) & 255u], 1u);
      __syncthreads();
      if (tid < 64) {  // digits from the top: lane l holds 255 - 4 l .. 252 - 4 l
        uint32_t c[4], x = 0;
        for (int j = 0; j < 4; ++j) x += c[j] = hist[255 - 4 * lane - j];
        uint32_t y = x;
        for (int d = 1; d < 64; d <<= 1) {
          const uint32_t z = __shfl_up(y, d, 64);
          if (lane >= uint32_t(d)) y += z;
        }
        uint32_t above = y - x;
        for (int j = 0; j < 4; ++j) {
          if (above < want && above + c[j] >= want) {
            pick[0] = 255 - 4 * lane - j;
            pick[1] = want - above;
          }
          above += c[j];
        }
      }
      __syncthreads();
      prefix = (prefix << 8) | pick[0];
      want = pick[1];
    }
    uint32_t equal = 0, dummy;
#pragma unroll
    for (int i = 0; i < I; ++i)
      if ((compete >> i) & 1u) {
        if (bits[i] > prefix) kept |= 1u << i;
        if (bits[i] == prefix) equal |= 1u << i;
      }
    uint32_t rank = block_scan(__popc(equal), sh, dummy);
#pragma unroll
    for (int i = 0; i < I; ++i)
      if ((equal >> i) & 1u)
        if (rank++ < want) kept |= 1u << i;
  }
  uint32_t holes = 0, movers = 0;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const uint32_t s = tid * I + i;
    const bool k = (kept >> i) & 1u;
    if (s < m && !k) holes |= 1u << i;
    if (s >= m && s < n && k) movers |= 1u << i;
    if (s < m && k) {
      a.scores_out[base + s] = sc[i];
      a.positions_out[base + s] = pos[i];
    }
  }
  uint32_t n_holes, n_movers;
  uint32_t hr = block_scan(__popc(holes), sh, n_holes), mr = block_scan(__popc(movers), sh, n_movers);
  uint16_t* list = reinterpret_cast<uint16_t*>(moves + size_t(blockIdx.x) * max_moves);  // (to, from) pairs
#pragma unroll
  for (int i = 0; i < I; ++i) {
    if ((holes >> i) & 1u) list[2 * hr++] = uint16_t(tid * I + i);
    if ((movers >> i) & 1u) list[2 * mr++ + 1] = uint16_t(tid * I + i);
  }
  if (tid == 0) counts[2 * blockIdx.x] = n_movers;
  __syncthreads();  // the block's own stores to global memory are visible to it
  for (uint32_t i = tid; i < n_movers; i += 1024) {
    const uint32_t to = list[2 * i], from = list[2 * i + 1];
    a.scores_out[base + to] = a.scores[base + from];
    a.positions_out[base + to] = a.positions[base + from];
  }
}

// Rows of 16-byte pieces; blockIdx.y = (layer, request, kv head) of the launch.
template <int HD, bool KH>
__global__ __launch_bounds__(256) void kv_move_kernel(KvEvictArgs a, uint32_t seq0, uint32_t max_moves, const uint32_t* moves, const uint32_t* counts) {
  using T = Elem<KH>;
  constexpr uint32_t LP = HD * sizeof(T) / 16, RPB = 256 / LP;
  const uint32_t tid = threadIdx.x, sg = seq0 + blockIdx.y, g = sg % a.s.G, lb = sg / a.s.G, l = lb / a.c.R, b = lb % a.c.R;
  const uint32_t n_moves = counts[2 * blockIdx.y], left = counts[2 * blockIdx.y + 1];
  if (blockIdx.x == 0 && tid == 0 && l == 0 && g == 0 && left != 0xffffffffu) a.lens_out[b] = int32_t(left);
  const size_t base = l * a.layer_stride + b * a.c.req_stride + g * a.c.head_stride;
  for (uint32_t i = blockIdx.x * RPB + tid / LP; i < n_moves; i += gridDim.x * RPB) {
    const uint32_t mv = moves[size_t(blockIdx.y) * max_moves + i], to = mv & 0xffffu, from = mv >> 16;
    const size_t d = (tid % LP) * (16 / sizeof(T));
    T* k = static_cast<T*>(a.c.k) + base + d;
    T* v = static_cast<T*>(a.c.v) + base + d;
    const uint4 x = *reinterpret_cast<const uint4*>(k + from * a.c.slot_stride);
    const uint4 y = *reinterpret_cast<const uint4*>(v + from * a.c.slot_stride);
    *reinterpret_cast<uint4*>(k + to * a.c.slot_stride) = x;
    *reinterpret_cast<uint4*>(v + to * a.c.slot_stride) = y;
  }
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
    hipLaunchKernelGGL((kv_append_kernel<HD(), KH()>), dim3(a.c.R * a.c.n), dim3(256), 0, s, a);
    return hipGetLastError();
  });
}

hipError_t launch_kv_attend(uint32_t hd, bool f16, const KvAttendArgs& a, const KvWorkspace& w, hipStream_t s) {
  return by_shape(hd, f16, [&](auto HD, auto KH) {
    hipLaunchKernelGGL((kv_attend_row_kernel<HD(), KH()>), dim3(a.c.R * a.c.n * a.s.H), dim3(256), 0, s, a,
                       a.w_out ? w.stat : nullptr);
    if (a.w_out) {
      const uint32_t keys = a.pw_out ? max(a.c.P, a.c.cap) : a.c.cap;
      hipLaunchKernelGGL((kv_weigh_row_kernel<HD(), KH()>), dim3((keys + 255) / 256, a.s.G, a.c.R + (a.pw_out ? 1 : 0)),
                         dim3(256), 0, s, a, w.stat);
    }
    return hipGetLastError();
  });
}

hipError_t launch_kv_evict(uint32_t hd, bool f16, const KvEvictArgs& a, const KvWorkspace& w, hipStream_t s) {
  const uint32_t seqs = a.layers * a.c.R * a.s.G;
  const uint32_t max_moves = a.keep < a.c.cap ? min(a.keep, a.c.cap - a.keep) : 0u;
  // as many caches per launch as the lists have room for
  const uint32_t per = uint32_t(min(max_moves ? w.cap_moves / max_moves : w.cap_seqs, w.cap_seqs));
  for (uint32_t s0 = 0; s0 < seqs; s0 += per) {
    const uint32_t ns = min(per, seqs - s0);
    const dim3 grid(ns), block(1024);
    if (a.c.cap <= 1024)
      hipLaunchKernelGGL((kv_select_kernel<1>), grid, block, 0, s, a, s0, max_moves, w.moves, w.counts);
    else if (a.c.cap <= 4096)
      hipLaunchKernelGGL((kv_select_kernel<4>), grid, block, 0, s, a, s0, max_moves, w.moves, w.counts);
    else if (a.c.cap <= 16384)
      hipLaunchKernelGGL((kv_select_kernel<16>), grid, block, 0, s, a, s0, max_moves, w.moves, w.counts);
    else
      hipLaunchKernelGGL((kv_select_kernel<32>), grid, block, 0, s, a, s0, max_moves, w.moves, w.counts);
    const hipError_t e = by_shape(hd, f16, [&](auto HD, auto KH) {
      const uint32_t rows = 256 / (HD() * (KH() ? 2 : 4) / 16);
      hipLaunchKernelGGL((kv_move_kernel<HD(), KH()>), dim3(max(1u, min(64u, (max_moves + rows - 1) / rows)), ns), dim3(256), 0, s, a, s0,
                         max_moves, w.moves, w.counts);
      return hipGetLastError();
    });
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_kv_take_errors(uint32_t* err, uint32_t* taken, hipStream_t s) {
  hipLaunchKernelGGL(kv_take_errors_kernel, dim3(1), dim3(1), 0, s, err, taken);
  return hipGetLastError();
}

}  // namespace s2
