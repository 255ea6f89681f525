// kvops.h -- launch interface of the KV-cache operators (kvops.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace s2 {

// Head shape of a handle and its device words.
struct KvShape {
  uint32_t H, G, rep;  // query heads, kv heads, H / G
  float scale2;        // of the scores, times log2(e)
  float eps;
  const double* freq;  // [hd / 2] rope_base^(-2 i / hd)
  uint32_t* err;       // S2HIP_KV_ERR_* bits are or-ed in
};

// The caches of a call (strides in elements, all set).
struct KvCaches {
  void* k;
  void* v;
  const void* pk;
  const void* pv;
  const int32_t* lens;
  const int32_t* new_lens;  // nullable
  size_t req_stride, head_stride, slot_stride, p_head_stride, p_slot_stride;
  uint32_t R, cap, P, n;    // requests, capacity, prefix length, tokens per request
};

struct KvAppendArgs {
  KvShape s;
  KvCaches c;
  const float* qkv;
  const int32_t* positions;
  const float* q_norm;  // nullable, with k_norm
  const float* k_norm;
  float* q_out;
  float* scores;            // nullable
  int32_t* slot_positions;  // nullable
};

// Softmax states of 16 rows per (kv head, row tile, split): o [16][hd], (m, l) [16][2].
struct KvSplit {
  float* o;
  float* ml;
  uint32_t tiles, splits;
  uint32_t least;  // key tiles per split, at least (kv_tile_kernel)
  float up;        // o times this is the sum of weights with values (f32 caches)
};

// A step's scores, kept for the weights (nullable).
struct KvScores {
  float* own;     // [R][G][cap][n rep]
  float* prefix;  // [G][P][R n rep]
};

// Caches from which an eviction runs in one launch in place too, and a cache's
// longest list of moves (half of 32768 slots).
constexpr uint32_t KV_LISTS = 512, KV_LIST = 16384;

struct KvWorkspace {
  float* stat;  // [tokens][H][2]: a row's m and l (attention with weights)
  float* part;     // [cap_parts][16][hd]
  float* part_ml;  // [cap_parts][16][2]
  size_t cap_parts;
  float* weights;  // [cap_weights]: a step's scores, or the row splits' sums of weights
  size_t cap_weights;
  uint32_t* moves;   // [KV_LISTS][KV_LIST]: an eviction's moves (to | from << 16)
  uint32_t* counts;  // [KV_LISTS][2]: moves, slots left
};

struct KvAttendArgs {
  KvShape s;
  KvCaches c;
  const float* q;
  float* out;
  // with weights (nullable):
  const float* w_in;   // nullable
  float* w_out;
  const float* pw_in;  // nullable
  float* pw_out;       // nullable
  uint32_t pw_stride;  // prefix_capacity
};

struct KvEvictArgs {
  KvShape s;
  KvCaches c;
  size_t layer_stride;
  uint32_t layers, keep, recent, sinks;
  uint32_t elem;  // bytes of a cache element
  const float* scores;
  const int32_t* positions;
  float* scores_out;
  int32_t* positions_out;
  int32_t* lens_out;
};

hipError_t launch_kv_append(uint32_t hd, bool f16, const KvAppendArgs& a, hipStream_t s);
hipError_t launch_kv_attend(uint32_t hd, bool f16, const KvAttendArgs& a, const KvWorkspace& w, hipStream_t s);
hipError_t launch_kv_evict(const KvEvictArgs& a, const KvWorkspace& w, uint32_t hd, hipStream_t s);
hipError_t launch_kv_take_errors(uint32_t* err, uint32_t* taken, hipStream_t s);

}  // namespace s2
