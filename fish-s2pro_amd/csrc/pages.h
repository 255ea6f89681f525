// pages.h -- launch interface of the paged 4-bit KV cache (pages.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kvops.h"

namespace s2 {

// A pool of pages and the rows that hold them.
struct PgPool {
  uint8_t* pool;
  const int32_t* table;  // [R][width]
  uint32_t shift;        // log2(page_tokens)
  uint32_t pages, width;
  uint32_t chunk;        // bytes of a kv head's part of a page
};

struct PgRope {
  const double* turns;  // [dims / 2]: angles per position, in turns
  double gain;
  uint32_t dims, half;
};

struct PgAppendArgs {
  KvShape s;
  KvCaches c;  // lens, new_lens, R, n and cap (tokens)
  PgPool p;
  PgRope rope;
  const float* qkv;
  const int32_t* positions;
  const float* q_norm;  // nullable, with k_norm
  const float* k_norm;
  float* q_out;
  float* k_held;  // nullable
  float* v_held;  // nullable
};

// n / d for n below 2^31: m is above 2^(31 + s) / d by less than 2^s / d, where 2^s is at least d, so 2 n m is above
// 2^(32 + s) n / d by less than 2^(32 + s) / d.  (A division of the compiler's is 35 instructions, and a step's kernel begins
// with ten of them one behind the other.)
struct Div {
  uint32_t m, s;
  static Div by(uint32_t d) {
    uint32_t s = 0;
    while ((uint64_t(1) << s) < d) ++s;
    return {uint32_t((uint64_t(1) << (31 + s)) / d + 1), s};
  }
  __host__ __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return uint32_t((uint64_t(n + n) * m) >> 32) >> s; }
};

struct PgAttendArgs {
  KvAttendArgs a;  // shape, lens, new_lens, R, n, cap, q, out
  PgPool p;
  Div by_rows, by_rep, by_groups;  // n rep (a request's packed rows), rep, G
};

struct PgUpdateArgs {
  PgPool p;
  const int32_t* lens;
  const int32_t* source;  // nullable
  const int32_t* keep;    // nullable
  const int32_t* add;     // nullable
  const int32_t* refs;
  int32_t* refs_out;
  int32_t* table_out;
  int32_t* lens_out;
  int32_t* used_out;  // compact
  int32_t* moved_to;  // compact, nullable
  size_t layer_stride;
  uint32_t layers, R;
  uint32_t* err;
};

// Blocks that an attention in several splits is shared out to, and the 16-row states that they leave, at most: the tile kernel's
// 8 each (128 rows), the step kernel's 1 or 2.  (Calls of more row tiles have one split, and no states.)
constexpr uint32_t PG_TILE_BLOCKS = 512, PG_STEP_BLOCKS = 768, PG_STATES = 8 * PG_TILE_BLOCKS;
static_assert(PG_STATES >= 2 * PG_STEP_BLOCKS, "the step kernel's states fit");

struct PgWorkspace {
  float* part;     // [PG_STATES][16][hd]: attention states
  float* part_ml;  // [PG_STATES][16][2]
  uint2* ranges;   // [64]: a row tile's states
  int32_t* refs;   // [pages]
  int32_t* list;   // [2][pages]: free pages; holes and movers
  int32_t* table;  // [max_requests][width]
  int32_t* moves;  // [256][2]: pages that are copied, from and to; [0]: their number (compact)
};

hipError_t prepare_pg();  // of the current device, before the others
hipError_t launch_pg_append(uint32_t hd, const PgAppendArgs& a, hipStream_t s);
hipError_t launch_pg_attend(uint32_t hd, PgAttendArgs a, const PgWorkspace& w, hipStream_t s);
hipError_t launch_pg_update(const PgUpdateArgs& a, const PgWorkspace& w, uint32_t page_bytes, hipStream_t s);
hipError_t launch_pg_compact(const PgUpdateArgs& a, const PgWorkspace& w, uint32_t page_bytes, hipStream_t s);

}  // namespace s2
