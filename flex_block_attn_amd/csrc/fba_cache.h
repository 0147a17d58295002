// The paged cache of keys and values: what its kernels share.
//
// A pool of pages [pages, kv heads, page size, 128]; a page holds page_size slots of every kv head.  Sequence b's slot s is slot s % page_size of page
// table[b][s / page_size]; the first lengths[b] slots are filled.  positions and weights [pages, kv heads, page size] go with the slots.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fba_window.h"

namespace fba {

struct CacheView {
  char* k;
  char* v;
  int32_t* positions;
  float* weights;
  const int32_t* table;    // [batch, max_pages]
  const int32_t* lengths;  // [batch]
  int64_t pages;
  int kv_heads, page_log2, batch, max_pages;
  __host__ __device__ int64_t slots() const { return (int64_t)max_pages << page_log2; }  // that a sequence has room for
  // A length that the table has room for.
  __host__ __device__ bool holds(int64_t n) const { return n >= 0 && n <= slots(); }
  // Page of a slot below slots(), or -1 where the table names none of the pool's.
  __host__ __device__ int page_of(int b, int slot) const {
    const int page = table[(int64_t)b * max_pages + (slot >> page_log2)];
    return page >= 0 && page < pages ? page : -1;
  }
  // Number of a slot's row in the pool.
  __host__ __device__ int64_t row_of(int page, int head, int slot) const {
    return (((int64_t)page * kv_heads + head) << page_log2) + (slot & ((1 << page_log2) - 1));
  }
};

struct AppendParams {
  CacheView cache;
  Strided k, v;              // [batch, kv heads, tokens, 128]
  const int32_t* counts;     // null, or [batch]: tokens of each sequence
  const int32_t* first;      // null (the length), or [batch]: position of the first one
  const float* weights;      // null (zeros), or [batch, kv heads, tokens]
  int32_t* lengths_out;
  int tokens;
  int row_wgs;
};

struct AttendParams {
  CacheView cache;
  Strided q, o;              // [batch, heads, 1, 128]
  int heads, window, sinks;
  float scale_log2e;
  int target;                // shares that the tiles of all sequences are cut into, at most
  int head_tiles;            // work-groups that share a share of a kv head
  int slots;                 // places for parts of sequences
  // workspace: sums of the parts [slots, heads, 128], their references and denominators [slots, heads, 2], first place and number of parts of a sequence
  // [batch, 2], scores [batch, heads, cache.slots()] (null: weights are not added up)
  float* part;
  float* part_ml;
  int32_t* note;
  float* scores;
};

struct EvictParams {
  CacheView cache;
  int budget, recent, sinks;
  int32_t* lengths_out;
  // workspace: moves of every (sequence, kv head) [batch * kv heads, 1 + 2 * most]: their number, destinations, sources
  int32_t* moves;
  int most;
};

hipError_t launch_cache_append(AppendParams p, hipStream_t stream);
void plan_cache_attend(AttendParams& p, int compute_units);
int64_t cache_attend_bytes(const AttendParams& p, bool accumulate);
hipError_t launch_cache_attend(AttendParams p, bool half, hipStream_t stream);
int64_t cache_evict_bytes(EvictParams& p);
hipError_t launch_cache_evict(EvictParams p, hipStream_t stream);

}  // namespace fba
