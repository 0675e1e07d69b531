// The paged key/value cache as its kernels see it (csrc/paged_append.hip,
// csrc/paged_attention.hip).  Every index read from the device (page, slot,
// length, row offset) is checked before it is followed.
#pragma once

#include "common.h"

typedef uint8_t e4m3_t;

struct PagedCache {
  void* keys;
  void* values;
  int8_t* exponents;
  void* open_keys;
  void* open_values;
  int64_t pages;
  int page, kv_heads, head_dim, slots, open_pages;
};

struct PagedBatch {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* offsets;
  const int32_t* slot_of;
  int sequences, width, rows, max_rows, final_rows;

  // Row range of sequence b, inside the batch's rows.
  __device__ __forceinline__ int first_row(int b) const {
    return min(max(offsets[b], 0), rows);
  }
  // Tokens held before the step; -1 (the sequence takes no part) for a length that
  // is negative or past the table.
  __device__ __forceinline__ int held(int b, int page) const {
    const int n = lengths[b];
    return n >= 0 && (int64_t)n <= (int64_t)width * page ? n : -1;
  }
  // Rows of the step, as many as the table has places for behind `held`.
  __device__ __forceinline__ int row_count(int b, int held, int page) const {
    const int r0 = first_row(b);
    const int n = min(min(max(offsets[b + 1], r0), rows) - r0, max_rows);
    return (int)min((int64_t)n, (int64_t)width * page - held);
  }
  // Page of the pool, -1 where the table names none.
  __device__ __forceinline__ int64_t page_of(int b, int p, int64_t pages) const {
    if (p < 0 || p >= width) return -1;
    const int64_t id = table[(int64_t)b * width + p];
    return id >= 0 && id < pages ? id : -1;
  }
  // Slot of the open pages, -1 where there is none.
  __device__ __forceinline__ int slot(int b, int slots) const {
    const int s = slot_of ? slot_of[b] : b;
    return s >= 0 && s < slots ? s : -1;
  }
};

// Open page `p` of a slot: its index among all open pages.
__device__ __forceinline__ int64_t open_page(const PagedCache& c, int slot, int p) {
  return (int64_t)slot * c.open_pages + p % c.open_pages;
}

// 2^e as a float, e in [-126, 127].
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Host: checks of the two structs shared by the entry points (abi errors), and
// their device forms.
int paged_check(const alodlm_paged_cache* c, const alodlm_paged_batch* b);
PagedCache paged_cache(const alodlm_paged_cache* c);
PagedBatch paged_batch(const alodlm_paged_batch* b);
