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
  int pages, page, shift, kv_heads, head_dim, slots, open_pages;  // page = 1 << shift
};

struct PagedBatch {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* offsets;
  const int32_t* slot_of;
  int sequences, width, rows, max_rows, max_keys, final_rows;

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
  __device__ __forceinline__ int page_of(int b, int p, int pages) const {
    if (p < 0 || p >= width) return -1;
    const int id = table[(int64_t)b * width + p];
    return id >= 0 && id < pages ? id : -1;
  }
  // Slot of the open pages, -1 where there is none.
  __device__ __forceinline__ int slot(int b, int slots) const {
    const int s = slot_of ? slot_of[b] : b;
    return s >= 0 && s < slots ? s : -1;
  }
};

// Open page `p` of a slot: its index among all open pages.
__device__ __forceinline__ int open_page(const PagedCache& c, int slot, int p) {
  return slot * c.open_pages + p % c.open_pages;
}

// 2^e as a float, e in [-126, 127].
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// ----------------------------------------------------------------------------
// Attention (csrc/paged_attention.hip and its matrix-core kernels)
// ----------------------------------------------------------------------------
struct AttendArgs {
  const void* q;
  void* out;
  int64_t ldq;
  float* part;   // unnormalised outputs [chunks][rows * heads][head_dim]
  float2* stat;  // (maximum in base 2, sum) [chunks][rows * heads]
  int heads, group, chunk_keys, chunks, query_tiles, join_ways;
  float scale2;  // softmax scale * log2 e
  int zero_blocks;  // workgroups behind the launch's others that clear the rows without a result
};

// Zeros in the rows that no sequence has a result in, by `blocks` workgroups of 256
// threads: before the first sequence, behind the last, and past max_rows.
template <typename T>
__device__ __forceinline__ void zero_rest(const PagedBatch& bt, T* out, int64_t width, int block, int blocks) {
  auto clear = [&](int64_t from, int64_t to, int thread, int threads) {
    for (int64_t i = from * width + thread; i < to * width; i += threads) Elem<T>::store(out, i, 0.f);
  };
  const int thread = block * 256 + threadIdx.x, lane = threadIdx.x & 63;
  clear(0, bt.first_row(0), thread, blocks * 256);
  clear(bt.first_row(bt.sequences), bt.rows, thread, blocks * 256);
  if (bt.max_rows == bt.rows) return;
  // a sequence a lane; those with rows past max_rows one after the other by the wave
  for (int b0 = thread - lane; b0 < bt.sequences; b0 += blocks * 256) {
    const int b = b0 + lane;
    int from = 0, to = 0;
    if (b < bt.sequences) {
      from = bt.first_row(b) + bt.max_rows;
      to = min(bt.offsets[b + 1], bt.rows);
    }
    for (uint64_t left = __ballot(from < to); left; left &= left - 1) {
      const int which = __builtin_ctzll(left);
      clear(__shfl(from, which, 64), __shfl(to, which, 64), lane, 64);
    }
  }
}

// Where the 8-bit pages of a sequence end (keys before it are sealed).
__device__ __forceinline__ int sealed_keys(const PagedCache& c, const PagedBatch& bt, int held, int end,
                                           bool eight) {
  if (!eight) return end;
  return (bt.final_rows ? end : held) >> c.shift << c.shift;
}

// The end of the keys that are attended to: the tokens, as far as max_keys goes and open
// pages hold them (windows longer than those are refused by the host; this bounds what is
// read).
__device__ __forceinline__ int key_end(const PagedCache& c, const PagedBatch& bt, int sealed, int end,
                                       bool eight) {
  end = min(end, bt.max_keys);
  return eight ? (int)min((int64_t)end, (int64_t)sealed + (int64_t)c.open_pages * c.page) : end;
}

// Rows of sequence b that results are written for: those of the batch, up to max_rows,
// whether or not the sequence takes part.
__device__ __forceinline__ int given_rows(const PagedBatch& bt, int b) {
  const int r0 = bt.first_row(b);
  return min(min(max(bt.offsets[b + 1], r0), bt.rows) - r0, bt.max_rows);
}

// How a call is cut up, and which kernel takes it.
enum PagedKernel {
  PAGED_ROWS,         // csrc/paged_attention.hip: a wavefront per row and head
  PAGED_SPLIT,        // csrc/paged_split.hip: bf16 matrix cores, the keys over the waves
  PAGED_TILES,        // csrc/paged_tiles.hip: bf16 matrix cores, the query columns over the waves
  PAGED_F32_KEYS,     // csrc/paged_f32.hip: float32 matrix cores, the keys over the waves
  PAGED_F32_COLUMNS,  // csrc/paged_f32.hip: the query columns over the waves
};
struct AttendPlan {
  PagedKernel kernel;
  int column_tiles, query_tiles;  // 16-column tiles a wave, workgroups along a sequence's columns
  int64_t chunk_keys, chunks;
};
typedef void paged_launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, const AttendArgs& a,
                          const AttendPlan& p, unsigned blocks, hipStream_t st);
paged_launch paged_split_launch, paged_tiles_launch, paged_f32_launch;

// Host: checks of the two structs shared by the entry points (abi errors), and
// their device forms.
int paged_check(const alodlm_paged_cache* c, const alodlm_paged_batch* b);
PagedCache paged_cache(const alodlm_paged_cache* c);
PagedBatch paged_batch(const alodlm_paged_batch* b);
