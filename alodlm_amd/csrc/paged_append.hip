// Appending a step's keys and values to a paged cache, with the rotation on the
// way, and sealing the pages that fill up in 8 bits.
//
// Mathematics: a key is x * cos + rotate_half(x) * sin in float32, rounded once to
// the model's type; a page and head in 8 bits is e4m3(x * 2^-e) with the smallest
// e that keeps the largest magnitude within 448 * 2^e.  A floating 8-bit format
// gains nothing from a finer scale (only its smallest binade moves), and with a
// power of two neither the scaling nor its undoing rounds: one rounding in all.
//
// Work: one workgroup per sequence, head and page that the step touches.  A page
// that fills up is gathered in LDS (its older tokens from the open page, the new
// ones from the inputs), which also turns the values into their token-contiguous
// order and lets the page be read once for both the largest magnitude and the
// codes.  A page that does not fill up is written row by row.  The workgroup of a
// sequence's first page also writes the rows that stay open behind the last sealed
// page: they may take the places of the open rows that it reads, so it reads first.
//
// Bound by the bytes where there are many: eight prompts of 300 to 4000 rows, 241 MB, 60
// us (4.0 TB/s); a step of 64 rows 5 us, a launch and one round trip.  Into bf16 pages, whose
// values are written 2 bytes a lane: 16 windows of 16 to 32 rows 7 us.
#include "paged.h"

#define APPEND_THREADS 256

// 8 or 4 consecutive elements as floats.
template <int VEC, typename T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  if constexpr (VEC == 8) {
    Vec8<T>::load(p, v);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
    v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
  }
}
template <int VEC, typename T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  if constexpr (VEC == 8) {
    Vec8<T>::store(p, v);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  }
}

// VEC elements of a head and the VEC half a head behind them, rotated (each
// product and the sum rounded to float32; products of bf16 values are exact).
template <int VEC, typename T>
__device__ __forceinline__ void rotated_pair(const T* x, const T* cos_row, const T* sin_row, int j,
                                             int half, float* lo, float* hi) {
#pragma clang fp contract(off)
  load_vec<VEC>(x + j, lo);
  load_vec<VEC>(x + half + j, hi);
  if (!cos_row) return;
  float c0[VEC], c1[VEC], s0[VEC], s1[VEC];
  load_vec<VEC>(cos_row + j, c0);
  load_vec<VEC>(cos_row + half + j, c1);
  load_vec<VEC>(sin_row + j, s0);
  load_vec<VEC>(sin_row + half + j, s1);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float a = lo[i], b = hi[i];
    lo[i] = a * c0[i] + (-b) * s0[i];
    hi[i] = b * c1[i] + a * s1[i];
  }
}

template <typename T>
struct AppendInputs {
  const T *k, *v, *q, *cos_tab, *sin_tab;
  T* q_out;
  int64_t ldk, ldv, ldq;
  const int32_t* counts;  // retire: rows of the batch that are kept, all in open pages
  int heads, q_blocks, touched;
};

// Rows [lo, hi) of the page at `start` (positions start + row) written in the
// model's type: new rows, position p being batch row r0 + p - held.
template <int VEC, typename T>
__device__ void write_rows(const PagedCache& c, const AppendInputs<T>& in, T* kdst, T* vdst, int h,
                           int start, int lo, int hi, int64_t row0, int held) {
  const int dh = c.head_dim, half = dh / 2, units = half / VEC, n = hi - lo;
  for (int u = threadIdx.x; u < n * units; u += APPEND_THREADS) {
    const int r = lo + u / units, j = u % units * VEC;
    const int64_t row = row0 + start + r - held;
    const T* cr = in.cos_tab ? in.cos_tab + row * dh : nullptr;
    const T* sr = in.cos_tab ? in.sin_tab + row * dh : nullptr;
    float a[VEC], b[VEC];
    rotated_pair<VEC>(in.k + row * in.ldk + (int64_t)h * dh, cr, sr, j, half, a, b);
    store_vec<VEC>(kdst + (int64_t)r * dh + j, a);
    store_vec<VEC>(kdst + (int64_t)r * dh + half + j, b);
  }
  // token-contiguous values: neighbouring threads take neighbouring tokens
  for (int u = threadIdx.x; u < n * dh; u += APPEND_THREADS) {
    const int r = lo + u % n, d = u / n;
    const int64_t row = row0 + start + r - held;
    vdst[(int64_t)d * c.page + r] = in.v[row * in.ldv + (int64_t)h * dh + d];
  }
}

// Largest finite magnitude over the workgroup -> the page's exponent.
__device__ __forceinline__ int page_exponent(float largest, float* red) {
  largest = block_max(largest, red);
  if (!(largest > 0.f)) return -100;
  int e;
  const float m = frexpf(largest, &e);
  return max(m <= 0.875f ? e - 9 : e - 8, -100);
}

__device__ __forceinline__ float magnitude(float x) {
  const float a = fabsf(x);
  return a <= 3.4028235e38f ? a : 0.f;  // inf and NaN do not count
}

// Four values over the scale as e4m3 codes; inf and NaN become NaN.
__device__ __forceinline__ uint32_t pack_e4m3(const float* x, float inv) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = fabsf(x[i]) <= 3.4028235e38f ? x[i] * inv : NAN;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  return (uint32_t)w;
}

// Seals the page at `start` of sequence b for head h: rows before `held` come from
// the open page, the others from the inputs.
template <int VEC, typename T>
__device__ void seal_page(const PagedCache& c, const AppendInputs<T>& in, int64_t id, int64_t from,
                          int h, int start, int64_t row0, int held, T* lds, float* red) {
  const int dh = c.head_dim, half = dh / 2, units = half / VEC, ps = c.page, words = dh / 4;
  const int64_t block = (id * c.kv_heads + h) * (int64_t)ps * dh;
  const int64_t oblock = (from * c.kv_heads + h) * (int64_t)ps * dh;
  float largest = 0.f;
  for (int u = threadIdx.x; u < ps * units; u += APPEND_THREADS) {
    const int r = u / units, j = u % units * VEC;
    float a[VEC], b[VEC];
    if (start + r < held) {
      const T* src = (const T*)c.open_keys + oblock + (int64_t)r * dh;
      load_vec<VEC>(src + j, a);
      load_vec<VEC>(src + half + j, b);
    } else {
      const int64_t row = row0 + start + r - held;
      const T* cr = in.cos_tab ? in.cos_tab + row * dh : nullptr;
      const T* sr = in.cos_tab ? in.sin_tab + row * dh : nullptr;
      rotated_pair<VEC>(in.k + row * in.ldk + (int64_t)h * dh, cr, sr, j, half, a, b);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      a[i] = Elem<T>::round(a[i]);
      b[i] = Elem<T>::round(b[i]);
      largest = fmaxf(largest, fmaxf(magnitude(a[i]), magnitude(b[i])));
    }
    store_vec<VEC>(lds + r * dh + j, a);
    store_vec<VEC>(lds + r * dh + half + j, b);
  }
  int e = page_exponent(largest, red);  // its barriers also publish the rows
  if (threadIdx.x == 0) c.exponents[(id * 2) * c.kv_heads + h] = (int8_t)e;
  float inv = exp2_int(-e);
  for (int u = threadIdx.x; u < ps * words; u += APPEND_THREADS) {
    float x[4];
    load_vec<4>(lds + u * 4, x);
    reinterpret_cast<uint32_t*>((e4m3_t*)c.keys + block)[u] = pack_e4m3(x, inv);
  }
  __syncthreads();
  // values: rows into LDS, columns out of it
  largest = 0.f;
  for (int u = threadIdx.x; u < ps * dh / VEC; u += APPEND_THREADS) {
    const int r = u / (dh / VEC), j = u % (dh / VEC) * VEC;
    if (start + r < held) continue;
    float a[VEC];
    load_vec<VEC>(in.v + (row0 + start + r - held) * in.ldv + (int64_t)h * dh + j, a);
#pragma unroll
    for (int i = 0; i < VEC; ++i) largest = fmaxf(largest, magnitude(a[i]));
    store_vec<VEC>(lds + r * dh + j, a);
  }
  const int old = min(max(held - start, 0), ps);
  for (int u = threadIdx.x; u < old * dh; u += APPEND_THREADS) {
    const int r = u % old, d = u / old;
    const T x = ((const T*)c.open_values)[oblock + (int64_t)d * ps + r];
    largest = fmaxf(largest, magnitude(Elem<T>::load(&x, 0)));
    lds[r * dh + d] = x;
  }
  e = page_exponent(largest, red);
  if (threadIdx.x == 0) c.exponents[(id * 2 + 1) * c.kv_heads + h] = (int8_t)e;
  inv = exp2_int(-e);
  // neighbouring threads take neighbouring columns (no bank conflict), 16 tokens each
  for (int u = threadIdx.x; u < dh * (ps / 16); u += APPEND_THREADS) {
    const int d = u % dh, g = u / dh;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) x[t] = Elem<T>::load(lds, (g * 16 + i * 4 + t) * dh + d);
      w[i] = pack_e4m3(x, inv);
    }
    *reinterpret_cast<uint4*>((e4m3_t*)c.values + block + (int64_t)d * ps + g * 16) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
  __syncthreads();  // LDS and the open rows have been read
}

template <int VEC, typename T, bool EIGHT>
__global__ void __launch_bounds__(APPEND_THREADS)
paged_append_kernel(PagedCache c, PagedBatch bt, AppendInputs<T> in) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  __shared__ float red[APPEND_THREADS / 64];
  const int dh = c.head_dim, ps = c.page;
  if ((int)blockIdx.x < in.q_blocks) {  // the queries' rotation
    const int half = dh / 2, units = half / VEC;
    const int64_t total = (int64_t)bt.rows * in.heads * units;
    for (int64_t u = (int64_t)blockIdx.x * APPEND_THREADS + threadIdx.x; u < total;
         u += (int64_t)in.q_blocks * APPEND_THREADS) {
      const int j = (int)(u % units) * VEC;
      const int64_t head = u / units, row = head / in.heads;
      float a[VEC], b[VEC];
      rotated_pair<VEC>(in.q + row * in.ldq + head % in.heads * dh, in.cos_tab + row * dh,
                        in.sin_tab + row * dh, j, half, a, b);
      store_vec<VEC>(in.q_out + head * dh + j, a);
      store_vec<VEC>(in.q_out + head * dh + half + j, b);
    }
    return;
  }
  int id = blockIdx.x - in.q_blocks;
  const int i = id % in.touched;
  id /= in.touched;
  const int h = id % c.kv_heads, b = id / c.kv_heads;
  const int64_t row0 = bt.first_row(b);
  int held = bt.held(b, ps);
  if (held < 0) return;
  int n = bt.row_count(b, held, ps);
  const int first = held >> c.shift;
  if (in.counts) {  // retire: everything kept is in open pages already
    n = min(max(in.counts[b], 0), n);
    held += n;
    n = 0;
  }
  const int end = held + n;
  const int64_t head_block = (int64_t)ps * dh;
  if constexpr (!EIGHT) {
    const int p = first + i, start = p * ps;
    const int page = bt.page_of(b, p, c.pages);
    if (page < 0 || start >= end) return;
    const int64_t at = ((int64_t)page * c.kv_heads + h) * head_block;
    write_rows<VEC, T>(c, in, (T*)c.keys + at, (T*)c.values + at, h, start, max(held - start, 0),
                       min(end - start, ps), row0, held);
    return;
  }
  const int slot = bt.slot(b, c.slots);
  if (slot < 0) return;
  // pages [first, sealed) fill up; `sealed` is the first one that stays open
  const int sealed = bt.final_rows || in.counts ? end >> c.shift : first;
  if (first + i < sealed) {
    const int p = first + i;
    const int page = bt.page_of(b, p, c.pages);
    if (page >= 0)
      seal_page<VEC, T>(c, in, page, open_page(c, slot, p), h, p * ps, row0, held, (T*)lds_raw, red);
  }
  // rows that stay open: behind the sealed pages (the first page's workgroup, see
  // above), or wherever the step's rows lie when none is sealed
  const int p = sealed > first ? (i == 0 ? sealed : -1) : first + i;
  if (p < 0 || n == 0) return;
  const int start = p * ps;
  // rows further on than the open pages reach would take each other's place
  if (start >= end || p - sealed >= c.open_pages) return;
  const int64_t at = ((int64_t)open_page(c, slot, p) * c.kv_heads + h) * head_block;
  write_rows<VEC, T>(c, in, (T*)c.open_keys + at, (T*)c.open_values + at, h, start,
                     max(held - start, 0), min(end - start, ps), row0, held);
}

// ----------------------------------------------------------------------------
// Host
// ----------------------------------------------------------------------------
int paged_check(const alodlm_paged_cache* c, const alodlm_paged_batch* b) {
  ALODLM_CHECK_ARG(c && b, "paged: null struct");
  ALODLM_CHECK_ARG(c->keys && c->values && (!c->eight_bit || (c->exponents && c->open_keys && c->open_values)),
                   "paged: the cache lacks an array");
  ALODLM_CHECK_ARG(b->offsets && (b->sequences == 0 || (b->table && b->lengths)),
                   "paged: the batch lacks an array");
  ALODLM_CHECK_ARG(c->dtype == ALODLM_F32 || c->dtype == ALODLM_BF16, "paged: unknown dtype %d",
                   (int)c->dtype);
  const int64_t ps = c->page_size, dh = c->head_dim;
  ALODLM_CHECK_ARG(ps >= 16 && ps <= 128 && (ps & (ps - 1)) == 0,
                   "paged: page size must be 16, 32, 64 or 128, got %lld", (long long)ps);
  ALODLM_CHECK_ARG(dh >= 8 && dh <= 256 && dh % 8 == 0,
                   "paged: head_dim must be a multiple of 8 up to 256, got %lld", (long long)dh);
  ALODLM_CHECK_ARG(!c->eight_bit || ps * dh <= 16384,
                   "paged: 8-bit pages hold at most 16384 values a head (page size * head_dim)");
  ALODLM_CHECK_ARG(c->kv_heads >= 1 && c->kv_heads <= 1024, "paged: kv_heads out of range");
  ALODLM_CHECK_ARG(c->pages >= 1 && c->pages < (1ll << 31), "paged: pages out of range");
  ALODLM_CHECK_ARG(!c->eight_bit || (c->slots >= 1 && c->slots < (1ll << 31) &&
                                     c->open_pages >= 1 && c->open_pages < (1ll << 20) &&
                                     c->slots * c->open_pages < (1ll << 31)),
                   "paged: an 8-bit cache needs slots and open pages (fewer than 2^31)");
  ALODLM_CHECK_ARG(b->sequences >= 0 && b->sequences < (1ll << 24) && b->rows >= 0 &&
                       b->rows < (1ll << 30) && b->max_rows >= 0 && b->max_rows <= b->rows,
                   "paged: sequences, rows or max_rows out of range");
  // keys are counted in 32 bits, by the attention up to 8192 chunks' rounding to 64 past them
  ALODLM_CHECK_ARG(b->width >= 1 && b->width < (1ll << 31) && b->width * ps < (1ll << 31) - (1ll << 20),
                   "paged: the table's width is out of range");
  ALODLM_CHECK_ARG(b->max_keys >= 0 && b->max_keys <= b->width * ps,
                   "paged: max_keys exceeds the table's pages");
  ALODLM_CHECK_ARG(!c->eight_bit || b->final_rows || b->max_rows <= c->open_pages * ps - (ps - 1),
                   "paged: %lld open pages of %lld tokens do not hold a window of %lld rows",
                   (long long)c->open_pages, (long long)ps, (long long)b->max_rows);
  return ALODLM_OK;
}

PagedCache paged_cache(const alodlm_paged_cache* c) {
  return {c->keys, c->values, c->exponents, c->open_keys, c->open_values, (int)c->pages,
          (int)c->page_size, __builtin_ctz((unsigned)c->page_size), (int)c->kv_heads, (int)c->head_dim, (int)c->slots,
          (int)c->open_pages};
}

PagedBatch paged_batch(const alodlm_paged_batch* b) {
  return {b->table, b->lengths, b->offsets, b->slots, (int)b->sequences, (int)b->width,
          (int)b->rows, (int)b->max_rows, (int)b->max_keys, (int)b->final_rows};
}

template <typename T>
static int append_launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b,
                         AppendInputs<T> in, hipStream_t st) {
  const int64_t ps = c->page_size, dh = c->head_dim;
  const bool wide = dh % 16 == 0;
  const int64_t vec = wide ? 8 : 4;
  // a step's rows touch at most this many pages of a sequence
  in.touched = (int)((ps - 1 + b->max_rows + ps - 1) / ps);
  if (b->max_rows == 0 && !in.counts) in.touched = 0;
  const int64_t tasks = b->sequences * c->kv_heads * in.touched;
  const int64_t units = in.q ? b->rows * in.heads * (dh / 2 / vec) : 0;
  in.q_blocks = (int)min((units + APPEND_THREADS - 1) / APPEND_THREADS, (int64_t)8192);
  ALODLM_CHECK_ARG(tasks + in.q_blocks < (1ll << 31), "paged_append: too many pages in one call");
  if (tasks + in.q_blocks == 0) return ALODLM_OK;
  const PagedCache dc = paged_cache(c);
  const PagedBatch db = paged_batch(b);
  const unsigned grid = (unsigned)(tasks + in.q_blocks);
  const size_t lds = c->eight_bit ? ps * dh * sizeof(T) : 0;
#define ALODLM_APPEND(V, E) paged_append_kernel<V, T, E><<<grid, APPEND_THREADS, lds, st>>>(dc, db, in)
  if (wide && c->eight_bit) ALODLM_APPEND(8, true);
  else if (wide) ALODLM_APPEND(8, false);
  else if (c->eight_bit) ALODLM_APPEND(4, true);
  else ALODLM_APPEND(4, false);
#undef ALODLM_APPEND
  ALODLM_CHECK_LAUNCH("paged_append");
  return ALODLM_OK;
}

static bool aligned16(const void* p, int64_t ld_bytes) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld_bytes % 16 == 0;
}

extern "C" int alodlm_paged_append(const alodlm_paged_cache* cache, const alodlm_paged_batch* batch,
                                   const void* k, int64_t ldk, const void* v, int64_t ldv,
                                   const void* q, int64_t ldq, void* q_out, int64_t heads,
                                   const void* cos_tab, const void* sin_tab, void* stream) {
  const int rc = paged_check(cache, batch);
  if (rc) return rc;
  const int64_t width = cache->kv_heads * cache->head_dim;
  const int64_t es = cache->dtype == ALODLM_BF16 ? 2 : 4;
  ALODLM_CHECK_ARG((cos_tab == nullptr) == (sin_tab == nullptr), "paged_append: cos without sin");
  ALODLM_CHECK_ARG(!q || (cos_tab && q_out), "paged_append: q is given to be rotated");
  ALODLM_CHECK_ARG(ldk >= width && ldv >= width && (!q || ldq >= heads * cache->head_dim),
                   "paged_append: row strides below the row width");
  ALODLM_CHECK_ARG(!q || (heads >= 1 && heads <= 65536), "paged_append: heads out of range");
  ALODLM_CHECK_ARG(aligned16(k, ldk * es) && aligned16(v, ldv * es) && aligned16(q, q ? ldq * es : 0) &&
                       aligned16(q_out, 0) && aligned16(cos_tab, 0) && aligned16(sin_tab, 0) &&
                       aligned16(cache->keys, 0) && aligned16(cache->values, 0) &&
                       aligned16(cache->open_keys, 0) && aligned16(cache->open_values, 0),
                   "paged_append: rows must be 16-byte aligned");
  if (batch->rows == 0) return ALODLM_OK;
  ALODLM_CHECK_ARG(k && v, "paged_append: no rows");
  ALODLM_DISPATCH(cache->dtype, T, {
    AppendInputs<T> in = {(const T*)k, (const T*)v, (const T*)q, (const T*)cos_tab,
                          (const T*)sin_tab, (T*)q_out, ldk, ldv, ldq, nullptr, (int)heads, 0, 0};
    return append_launch<T>(cache, batch, in, as_stream(stream));
  });
}

extern "C" int alodlm_paged_retire(const alodlm_paged_cache* cache, const alodlm_paged_batch* batch,
                                   const int32_t* counts, void* stream) {
  const int rc = paged_check(cache, batch);
  if (rc) return rc;
  ALODLM_CHECK_ARG(!batch->final_rows, "paged_retire: the batch's rows are kept already");
  ALODLM_CHECK_ARG(counts || batch->sequences == 0, "paged_retire: no counts");
  if (!cache->eight_bit || batch->sequences == 0 || batch->rows == 0) return ALODLM_OK;
  ALODLM_DISPATCH(cache->dtype, T, {
    AppendInputs<T> in = {};
    in.counts = counts;
    return append_launch<T>(cache, batch, in, as_stream(stream));
  });
}
