// Attention of each sequence's new rows over its paged cache.
//
// Mathematics: o = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m) with s = scale * q.k,
// one pass over the keys with the running maximum m and sum (base 2: the scale
// carries log2 e).  The keys of a sequence are cut into chunks that run apart; their
// (m, sum, unnormalised o) in float32 are joined by a second launch, in chunk order.
//
// paged_rows_kernel takes the head sizes that the matrix-core kernels do not (they take
// 64 and 128): one wavefront per query row, head and chunk; 64 keys at a time, one per
// lane for the scores, then one output dimension per lane for the values, whose tokens lie
// together.  A lane's rows are its own, so the address unit is the limit: five sequences
// of up to 903 float32 tokens took 34 us this way, 14 on the float32 matrix cores.
#include "paged.h"

#define ROWS_WAVES 4
#define LOG2E 1.44269504088896341f

// Four e4m3 codes as floats.
__device__ __forceinline__ void unpack_e4m3(uint32_t w, float* v) {
  v[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
  v[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
  v[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
  v[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, float* v) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else if constexpr (sizeof(T) == 2) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
    v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
  } else {
    unpack_e4m3(*reinterpret_cast<const uint32_t*>(p), v);
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float x, float y, float z, float w) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(x, y, z, w);
  else *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x, y), pack_bf16x2(z, w));
}

// q . (the key at p) over dh dimensions, q in LDS.
template <typename T>
__device__ __forceinline__ float dot_key(const float* q, const T* p, int dh) {
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int d = 0; d < dh; d += 4) {
    float v[4];
    load4(p + d, v);
    const float4 x = *reinterpret_cast<const float4*>(q + d);
    acc[0] = fmaf(x.x, v[0], acc[0]);
    acc[1] = fmaf(x.y, v[1], acc[1]);
    acc[2] = fmaf(x.z, v[2], acc[2]);
    acc[3] = fmaf(x.w, v[3], acc[3]);
  }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

// acc + sum over the first n (<= 16) of 16 keys of p * v.
template <typename T>
__device__ __forceinline__ float add_values(float acc, const float* p, const T* v, int n,
                                            float scale) {
  float a = 0.f;
  if (n == 16) {
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      float x[4];
      load4(v + k, x);
      const float4 w = *reinterpret_cast<const float4*>(p + k);
      a = fmaf(w.x, x[0], a);
      a = fmaf(w.y, x[1], a);
      a = fmaf(w.z, x[2], a);
      a = fmaf(w.w, x[3], a);
    }
  } else {  // keys that the row does not see are not touched, whatever they hold
    for (int k = 0; k < n; ++k) {
      float x;
      if constexpr (sizeof(T) == 1) x = __builtin_amdgcn_cvt_f32_fp8((int)v[k], 0);
      else x = Elem<T>::load(v, k);
      a = fmaf(p[k], x, a);
    }
  }
  return fmaf(a, scale, acc);
}

template <typename T, bool EIGHT>
__global__ void __launch_bounds__(64 * ROWS_WAVES)
paged_rows_kernel(PagedCache c, PagedBatch bt, AttendArgs a) {
  __shared__ __attribute__((aligned(16))) float qs[ROWS_WAVES][256];
  __shared__ __attribute__((aligned(16))) float ps[ROWS_WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int dh = c.head_dim, page = c.page;
  const int64_t T_heads = (int64_t)bt.rows * a.heads;
  if (blockIdx.x >= gridDim.x - a.zero_blocks) {
    zero_rest(bt, (T*)a.out, (int64_t)a.heads * dh, gridDim.x - 1 - blockIdx.x, a.zero_blocks);
    return;
  }
  // unit: (chunk, sequence row, query head), heads of a row side by side
  const int64_t unit = (int64_t)blockIdx.x * ROWS_WAVES + wave;
  const int64_t per_chunk = (int64_t)bt.sequences * bt.max_rows * a.heads;
  const int chunk = (int)(unit / per_chunk);
  const int64_t rest = unit % per_chunk;
  const int head = (int)(rest % a.heads);
  const int i = (int)(rest / a.heads % bt.max_rows);
  const int b = (int)(rest / a.heads / bt.max_rows);
  bool live = chunk < a.chunks;
  int held = 0, limit = 0, sealed = 0, last = 0, slot = -1;
  int64_t row = 0;
  if (live) {
    held = bt.held(b, page);
    const int n = held < 0 ? 0 : bt.row_count(b, held, page);
    row = (int64_t)bt.first_row(b) + i;
    live = i < given_rows(bt, b);
    if (i < n) {
      const int end = held + n;
      sealed = sealed_keys(c, bt, held, end, EIGHT);
      last = key_end(c, bt, sealed, end, EIGHT);
      limit = min(held + i + 1, last);
      if (EIGHT) slot = bt.slot(b, c.slots);
    }
  }
  const int k0 = chunk * a.chunk_keys;
  const int k1 = min(limit, k0 + a.chunk_keys);
  float* q = qs[wave];
  if (live && k1 > k0)
    for (int d = lane; d < dh; d += 64)
      q[d] = Elem<T>::load((const T*)a.q + row * a.ldq + (int64_t)head * dh, d) * a.scale2;
  __builtin_amdgcn_wave_barrier();
  const int kvh = head / a.group;
  const int64_t block = (int64_t)page * dh;
  float m = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  // the place of the 16 keys from `key` on: codes (and their exponents' place), or rows
  auto locate = [&](int key, int64_t* at, int64_t* id) {
    const int p = key >> c.shift;
    if (EIGHT && key >= sealed) {
      *id = -1;
      *at = slot < 0 ? -1 : ((int64_t)open_page(c, slot, p) * c.kv_heads + kvh) * block;
    } else {
      *id = bt.page_of(b, p, c.pages);
      *at = *id < 0 ? -1 : (*id * c.kv_heads + kvh) * block;
    }
  };
  for (int t = k0; live && t < k1; t += 64) {
    const int key = t + lane;
    float s = -INFINITY;
    if (key < k1) {
      int64_t at, id;
      locate(key, &at, &id);
      if (at >= 0) {
        const int64_t k_at = at + (int64_t)(key & (page - 1)) * dh;
        if (!EIGHT) s = dot_key(q, (const T*)c.keys + k_at, dh);
        else if (id < 0) s = dot_key(q, (const T*)c.open_keys + k_at, dh);
        else s = dot_key(q, (const e4m3_t*)c.keys + k_at, dh) *
                 exp2_int(c.exponents[id * 2 * c.kv_heads + kvh]);
      }
    }
    const float m_new = fmaxf(m, wave_max(s));
    // a NaN score makes the row's sum, and with it the row, NaN
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float p = exp2f(s - base);
    const float alpha = exp2f(m - base);
    m = m_new;
    sum = fmaf(sum, alpha, wave_sum(p));
    ps[wave][lane] = p;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] *= alpha;
    for (int g = 0; g < 64 && t + g < k1; g += 16) {
      int64_t at, id;
      locate(t + g, &at, &id);
      if (at < 0) continue;
      const int n = min(k1 - t - g, 16);
      const float scale = EIGHT && id >= 0 ? exp2_int(c.exponents[(id * 2 + 1) * c.kv_heads + kvh]) : 1.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = lane + 64 * j;
        if (d >= dh) break;
        const int64_t v_at = at + (int64_t)d * page + ((t + g) & (page - 1));
        if (!EIGHT) o[j] = add_values(o[j], ps[wave] + g, (const T*)c.values + v_at, n, 1.f);
        else if (id < 0) o[j] = add_values(o[j], ps[wave] + g, (const T*)c.open_values + v_at, n, 1.f);
        else o[j] = add_values(o[j], ps[wave] + g, (const e4m3_t*)c.values + v_at, n, scale);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (!live) return;
  const int64_t at = row * a.heads + head;
  if (a.chunks == 1) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees no key is zero
    for (int j = 0, d = lane; d < dh; ++j, d += 64)
      Elem<T>::store((T*)a.out + at * dh, d, o[j] * inv);
    return;
  }
  if (k1 <= k0 && chunk > 0) return;  // the join knows which chunks a row has
  if (lane == 0) a.stat[chunk * T_heads + at] = make_float2(m, sum);
  for (int j = 0, d = lane; d < dh; ++j, d += 64) a.part[(chunk * T_heads + at) * dh + d] = o[j];
}

// Joins the chunks of every row and head (5 to 8 us: waits, not bytes).  Four dimensions a
// thread, a.join_ways threads' worth of chunks at once, as many rows and heads a workgroup
// as that leaves room for; a way takes every join_ways-th chunk, and the ways are added in
// order.  Four chunks' loads at once: 7.9 -> 6.7 us for 432 rows of 32 heads and four
// chunks.  LDS: a way's (o, m, sum), 24 bytes a thread.
template <typename T, bool EIGHT>
__global__ void __launch_bounds__(1024)
paged_join_kernel(PagedCache c, PagedBatch bt, AttendArgs a) {
  extern __shared__ float4 o_of[];
  float *m_of = reinterpret_cast<float*>(o_of + blockDim.x), *sum_of = m_of + blockDim.x;
  const int dh = c.head_dim, page = c.page, quads = dh / 4, ways = a.join_ways;
  const int64_t T_heads = (int64_t)bt.rows * a.heads;
  const int per_unit = quads * ways, inside = threadIdx.x % per_unit;
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x / per_unit) + threadIdx.x / per_unit;
  const int way = inside / quads, d = inside % quads * 4;
  const int head = (int)(unit % a.heads);
  const int i = (int)(unit / a.heads % bt.max_rows);
  const int b = (int)(unit / a.heads / bt.max_rows);
  const bool live = threadIdx.x < blockDim.x / per_unit * per_unit && b < bt.sequences && i < given_rows(bt, b);
  float m = -INFINITY, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  int64_t at = 0;
  if (live) {
    const int held = bt.held(b, page);
    const int n = held < 0 ? 0 : bt.row_count(b, held, page);
    int limit = 0;
    if (i < n) {
      const int end = held + n, sealed = sealed_keys(c, bt, held, end, EIGHT);
      limit = min(held + i + 1, key_end(c, bt, sealed, end, EIGHT));
    }
    const int count = max((limit + a.chunk_keys - 1) / a.chunk_keys, 1);
    at = ((int64_t)bt.first_row(b) + i) * a.heads + head;
    for (int first = way; first < count; first += 4 * ways) {
      float2 st[4];
      float4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // the last one again where there is none: loads behind branches would wait in turn
        const int64_t k = min(first + j * ways, count - 1);
        st[j] = a.stat[k * T_heads + at];
        x[j] = *reinterpret_cast<const float4*>(a.part + (k * T_heads + at) * dh + d);
      }
#pragma unroll
      for (int j = 1; j < 4; ++j)
        if (first + j * ways >= count) {
          st[j] = make_float2(-INFINITY, 0.f);
          x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      const float M = fmaxf(fmaxf(fmaxf(m, st[0].x), fmaxf(st[1].x, st[2].x)), st[3].x);
      const float base = M == -INFINITY ? 0.f : M, rescale = exp2f(m - base);
      m = M;
      sum *= rescale;
      o = make_float4(o.x * rescale, o.y * rescale, o.z * rescale, o.w * rescale);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = exp2f(st[j].x - base);
        sum = fmaf(st[j].y, f, sum);
        o.x = fmaf(x[j].x, f, o.x);
        o.y = fmaf(x[j].y, f, o.y);
        o.z = fmaf(x[j].z, f, o.z);
        o.w = fmaf(x[j].w, f, o.w);
      }
    }
  }
  if (ways > 1) {
    o_of[threadIdx.x] = o;
    m_of[threadIdx.x] = m;
    sum_of[threadIdx.x] = sum;
    __syncthreads();
    if (way != 0) return;
    float M = m;
#pragma unroll 4
    for (int w = 1; w < ways; ++w) M = fmaxf(M, m_of[threadIdx.x + w * quads]);
    const float base = M == -INFINITY ? 0.f : M;
    sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int w = 0; w < ways; ++w) {
      const int t = threadIdx.x + w * quads;
      const float f = exp2f(m_of[t] - base);
      const float4 x = o_of[t];
      sum = fmaf(sum_of[t], f, sum);
      o.x = fmaf(x.x, f, o.x);
      o.y = fmaf(x.y, f, o.y);
      o.z = fmaf(x.z, f, o.z);
      o.w = fmaf(x.w, f, o.w);
    }
  }
  if (!live) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  store4((T*)a.out + at * dh + d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// ----------------------------------------------------------------------------
// Host
// ----------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Keys per chunk, in whole 64-key tiles: `want` workgroups or wavefronts in all where
// `units` take a chunk each, but no chunk below `least` keys.
static void cut_keys(AttendPlan& p, int64_t max_keys, int64_t units, int64_t want, int64_t least) {
  const int64_t most = max(ceil_div(max_keys, least), (int64_t)1);
  const int64_t chunks = min(units > 0 ? ceil_div(want, units) : 1, most);
  p.chunk_keys = max(ceil_div(ceil_div(max_keys, chunks), 64) * 64, (int64_t)64);
  p.chunks = max(ceil_div(max_keys, p.chunk_keys), (int64_t)1);
}

static AttendPlan attend_plan(const alodlm_paged_cache* c, const alodlm_paged_batch* b, int64_t heads) {
  AttendPlan p = {};
  const int64_t columns = max(b->max_rows * (heads / c->kv_heads), (int64_t)1);
  if (c->head_dim != 64 && c->head_dim != 128) {
    p.kernel = PAGED_ROWS;
    cut_keys(p, b->max_keys, b->sequences * b->max_rows * heads, 8192, 128);
    return p;
  }
  const bool f32 = c->dtype == ALODLM_F32;
  // Few columns: the keys over the waves, whose outputs are joined; else the columns, which
  // reads a tile once for 64 of them.  16 sequences of up to 3100 tokens, 32 columns: codes
  // 38 us with the keys over the waves and 41 with the columns, pages in bf16 55 and 45;
  // 33 to 64 columns: codes 45 and 44, bf16 66 and 48.
  const bool keys = columns <= (c->eight_bit && !f32 ? 32 : 16);
  p.kernel = f32 ? (keys ? PAGED_F32_KEYS : PAGED_F32_COLUMNS) : keys ? PAGED_SPLIT : PAGED_TILES;
  const int waves = keys ? 1 : 4;
  p.column_tiles = f32 || keys || columns <= 16 * waves ? 1 : 2;
  p.query_tiles = (int)ceil_div(columns, 16 * p.column_tiles * waves);
  // One sequence fills the chip evenly with two workgroups a compute unit twice over;
  // several of different lengths with smaller chunks.  Below 512 keys (256 in float32) a
  // chunk's own start and join weigh more than its keys: eight windows of 17 to 28 rows and
  // 32 heads behind 6000 tokens take 38 us with 512 and 54 with 1024, 24 behind 2200 tokens
  // 53 and 46, and 10 % less with 512 over lengths to 6000 and 1 to 24 windows.
  cut_keys(p, b->max_keys, b->sequences * c->kv_heads * p.query_tiles,
           keys && b->sequences > 1 ? 2048 : 1024, f32 ? 256 : 512);
  return p;
}

static int64_t attend_floats(const alodlm_paged_cache* c, const alodlm_paged_batch* b, int64_t heads) {
  const AttendPlan p = attend_plan(c, b, heads);
  return p.chunks == 1 ? 0 : p.chunks * b->rows * heads * (c->head_dim + 2);
}

extern "C" int64_t alodlm_paged_attention_workspace(const alodlm_paged_cache* cache,
                                                    const alodlm_paged_batch* batch, int64_t heads) {
  if (paged_check(cache, batch) || heads < 1 || heads % cache->kv_heads) return 0;
  return attend_floats(cache, batch, heads);
}

template <typename T, bool EIGHT>
static int attend_launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, AttendArgs a,
                         const AttendPlan& plan, hipStream_t st) {
  const PagedCache dc = paged_cache(c);
  const PagedBatch db = paged_batch(b);
  const int64_t units = b->sequences * b->max_rows * a.heads;
  const int64_t main = plan.kernel != PAGED_ROWS ? b->sequences * c->kv_heads * plan.query_tiles * a.chunks
                                        : ceil_div(units * a.chunks, ROWS_WAVES);
  const int64_t blocks = (units ? main : 0) + a.zero_blocks;
  ALODLM_CHECK_ARG(blocks < (1ll << 31) && units < (1ll << 31), "paged_attention: too many rows in one call");
  if (blocks == 0) return ALODLM_OK;
  if (plan.kernel == PAGED_SPLIT) paged_split_launch(c, b, a, plan, (unsigned)blocks, st);
  else if (plan.kernel == PAGED_TILES) paged_tiles_launch(c, b, a, plan, (unsigned)blocks, st);
  else if (plan.kernel != PAGED_ROWS) paged_f32_launch(c, b, a, plan, (unsigned)blocks, st);
  else paged_rows_kernel<T, EIGHT><<<(unsigned)blocks, 64 * ROWS_WAVES, 0, st>>>(dc, db, a);
  if (a.chunks > 1 && units) {
    // More ways while workgroups are few: 127 chunks of one row's 16 heads take 9.6 us with
    // eight ways and 9.0 with 32 (7.1 with four chunks' loads at once), but six of 432 rows
    // and 32 heads 12.8 with two ways and 7.9 with one.
    const int64_t quads = c->head_dim / 4;
    int64_t ways = 1;
    while (ways < 32 && ways * 4 < a.chunks && quads * ways * 2 <= 1024 && units * quads * ways < 1024 * 256) ways *= 2;
    const int64_t threads = quads * ways > 256 ? 1024 : 256;
    a.join_ways = (int)ways;
    paged_join_kernel<T, EIGHT><<<(unsigned)ceil_div(units, threads / (quads * ways)), (unsigned)threads,
                                  ways > 1 ? (size_t)threads * 24 : 0, st>>>(dc, db, a);
  }
  ALODLM_CHECK_LAUNCH("paged_attention");
  return ALODLM_OK;
}

extern "C" int alodlm_paged_attention(const alodlm_paged_cache* cache, const alodlm_paged_batch* batch,
                                      const void* q, int64_t ldq, void* out, int64_t heads,
                                      float scale, int zero_rest, float* workspace, void* stream) {
  const int rc = paged_check(cache, batch);
  if (rc) return rc;
  const int64_t es = cache->dtype == ALODLM_BF16 ? 2 : 4;
  ALODLM_CHECK_ARG(heads >= 1 && heads <= 65536 && heads % cache->kv_heads == 0,
                   "paged_attention: heads must be a multiple of the cache's kv_heads");
  ALODLM_CHECK_ARG(ldq >= heads * cache->head_dim, "paged_attention: row stride below the row width");
  ALODLM_CHECK_ARG(scale > 0.f && scale * LOG2E < INFINITY,
                   "paged_attention: scale must be positive, and finite times log2 e");
  ALODLM_CHECK_ARG((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0 &&
                       ldq * es % 16 == 0,
                   "paged_attention: rows must be 16-byte aligned");
  if (batch->rows == 0) return ALODLM_OK;
  ALODLM_CHECK_ARG(q && out, "paged_attention: no rows");
  const AttendPlan plan = attend_plan(cache, batch, heads);
  ALODLM_CHECK_ARG(plan.chunks == 1 || workspace, "paged_attention: no workspace");
  AttendArgs a = {q, out, ldq, workspace, nullptr, (int)heads, (int)(heads / cache->kv_heads),
                  (int)plan.chunk_keys, (int)plan.chunks, plan.query_tiles, 1, scale * LOG2E, 0};
  if (zero_rest) a.zero_blocks = (int)min(ceil_div(batch->rows * heads * cache->head_dim, 8192), (int64_t)64);
  a.stat = reinterpret_cast<float2*>(workspace + plan.chunks * batch->rows * heads * cache->head_dim);
  ALODLM_DISPATCH(cache->dtype, T, {
    if (cache->eight_bit) return attend_launch<T, true>(cache, batch, a, plan, as_stream(stream));
    return attend_launch<T, false>(cache, batch, a, plan, as_stream(stream));
  });
}
