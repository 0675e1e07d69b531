// Log probabilities of given tokens, entropy and top alternatives of logits over the
// vocabulary, and the gradient in the logits.
//
// Mathematics: with x = logits / T and m = max x, one pass keeps s = sum exp(x - m)
// and t = sum exp(x - m) (x - m) in float32 (rescaled when m moves), from which
// log p = (x - m) - log s and the entropy is log s - t / s: everything is summed
// relative to the maximum, so nothing large cancels.
//
// Alternatives in the same pass: every thread also knows its own largest logit.  The
// top-th largest of those, tau, is a lower bound of the top-th largest logit, and only
// the threads whose largest reaches it hold candidates: their logits are read again
// (about top / 256 of the row), those >= tau are listed in LDS and ranked by
// comparison.  Where too many reach tau (rows of equal logits, masked vocabularies),
// a radix select over the row finds the threshold and the first of its equals.
//
// Split: one workgroup per row where there are rows enough, else a row is cut into
// chunks whose sums and ordered candidates a second launch joins.
//
// Measured (medians of a trace): 4096 rows of 151936 bf16 logits 246 us (5.1 TB/s; 215 at
// best) and their gradient 410 us (6.1 TB/s read and written); 700 rows of 10007 float32
// logits with five alternatives 16 us and 14; eight rows with 20 alternatives 11 us and 8
// for the join, both a chain of waits: a chunk's loads, the sums, the threshold by 256
// comparisons a thread, the ranks.
#include "common.h"

#define LP_THREADS 256
#define LP_WAVES (LP_THREADS / 64)
#define LP_MAX_TOP 64
#define LP_LIST 512  // candidates ranked by comparison
#define LP_LOG2E 1.44269504088896341f
#define LP_LN2 0.69314718055994531f

// Running maximum of the raw logits and sums in base 2: with y = (logit - m) * c, c =
// log2 e / T, s = sum 2^y and t = sum 2^y y.
struct Softmax {
  float m, s, t;
  static __device__ __forceinline__ Softmax none() { return {-INFINITY, 0.f, 0.f}; }
  __device__ __forceinline__ void rescale(float to, float c) {
    if (m > -INFINITY) {
      const float d = fmaxf((m - to) * c, -1e30f), f = __builtin_amdgcn_exp2f(d);
      t = f * fmaf(s, d, t);
      s *= f;
    }
    m = to;
  }
  __device__ __forceinline__ void join(const Softmax& o, float c) {
    const float to = fmaxf(m, o.m);
    Softmax b = o;
    if (to > m) rescale(to, c);
    if (to > b.m) b.rescale(to, c);
    s += b.s;
    t += b.t;
  }
  template <int N>
  __device__ __forceinline__ void add(const float* x, float c) {
    float g = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) g = fmaxf(g, x[i]);
    if (g > m) rescale(g, c);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = (x[i] - base) * c;
      const float e = __builtin_amdgcn_exp2f(y);
      s += e;
      t = fmaf(e, fmaxf(y, -1e30f), t);  // 0 * -inf does not count
    }
  }
};

__device__ __forceinline__ Softmax wave_join(Softmax a, float c) {
  const float to = wave_max(a.m);  // one rescaling, then sums
  if (to > a.m) a.rescale(to, c);
  a.s = wave_sum(a.s);
  a.t = wave_sum(a.t);
  return a;
}

// Unsigned keys in the order of the floats; NaN lowest, both zeros alike.  0 is
// below every key.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (!(x == x)) return 1u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k <= 1u) return NAN;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// One whole number per logit: larger ones first, the lower index among equals.
__device__ __forceinline__ uint64_t entry_of(uint32_t key, uint32_t index) {
  return (uint64_t)key << 32 | (0xffffffffu - index);
}

// 16 bytes of a row.
template <typename T> struct Granule;
template <> struct Granule<bf16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const bf16_t* p, float* v) { Vec8<bf16_t>::load(p, v); }
};
template <> struct Granule<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
};

// A row's elements: up to N - 1 before the first 16-byte boundary, whole granules, and
// up to N - 1 behind them.
struct RowParts {
  int head, granules, tail;  // tail: its first element
  template <typename T> static __device__ __forceinline__ RowParts of(const T* x, int V) {
    constexpr int N = Granule<T>::N;
    const int head = min((int)(-(intptr_t)x & 15) / (int)sizeof(T), V);
    const int g = (V - head) / N;
    return {head, g, head + g * N};
  }
};

struct TopShared {
  uint64_t list[LP_LIST];
  uint64_t sorted[LP_MAX_TOP];
  uint32_t keys[LP_THREADS];
  uint32_t hist[256];
  int members[LP_THREADS];
  int scan[LP_WAVES];
  uint32_t threshold, digit;
  int count, listed, above;
};

// The top-th largest of the workgroup's keys into sh.threshold: the smallest of those
// that fewer than `top` exceed.
__device__ __forceinline__ void publish_threshold(TopShared& sh, uint32_t key, int top) {
  sh.keys[threadIdx.x] = key;
  if (threadIdx.x == 0) {
    sh.count = sh.listed = 0;
    sh.threshold = 0xffffffffu;
  }
  __syncthreads();
  int above = 0;
  const uint4* k4 = reinterpret_cast<const uint4*>(sh.keys);
#pragma unroll 8
  for (int i = 0; i < LP_THREADS / 4; ++i) {
    const uint4 k = k4[i];
    above += (k.x > key) + (k.y > key) + (k.z > key) + (k.w > key);
  }
  if (above < top) atomicMin(&sh.threshold, key);
  __syncthreads();
}

// The `top` largest of the listed entries, in order, into sh.sorted; 0 where there are
// fewer.
__device__ __forceinline__ void rank_list(TopShared& sh, int n, int top) {
  for (int i = threadIdx.x; i < top; i += LP_THREADS) sh.sorted[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += LP_THREADS) {
    const uint64_t e = sh.list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += sh.list[j] > e;
    if (rank < top) sh.sorted[rank] = e;
  }
  __syncthreads();
}

// Radix select of the elements [first, last) of a row: those above the top-th largest
// key, and the first of its equals, are listed (top of them, fewer if the range has
// fewer).  Any data, whole passes over the range.
template <typename T>
__device__ void select_any(TopShared& sh, const T* x, int first, int last, int top) {
  const int n = last - first, want = min(top, n);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t prefix = 0;
  int need = want;  // rank of the threshold among the keys with the prefix found so far
  for (int shift = 24; shift >= 0; shift -= 8) {
    sh.hist[threadIdx.x] = 0;
    __syncthreads();
    for (int c = first + threadIdx.x; c < last; c += LP_THREADS) {
      const uint32_t k = order_key(Elem<T>::load(x, c));
      if (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
      // the first lane's digit is counted once for all lanes that have it: rows of
      // equal logits would queue up at one counter
      const uint32_t digit = (k >> shift) & 255u, first_digit = __builtin_amdgcn_readfirstlane(digit);
      const uint64_t alike = __ballot(digit == first_digit);
      if (digit != first_digit) atomicAdd(&sh.hist[digit], 1u);
      else if ((alike & ((1ull << lane) - 1)) == 0) atomicAdd(&sh.hist[digit], (uint32_t)__popcll(alike));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int left = need, d = 255;
      while (d > 0 && (int)sh.hist[d] < left) left -= sh.hist[d--];
      sh.digit = d;
      sh.above = left;
    }
    __syncthreads();
    prefix |= sh.digit << shift;
    need = sh.above;
    __syncthreads();
  }
  // listed: everything above the threshold (fewer than want), then the first `need` equals
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
  int equals = 0;
  for (int base = first; base < last; base += LP_THREADS) {
    const int c = base + threadIdx.x;
    const uint32_t k = c < last ? order_key(Elem<T>::load(x, c)) : 0u;
    if (k > prefix) sh.list[atomicAdd(&sh.listed, 1)] = entry_of(k, c);
    const uint64_t same = __ballot(k == prefix);
    if (lane == 0) sh.scan[wave] = __popcll(same);
    __syncthreads();
    int before = equals, all = equals;
    for (int w = 0; w < LP_WAVES; ++w) {
      if (w < wave) before += sh.scan[w];
      all += sh.scan[w];
    }
    before += __popcll(same & ((1ull << lane) - 1));
    // places from the end of the list: the ones above the threshold fill its start
    if (k == prefix && before < need) sh.list[want - 1 - before] = entry_of(k, c);
    equals = all;
    __syncthreads();
  }
}

// The `top` first of the elements that this workgroup's threads went through, sorted
// into sh.sorted: granules [g0, g1) (thread j those at g0 + j + 256 i), the row's head
// and tail where they belong to it (thread j its element j).  `each` gives a thread's
// granules again where it holds them, else (HELD false) the members' are read again.
template <bool HELD, typename T, typename Each>
__device__ void select_top(TopShared& sh, const T* x, const RowParts& parts, int g0, int g1,
                           bool has_head, bool has_tail, int V, float largest, int top, Each each) {
  constexpr int N = Granule<T>::N;
  publish_threshold(sh, order_key(largest), top);
  const uint32_t tau = sh.threshold;
  const bool member = order_key(largest) >= tau;
  if (member) {
    const int at = atomicAdd(&sh.count, 1);
    if (!HELD) sh.members[at] = threadIdx.x;
  }
  __syncthreads();
  const int members = sh.count, rounds = (g1 - g0 + LP_THREADS - 1) / LP_THREADS;
  auto list = [&](float v, int index) {
    const uint32_t k = order_key(v);
    if (k < tau) return;
    const int at = atomicAdd(&sh.listed, 1);
    if (at < LP_LIST) sh.list[at] = entry_of(k, index);
  };
  const int lo = has_head ? 0 : parts.head + g0 * N, hi = has_tail ? V : parts.head + g1 * N;
  // distinct logits have `top` members; with far more of them tau is a value that the
  // row is full of, which the list cannot hold
  const bool few = members <= 2 * top + 64;
  if (few) {
    if constexpr (HELD) {
      if (member) each(list);
    } else {
      for (int u = threadIdx.x; u < members * rounds; u += LP_THREADS) {
        const int g = g0 + sh.members[u % members] + u / members * LP_THREADS;
        if (g >= g1) continue;
        float v[N];
        const int c = parts.head + g * N;
        Granule<T>::load(x + c, v);
#pragma unroll
        for (int i = 0; i < N; ++i) list(v[i], c + i);
      }
    }
    if (has_head && (int)threadIdx.x < parts.head) list(Elem<T>::load(x, threadIdx.x), threadIdx.x);
    if (has_tail && parts.tail + (int)threadIdx.x < V)
      list(Elem<T>::load(x, parts.tail + threadIdx.x), parts.tail + threadIdx.x);
  }
  __syncthreads();
  int n = sh.listed;
  const int want = min(top, hi - lo);
  __syncthreads();
  if (!few || n > LP_LIST || n < want) {  // fewer: NaN, which no thread's largest shows
    select_any(sh, x, lo, hi, top);
    n = want;
  }
  rank_list(sh, n, top);
}

struct LogProbArgs {
  const int64_t* targets;
  float *log_prob, *entropy, *stats, *top_log_prob;
  int64_t* top_ids;
  Softmax* part;      // [rows, chunks]
  uint64_t* entries;  // [rows, chunks, top]
  int64_t ld, ignore;
  int V, top, chunks, chunk_granules;
  float inv_t;
};

// A row's results from its sums (every thread) and its ordered entries (LDS).
template <typename T>
__device__ void finish_row(const LogProbArgs& a, const T* x, int64_t row, const Softmax& r,
                           const uint64_t* sorted) {
  const bool empty = r.m == -INFINITY && r.s == 0.f;
  const float log_s = logf(r.s);
  if (threadIdx.x == 0) {
    const int64_t tg = a.targets[row];
    float lp = 0.f;
    if (tg != a.ignore) {
      const bool known = tg >= 0 && tg < a.V;
      lp = !known ? NAN : empty ? -INFINITY : (Elem<T>::load(x, tg) - r.m) * a.inv_t - log_s;
    }
    a.log_prob[row] = lp;
    a.entropy[row] = empty ? 0.f : log_s - r.t / r.s * LP_LN2;
    a.stats[2 * row] = r.m;
    a.stats[2 * row + 1] = log_s;
  }
  for (int k = threadIdx.x; k < a.top; k += LP_THREADS) {
    const uint64_t e = sorted[k];
    a.top_ids[row * a.top + k] = 0xffffffffu - (uint32_t)e;
    a.top_log_prob[row * a.top + k] =
        empty ? -INFINITY : (key_value((uint32_t)(e >> 32)) - r.m) * a.inv_t - log_s;
  }
}

#define LP_HELD 4  // granules a thread holds where a chunk has no more than that

template <typename T, bool TOP, bool HELD>
__global__ void __launch_bounds__(LP_THREADS)
token_log_probs_kernel(const T* __restrict__ logits, LogProbArgs a) {
  constexpr int N = Granule<T>::N;
  __shared__ __attribute__((aligned(16))) TopShared sh;
  __shared__ float red[3][LP_WAVES];
  const int64_t row = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x % a.chunks);
  const T* x = logits + row * a.ld;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const RowParts parts = RowParts::of(x, a.V);
  const int g0 = min(chunk * a.chunk_granules, parts.granules);
  const int g1 = chunk == a.chunks - 1 ? parts.granules : min(g0 + a.chunk_granules, parts.granules);
  const bool has_head = chunk == 0, has_tail = chunk == a.chunks - 1;
  const float c = a.inv_t * LP_LOG2E;
  Softmax r = Softmax::none();
  float v[LP_HELD][N];
  int g = g0 + threadIdx.x;
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < LP_HELD; ++j)
      if (g + j * LP_THREADS < g1) Granule<T>::load(x + parts.head + (g + j * LP_THREADS) * N, v[j]);
#pragma unroll
    for (int j = 0; j < LP_HELD; ++j)
      if (g + j * LP_THREADS < g1) r.add<N>(v[j], c);
  } else {
    for (; g + (LP_HELD - 1) * LP_THREADS < g1; g += LP_HELD * LP_THREADS) {
#pragma unroll
      for (int j = 0; j < LP_HELD; ++j) Granule<T>::load(x + parts.head + (g + j * LP_THREADS) * N, v[j]);
      r.add<LP_HELD * N>(v[0], c);
    }
    for (; g < g1; g += LP_THREADS) {
      Granule<T>::load(x + parts.head + g * N, v[0]);
      r.add<N>(v[0], c);
    }
  }
  if (has_head && (int)threadIdx.x < parts.head) {
    const float v = Elem<T>::load(x, threadIdx.x);
    r.add<1>(&v, c);
  }
  if (has_tail && parts.tail + (int)threadIdx.x < a.V) {
    const float v = Elem<T>::load(x, parts.tail + threadIdx.x);
    r.add<1>(&v, c);
  }
  const float mine = r.m;  // this thread's largest logit
  r = wave_join(r, c);
  if (lane == 0) { red[0][wave] = r.m; red[1][wave] = r.s; red[2][wave] = r.t; }
  __syncthreads();
  r = {red[0][0], red[1][0], red[2][0]};
#pragma unroll
  for (int w = 1; w < LP_WAVES; ++w) r.join({red[0][w], red[1][w], red[2][w]}, c);
  if constexpr (TOP)
    select_top<HELD>(sh, x, parts, g0, g1, has_head, has_tail, a.V, mine, a.top, [&](auto list) {
#pragma unroll
      for (int j = 0; j < LP_HELD; ++j)
        if (g + j * LP_THREADS < g1)
#pragma unroll
          for (int i = 0; i < N; ++i) list(v[j][i], parts.head + (g + j * LP_THREADS) * N + i);
    });
  if (a.chunks == 1) {
    finish_row(a, x, row, r, sh.sorted);
    return;
  }
  const int64_t at = row * a.chunks + chunk;
  if (threadIdx.x == 0) a.part[at] = r;
  if constexpr (TOP)
    for (int k = threadIdx.x; k < a.top; k += LP_THREADS) a.entries[at * a.top + k] = sh.sorted[k];
}

// Joins a row's chunks, one workgroup each: sums in chunk order, then the largest of
// the chunks' entries.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
token_log_probs_join_kernel(const T* __restrict__ logits, LogProbArgs a) {
  __shared__ __attribute__((aligned(16))) TopShared sh;
  const int64_t row = blockIdx.x;
  const float c = a.inv_t * LP_LOG2E;
  const int lane = threadIdx.x & 63;
  // every wave sums the same way
  Softmax r = Softmax::none();
  for (int k = lane; k < a.chunks; k += 64) r.join(a.part[row * a.chunks + k], c);
  r = wave_join(r, c);
  if (a.top) {
    // a chunk's entries are in order: its first bounds the rest
    const uint64_t* e = a.entries + row * a.chunks * a.top;
    const int n = a.chunks * a.top;
    uint64_t best = 0;
    for (int i = threadIdx.x; i < n; i += LP_THREADS) best = max(best, e[i]);
    publish_threshold(sh, (uint32_t)(best >> 32), a.top);
    const uint32_t tau = sh.threshold;
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
      const uint64_t v = e[i];
      if (v == 0 || (uint32_t)(v >> 32) < tau) continue;
      const int at = atomicAdd(&sh.listed, 1);
      if (at < LP_LIST) sh.list[at] = v;
    }
    __syncthreads();
    const int listed = sh.listed;
    __syncthreads();
    if (listed <= LP_LIST) {
      rank_list(sh, listed, a.top);
    } else {  // many equals: each next one is the largest below the one before
      uint64_t last = ~0ull;
      for (int k = 0; k < a.top; ++k) {
        uint64_t m = 0;
        for (int i = threadIdx.x; i < n; i += LP_THREADS)
          if (e[i] < last) m = max(m, e[i]);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) m = max(m, (uint64_t)__shfl_xor((unsigned long long)m, off, 64));
        __syncthreads();
        if (lane == 0) sh.list[threadIdx.x >> 6] = m;
        __syncthreads();
        for (int w = 0; w < LP_WAVES; ++w) m = max(m, sh.list[w]);
        if (threadIdx.x == 0) sh.sorted[k] = m;
        last = m;
      }
      __syncthreads();
    }
  }
  finish_row(a, logits + row * a.ld, row, r, sh.sorted);
}

// dlogits = (g_target [c = target] + sum_k g_k [c = top_k] - p (g_target + sum_k g_k)
//            - g_entropy p (log p + entropy)) / T,  log p = (x - m) - log s.
// A stream: each logit read once and each gradient written once, 16 bytes a thread.  The
// few elements with a term of their own are written again behind a barrier.
struct LogProbGrad {
  const int64_t *targets, *top_ids;
  const float *stats, *entropy, *d_log_prob, *d_entropy, *d_top;
  int64_t ld, ignore;
  int V, top, chunks;
  float inv_t;
};

#define LP_BWD_GRANULES (LP_THREADS * 4)

template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
token_log_probs_bwd_kernel(const T* __restrict__ logits, LogProbGrad a, T* __restrict__ dlogits) {
  constexpr int N = Granule<T>::N;
  const int64_t row = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x % a.chunks);
  const T* x = logits + row * a.ld;
  T* out = dlogits + row * (int64_t)a.V;
  const float m = a.stats[2 * row], log_s = a.stats[2 * row + 1];
  const bool empty = m == -INFINITY && log_s == -INFINITY;
  const int64_t tg = a.targets[row];
  float gt = a.d_log_prob && tg != a.ignore ? a.d_log_prob[row] : 0.f;
  const bool bad = gt != 0.f && (tg < 0 || tg >= a.V);
  if (bad) gt = NAN;  // as the log probability is
  const float none = bad ? NAN : 0.f;  // the gradient of a row in which no token can be
  const float gh = a.d_entropy ? a.d_entropy[row] : 0.f;
  float all = gt;
  if (a.d_top)
    for (int k = 0; k < a.top; ++k) all += a.d_top[row * a.top + k];
  const float flat = fmaf(gh, a.entropy[row], all);
  const float base = empty ? 0.f : m;
  auto gradient = [&](float v) {  // without the elements' own terms
    const float lp = (v - base) * a.inv_t - log_s;
    const float p = __builtin_amdgcn_exp2f(lp * LP_LOG2E);
    return -p * fmaf(gh, fmaxf(lp, -1e4f), flat) * a.inv_t;  // p is 0 long before -1e4
  };
  // parts by the gradient's alignment; logits that lie otherwise are read one by one
  const RowParts parts = RowParts::of(out, a.V);
  const bool together = ((uintptr_t)(x + parts.head) & 15) == 0;
  // chunks are counted for the most granules a row can have: the last one may start behind
  // this row's, and its elements are then the tail alone
  const int g0 = min(chunk * LP_BWD_GRANULES, parts.granules), g1 = min(g0 + LP_BWD_GRANULES, parts.granules);
#pragma unroll 2
  for (int g = g0 + threadIdx.x; g < g1; g += LP_THREADS) {
    const int at = parts.head + g * N;
    float v[N];
    if (together) Granule<T>::load(x + at, v);
    else
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = Elem<T>::load(x, at + i);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = empty ? none : gradient(v[i]);
    if constexpr (N == 8) Vec8<T>::store_nt(out + at, v);
    else __builtin_nontemporal_store(nt_f32x4_t{v[0], v[1], v[2], v[3]}, reinterpret_cast<nt_f32x4_t*>(out + at));
  }
  const bool last = chunk == a.chunks - 1;
  auto single = [&](int at) { Elem<T>::store(out, at, empty ? none : gradient(Elem<T>::load(x, at))); };
  if (chunk == 0 && (int)threadIdx.x < parts.head) single(threadIdx.x);
  if (last && parts.tail + (int)threadIdx.x < a.V) single(parts.tail + threadIdx.x);
  if (empty) return;
  __syncthreads();
  const int lo = chunk == 0 ? 0 : parts.head + g0 * N, hi = last ? a.V : parts.head + g1 * N;
  const int n = a.d_top ? a.top : 0;
  for (int k = threadIdx.x; k <= n; k += LP_THREADS) {
    const int64_t at = k < n ? a.top_ids[row * a.top + k] : tg;
    if (at < lo || at >= hi || (k == n && gt == 0.f)) continue;
    float own = at == tg ? gt : 0.f;
    bool listed = false;
    for (int j = 0; j < n; ++j)
      if (a.top_ids[row * a.top + j] == at) {
        own += a.d_top[row * a.top + j];
        listed = true;
      }
    if (k == n && listed) continue;  // the alternative's thread writes it
    Elem<T>::store(out, at, fmaf(own, a.inv_t, gradient(Elem<T>::load(x, at))));
  }
}

// ----------------------------------------------------------------------------
// Host
// ----------------------------------------------------------------------------
static int check_shape(int64_t rows, int64_t vocab, int64_t top, int64_t ld, float inv_t) {
  ALODLM_CHECK_ARG(rows >= 0 && rows < (1ll << 24), "token_log_probs: rows out of range");
  ALODLM_CHECK_ARG(vocab >= 1 && vocab < (1ll << 30) && ld >= vocab,
                   "token_log_probs: vocabulary or row stride out of range");
  ALODLM_CHECK_ARG(top >= 0 && top <= LP_MAX_TOP && top <= vocab,
                   "token_log_probs: top must be 0 to 64 and at most the vocabulary");
  ALODLM_CHECK_ARG(inv_t > 0.f && inv_t * LP_LOG2E < INFINITY,
                   "token_log_probs: the temperature must be positive, its inverse times log2 e finite");
  return ALODLM_OK;
}

// Chunks of a row: one where the rows alone give every compute unit two workgroups,
// else as many as make 256 workgroups (few rows, where the join's latency counts) or
// 1024, of 2048 elements at least.
static int64_t row_chunks(int64_t rows, int64_t vocab) {
  if (rows >= 512 || rows == 0) return 1;
  const int64_t total = rows < 32 ? 256 : 1024;
  const int64_t want = (total + rows - 1) / rows, most = max(vocab / 2048, (int64_t)1);
  return min(min(want, most), (int64_t)128);
}

extern "C" int64_t alodlm_token_log_probs_workspace(int64_t rows, int64_t vocab, int64_t top) {
  const int64_t chunks = row_chunks(rows, vocab);
  // 8-byte entries first, then three floats a chunk
  return chunks == 1 ? 0 : rows * chunks * (2 * top + 3);
}

extern "C" int alodlm_token_log_probs(const void* logits, int64_t ld, const int64_t* targets,
                                      int64_t rows, int64_t vocab, int64_t top,
                                      float inv_temperature, int64_t ignore, float* log_prob,
                                      float* entropy, float* stats, float* top_log_prob,
                                      int64_t* top_ids, float* workspace, int dtype, void* stream) {
  const int rc = check_shape(rows, vocab, top, ld, inv_temperature);
  if (rc) return rc;
  if (rows == 0) return ALODLM_OK;
  ALODLM_CHECK_ARG(top == 0 || (top_log_prob && top_ids), "token_log_probs: no room for the alternatives");
  ALODLM_CHECK_ARG(logits && targets && log_prob && entropy && stats, "token_log_probs: the call lacks an array");
  const int64_t chunks = row_chunks(rows, vocab);
  ALODLM_CHECK_ARG(chunks == 1 || workspace, "token_log_probs: no workspace");
  ALODLM_CHECK_ARG(chunks == 1 || (uintptr_t)workspace % 8 == 0, "token_log_probs: workspace not 8-byte aligned");
  const hipStream_t st = as_stream(stream);
  ALODLM_DISPATCH(dtype, T, {
    const int64_t granules = (vocab * (int64_t)sizeof(T) + 15) / 16;
    LogProbArgs a = {targets, log_prob, entropy, stats, top_log_prob, top_ids, nullptr,
                     reinterpret_cast<uint64_t*>(workspace), ld, ignore, (int)vocab, (int)top,
                     (int)chunks, (int)((granules + chunks - 1) / chunks), inv_temperature};
    if (chunks > 1) a.part = reinterpret_cast<Softmax*>(workspace + 2 * rows * chunks * top);
    const unsigned grid = (unsigned)(rows * chunks);
    // the last chunk has what the others leave, never more than they have
    const bool held = a.chunk_granules <= LP_HELD * LP_THREADS;
    if (!top) token_log_probs_kernel<T, false, false><<<grid, LP_THREADS, 0, st>>>((const T*)logits, a);
    else if (held) token_log_probs_kernel<T, true, true><<<grid, LP_THREADS, 0, st>>>((const T*)logits, a);
    else token_log_probs_kernel<T, true, false><<<grid, LP_THREADS, 0, st>>>((const T*)logits, a);
    if (chunks > 1) token_log_probs_join_kernel<T><<<(unsigned)rows, LP_THREADS, 0, st>>>((const T*)logits, a);
  });
  ALODLM_CHECK_LAUNCH("token_log_probs");
  return ALODLM_OK;
}

extern "C" int alodlm_token_log_probs_bwd(const void* logits, int64_t ld, const int64_t* targets,
                                          const int64_t* top_ids, const float* stats,
                                          const float* entropy, const float* d_log_prob,
                                          const float* d_entropy, const float* d_top, int64_t rows,
                                          int64_t vocab, int64_t top, float inv_temperature,
                                          int64_t ignore, void* dlogits, int dtype, void* stream) {
  const int rc = check_shape(rows, vocab, top, ld, inv_temperature);
  if (rc) return rc;
  if (rows == 0) return ALODLM_OK;
  ALODLM_CHECK_ARG(!d_top || top == 0 || top_ids, "token_log_probs_bwd: no alternatives");
  ALODLM_CHECK_ARG(logits && targets && stats && entropy && dlogits, "token_log_probs_bwd: the call lacks an array");
  ALODLM_DISPATCH(dtype, T, {
    const int64_t granules = (vocab * (int64_t)sizeof(T) + 15) / 16;
    const int64_t chunks = (granules + LP_BWD_GRANULES - 1) / LP_BWD_GRANULES;
    ALODLM_CHECK_ARG(rows * chunks < (1ll << 31), "token_log_probs_bwd: too many rows in one call");
    const LogProbGrad a = {targets, top_ids, stats, entropy, d_log_prob, d_entropy, d_top, ld, ignore,
                           (int)vocab, (int)top, (int)chunks, inv_temperature};
    token_log_probs_bwd_kernel<T><<<(unsigned)(rows * chunks), LP_THREADS, 0, as_stream(stream)>>>(
        (const T*)logits, a, (T*)dlogits);
  });
  ALODLM_CHECK_LAUNCH("token_log_probs_bwd");
  return ALODLM_OK;
}
