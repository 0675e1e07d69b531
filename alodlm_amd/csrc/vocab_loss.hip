// Losses against a few known tokens a row over logits in memory: the rows' known tokens,
// sums over the vocabulary, losses, gradients; and a teacher's divergence from a student's
// logits (vocab_loss.h has the mathematics).  linear_loss.hip has the same without logits.
//
// The known tokens are marked in a bit map of the row's part in LDS, whose bytes lie as the
// 16-byte pieces of the row do: one byte read a piece says whether any of its logits has to
// be left out, so the pass over the row stays a stream.
#include <type_traits>

#include "vocab_loss.h"

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int64_t MAX_PART = 1 << 18;  // tokens of a part

// ---------------------------------------------------------------------------
// A row's known tokens, a wave a row: lane l has the places l + 64 j.
// ---------------------------------------------------------------------------
constexpr int HELD = VL_MAX_KNOWN / 64;

struct RowKnown {
  int id[HELD];          // VL_NONE: none
  float q[HELD], log_q[HELD];
  int place[HELD];       // where it is kept: the ids in ascending order, each once
  float mass, q_rest;
  bool bad, counted;
};

// Ranks come from comparisons with all others (LDS broadcasts of four).  `ids`: this wave's,
// room for the known tokens rounded up to four.
__device__ __forceinline__ void known_of_row(const GivenRows& given, int64_t row, int* ids, RowKnown& r) {
  const int lane = threadIdx.x & 63, K = given.known;
  bool bad = false, any = false;
  double mass = 0.0;
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int i = lane + 64 * j;
    r.id[j] = VL_NONE;
    r.q[j] = r.log_q[j] = 0.f;
    r.place[j] = i;
    if (64 * j >= K) continue;
    if (i < K) {
      const int64_t id = given.targets ? given.targets[row] : given.ids[row * K + i];
      const bool none = given.targets ? id == given.ignore : id < 0;
      bad |= !none && !(id >= 0 && id < given.vocab);
      any |= !none;
      if (!none && id >= 0 && id < given.vocab) {
        r.id[j] = (int)id;
        const double q = given.targets ? 1.0 : exp((double)given.log_q[row * K + i]);
        mass += q;
        r.q[j] = (float)q;
        // 0 ln 0 = 0; NaN stays
        r.log_q[j] = given.targets || q == 0.0 ? 0.f : given.log_q[row * K + i];
      }
    }
    if (i < (K + 3) / 4 * 4) ids[i] = r.id[j];
  }
  __builtin_amdgcn_wave_barrier();
  __threadfence_block();
  r.mass = (float)wave_sum_d(mass);
  r.counted = __any(any);
  r.bad = __any(bad);
  r.q_rest = given.rest && r.counted ? (float)fmax(1.0 - wave_sum_d(mass), 0.0) : 0.f;
  // places whose id no earlier place has
  uint64_t firsts[HELD];
  bool twice = false;
  const int4* four = reinterpret_cast<const int4*>(ids);
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int i = lane + 64 * j, id = r.id[j];
    firsts[j] = 0;
    if (64 * j >= K) continue;
    int rank = 0;
    bool again = false;
#pragma unroll 4
    for (int n = 0; n < (K + 3) / 4; ++n) {
      const int4 o = four[n];
      const int other[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool before = 4 * n + e < i;
        rank += other[e] < id || (other[e] == id && before);
        again |= other[e] == id && before;
      }
    }
    r.place[j] = rank;  // the absent behind the others
    firsts[j] = __ballot(id != VL_NONE && !again);
    twice |= id != VL_NONE && again;
  }
  if (!__any(twice)) return;
  // an id given more than once: its first place takes the others' probabilities, and they
  // go behind the known ones
  auto is_first = [&](int n) {
    return ((n < 64 ? firsts[0] : n < 128 ? firsts[1] : n < 192 ? firsts[2] : firsts[3]) >> (n & 63) & 1) != 0;
  };
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int i = lane + 64 * j, id = r.id[j];
    if (i >= K) continue;
    const bool known = (firsts[j] >> lane & 1) != 0;
    int place = 0;
    double q = 0.0, terms = 0.0;
#pragma unroll 1
    for (int n = 0; n < K; ++n) {
      const int other = ids[n];
      place += is_first(n) ? !known || other < id : !known && n < i;
      if (known && other == id) {
        const double lq = given.log_q[row * K + n], one = exp(lq);
        q += one;
        if (one != 0.0) terms += one * lq;
      }
    }
    r.id[j] = known ? id : VL_NONE;
    r.q[j] = (float)q;
    r.log_q[j] = q != 0.0 ? (float)(terms / q) : 0.f;
    r.place[j] = place;
  }
}

__device__ __forceinline__ void write_info(float* info, const RowKnown& r) {
  info[RI_MASS] = r.mass;
  info[RI_REST] = r.q_rest;
  info[RI_BAD] = r.bad ? 1.f : 0.f;
  info[RI_COUNTED] = r.counted ? 1.f : 0.f;
}

__global__ void __launch_bounds__(THREADS)
known_prepare_kernel(KnownRows k, GivenRows given, int64_t rows) {
  __shared__ __attribute__((aligned(16))) int ids[WAVES][VL_MAX_KNOWN];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * WAVES + wave;
  if (row >= rows) return;
  RowKnown r;
  known_of_row(given, row, ids[wave], r);
#pragma unroll
  for (int j = 0; j < HELD; ++j)
    if (lane + 64 * j < k.known) {
      const int64_t at = row * k.known + r.place[j];
      k.ids[at] = r.id[j];
      k.weight[at] = r.q[j];
      k.log_q[at] = r.log_q[j];
    }
  if (lane == 0) write_info(k.info + 8 * row, r);
}

// ---------------------------------------------------------------------------
// Row sums
// ---------------------------------------------------------------------------
// 16 bytes of a row.
template <typename T> struct Piece;
template <> struct Piece<bf16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const bf16_t* p, float* v) { Vec8<bf16_t>::load(p, v); }
  static __device__ __forceinline__ void store(bf16_t* p, const float* v) { Vec8<bf16_t>::store_nt(p, v); }
};
template <> struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  static __device__ __forceinline__ void store(float* p, const float* v) {
    __builtin_nontemporal_store(nt_f32x4_t{v[0], v[1], v[2], v[3]}, reinterpret_cast<nt_f32x4_t*>(p));
  }
};

struct Running {
  float m, sum;
  template <int N>
  __device__ __forceinline__ void add(const float* x, float c) {
    float g = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) g = fmaxf(g, x[i]);
    if (g > m) {
      if (m > -INFINITY) sum *= __builtin_amdgcn_exp2f((m - g) * c);
      m = g;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += __builtin_amdgcn_exp2f((x[i] - base) * c);
  }
};

// Part blockIdx.x % chunks of row blockIdx.x / chunks: the tokens [lo, hi) of a row's
// `width`.  PREPARED: the known tokens are in k, and their logits go there.
template <typename T, bool PREPARED>
__global__ void __launch_bounds__(THREADS)
row_stats_kernel(const T* __restrict__ logits, int64_t ld, int64_t rows, int width, int64_t first,
                 KnownRows k, GivenRows given, float c, int chunks, int chunk_width,
                 Part* __restrict__ part) {
  constexpr int N = Piece<T>::N;
  extern __shared__ uint32_t map[];
  __shared__ float red[2][WAVES];
  const int64_t row = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x % chunks);
  const int lo = min(chunk * chunk_width, width), hi = min(lo + chunk_width, width);
  const T* x = logits + row * ld + lo;
  const int n = hi - lo;
  // up to N - 1 tokens before the first 16-byte boundary, whole pieces, the rest
  const int head = min((int)(-(intptr_t)x & 15) / (int)sizeof(T), n);
  const int pieces = (n - head) / N, tail = head + pieces * N;
  // token t of the part has bit t - head + N: a piece has its own N bits
  const int words = (n + 2 * N + 31) / 32;
  for (int i = threadIdx.x; i < words; i += THREADS) map[i] = 0;
  __syncthreads();
  const int known = PREPARED ? k.known : given.known;
  for (int i = threadIdx.x; i < known; i += THREADS) {
    int64_t id;
    bool none;
    if constexpr (PREPARED) {
      id = k.ids[row * known + i];
      none = id == VL_NONE;
    } else {
      id = given.targets ? given.targets[row] : given.ids[row * known + i];
      none = given.targets && id == given.ignore;
    }
    // (an id that is none, or outside the vocabulary, is not of any part)
    if (none || id < first + lo || id >= first + hi) continue;
    const int t = (int)(id - first - lo), bit = t - head + N;
    atomicOr(&map[bit >> 5], 1u << (bit & 31));
    if constexpr (PREPARED) k.logit[row * known + i] = Elem<T>::load(x, t);
  }
  __syncthreads();
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(map);
  auto marks = [&](int p) -> uint32_t {  // of piece p
    if constexpr (N == 8) return bytes[p + 1];
    else return bytes[(p + 1) >> 1] >> (4 * ((p + 1) & 1)) & 15u;
  };
  Running r = {-INFINITY, 0.f};
  constexpr int AHEAD = 4;
  float v[AHEAD][N];
  int p = threadIdx.x;
  auto leave_out = [&](float* v, uint32_t bits) {
    if (bits)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = bits >> i & 1 ? -INFINITY : v[i];
  };
  for (; p + (AHEAD - 1) * THREADS < pieces; p += AHEAD * THREADS) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) Piece<T>::load(x + head + (p + j * THREADS) * N, v[j]);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) leave_out(v[j], marks(p + j * THREADS));
    r.add<AHEAD * N>(v[0], c);
  }
  for (; p < pieces; p += THREADS) {
    Piece<T>::load(x + head + p * N, v[0]);
    leave_out(v[0], marks(p));
    r.add<N>(v[0], c);
  }
  auto single = [&](int t) {
    const int bit = t - head + N;
    const float v = map[bit >> 5] >> (bit & 31) & 1 ? -INFINITY : Elem<T>::load(x, t);
    r.add<1>(&v, c);
  };
  if ((int)threadIdx.x < head) single(threadIdx.x);
  if (tail + (int)threadIdx.x < n) single(tail + threadIdx.x);
  // one rescaling, then sums
  const float m = wave_max(r.m), base = m == -INFINITY ? 0.f : m;
  const float s = wave_sum(r.sum * __builtin_amdgcn_exp2f((r.m - base) * c));
  if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = m; red[1][threadIdx.x >> 6] = s; }
  __syncthreads();
  if (threadIdx.x == 0) {
    Part a = {red[0][0], red[1][0]};
    for (int w = 1; w < WAVES; ++w) a = part_join(a, {red[0][w], red[1][w]}, c);
    part[(int64_t)chunk * rows + row] = a;
  }
}

// ---------------------------------------------------------------------------
// Losses: 16 rows a workgroup.  Its threads first take the parts of 16 neighbouring rows
// together, then a wave a row.
// ---------------------------------------------------------------------------
constexpr int FIN_ROWS = 16, FIN_LANES = 64;

// The sum or mean of the rows' losses, by a workgroup of 1024 threads in a fixed order.
__device__ __forceinline__ void reduce_losses(const KnownRows& k, int64_t rows, bool mean, float* loss) {
  __shared__ double total[16], count[16];
  double t = 0.0, n = 0.0;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < rows; r += 1024) {
    t += (double)k.info[8 * r + RI_LOSS];
    n += (double)k.info[8 * r + RI_COUNTED];
  }
  t = wave_sum_d(t);
  n = wave_sum_d(n);
  if ((threadIdx.x & 63) == 0) { total[threadIdx.x >> 6] = t; count[threadIdx.x >> 6] = n; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) { t += total[w]; n += count[w]; }
    const double by = mean ? fmax(n, 1.0) : 1.0;
    loss[0] = (float)(t / by);
    k.call[0] = (float)(1.0 / by);
  }
}

// GIVEN: the known tokens come from the caller, their logits from `logits`.  SCALED: the
// references are whole exponents.
template <typename T, bool GIVEN, bool SCALED>
__global__ void __launch_bounds__(FIN_ROWS * FIN_LANES)
known_finish_kernel(KnownRows k, GivenRows given, const T* __restrict__ logits, int64_t ld,
                    const Part* __restrict__ part, int64_t parts, int64_t rows, float c, int reduction,
                    float* __restrict__ loss) {
  __shared__ Part red[FIN_ROWS][FIN_LANES + 1];
  __shared__ __attribute__((aligned(16))) int ids[GIVEN ? FIN_ROWS : 1][VL_MAX_KNOWN];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, K = k.known;
  const bool cross = given.targets != nullptr;
  const float step = SCALED ? 1.f : c;  // of differences of references
  auto exponent = [&](float z, float ref) { return SCALED ? fmaf(z, c, -ref) : (z - ref) * c; };
  const int64_t row = (int64_t)blockIdx.x * FIN_ROWS + wave;
  RowKnown r;
  float z[HELD];
  if (row < rows) {
    float* info = k.info + 8 * row;
    if constexpr (GIVEN) {
      known_of_row(given, row, ids[wave], r);
#pragma unroll
      for (int j = 0; j < HELD; ++j)
        z[j] = r.id[j] != VL_NONE ? Elem<T>::load(logits, row * ld + r.id[j]) : -INFINITY;
      if (lane == 0) write_info(info, r);
    } else {
#pragma unroll
      for (int j = 0; j < HELD; ++j) {
        const int i = lane + 64 * j;
        const int64_t at = row * K + i;
        r.id[j] = i < K ? k.ids[at] : VL_NONE;
        const bool known = r.id[j] != VL_NONE;
        z[j] = known ? k.logit[at] : -INFINITY;
        r.q[j] = known ? k.weight[at] : 0.f;
        r.log_q[j] = known ? k.log_q[at] : 0.f;
        r.place[j] = i;
      }
      r.mass = info[RI_MASS];
      r.q_rest = info[RI_REST];
      r.bad = info[RI_BAD] != 0.f;
      r.counted = info[RI_COUNTED] != 0.f;
    }
  }
  {
    const int n = threadIdx.x % FIN_ROWS, l = threadIdx.x / FIN_ROWS;
    const int64_t at = (int64_t)blockIdx.x * FIN_ROWS + n;
    Part a = {-INFINITY, 0.f};
    if (at < rows)
#pragma unroll 4
      for (int64_t p = l; p < parts; p += FIN_LANES) a = part_join(a, part[p * rows + at], step);
    red[n][l] = a;
  }
  __syncthreads();
  if (row < rows) {
    const Part mine = red[wave][lane];
    float m = wave_max(mine.m);
    const float base = m == -INFINITY ? 0.f : m;
    const float s_rest = wave_sum(mine.sum * __builtin_amdgcn_exp2f((mine.m - base) * step));
    const bool others = !(s_rest == 0.f);  // a token that is not known can be (or NaN)
    const float m_rest = m;
    // the known tokens join
#pragma unroll
    for (int j = 0; j < HELD; ++j) m = fmaxf(m, SCALED ? part_ref(z[j], c) : z[j]);
    m = wave_max(m);
    const bool none = m == -INFINITY;
    const float top = none ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < HELD; ++j)
      if (r.id[j] != VL_NONE) s += __builtin_amdgcn_exp2f(exponent(z[j], top));
    s = wave_sum(s) + (others ? s_rest * __builtin_amdgcn_exp2f((m_rest - top) * step) : 0.f);
    const float log_s = log2f(s);
    const float log_rest = others ? (m_rest - top) * step + log2f(s_rest) : -INFINITY;
    const bool empty = none && s == 0.f;  // no token can be
    const float p_rest = others ? __builtin_amdgcn_exp2f(log_rest - log_s) : 0.f;
    const float q_rest = others ? r.q_rest : 0.f;
    const float mass = r.mass + q_rest;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      if (lane + 64 * j >= K) continue;
      const int64_t at = row * K + r.place[j];
      if constexpr (GIVEN) k.ids[at] = r.id[j];
      if (r.id[j] == VL_NONE) continue;
      const float own = exponent(z[j], top), log_p = own - log_s;
      if (cross) {
        // -ln p = ln(1 + others / own): small losses keep their digits
        const float x = VL_LN2 * (log_rest - own);
        sum = !others ? 0.f : x > 0.f ? x + log1pf(expf(-x)) : log1pf(expf(x));
        if (!(z[j] < INFINITY)) sum = NAN;
      } else if (r.q[j] != 0.f) {
        sum += r.q[j] * (r.log_q[j] - VL_LN2 * log_p);
      }
      const float p = __builtin_amdgcn_exp2f(log_p);
      k.weight[at] = r.bad ? NAN : empty ? 0.f : cross ? -p_rest : fmaf(mass, p, -r.q[j]);
    }
    sum = wave_sum(sum);
    if (q_rest != 0.f) sum += q_rest * (logf(q_rest) - VL_LN2 * (log_rest - log_s));
    if (empty) sum = r.mass != 0.f ? INFINITY : 0.f;
    if (!r.counted) sum = 0.f;
    if (r.bad) sum = NAN;
    if (lane == 0) {
      float* info = k.info + 8 * row;
      info[RI_M] = top;
      info[RI_LOG] = log_rest;
      info[RI_FACTOR] = r.bad ? NAN : !r.counted || !others ? 0.f : fmaf(mass, p_rest, -q_rest);
      info[RI_LOSS] = sum;
      if (reduction == VL_EACH) loss[row] = sum;
    }
  }
  // one workgroup's rows are all there are (more take a launch of their own: the last
  // workgroup adding up the others' rows needs device-wide fences, which took 70 us of 256)
  if (reduction != VL_EACH && gridDim.x == 1) {
    __syncthreads();
    reduce_losses(k, rows, reduction == VL_MEAN, loss);
  }
}

__global__ void __launch_bounds__(1024)
known_reduce_kernel(KnownRows k, int64_t rows, int mean, float* __restrict__ loss) {
  reduce_losses(k, rows, mean, loss);
}

// ---------------------------------------------------------------------------
// Gradients: a stream.  The known tokens' are written again behind a barrier.  The last rows
// come first: the forward read them last, and the last-level cache may hold them.
// ---------------------------------------------------------------------------
constexpr int GRAD_PIECES = THREADS * 2;

// PARTS: two bf16 parts of each, the value's rounding and what that leaves, in rows r and
// rows + r.
template <typename TI, typename TO, bool PARTS>
__global__ void __launch_bounds__(THREADS)
row_grads_kernel(const TI* logits, int64_t ld, int64_t rows, int width, int64_t first, KnownRows k,
                 float c, Upstream up, TO* out, int64_t ldo, int padded, int chunks) {
  constexpr int N = 8;  // tokens a thread takes at a time
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  int64_t row = block / chunks;
  const int chunk = (int)(block % chunks);
  const bool live = row < rows;
  if (PARTS && !live) row += rows;  // behind both parts
  TO* o = out + row * ldo;
  // the second part
  auto left = [](float v) { const float by = v - bf16_to_float(float_to_bf16(v)); return by - by == 0.f ? by : 0.f; };
  TO* o2 = o + rows * ldo;
  // pieces by the gradient's 16-byte (bf16) or 32-byte (float) alignment
  const int head = min((int)(-(intptr_t)o & (8 * (int)sizeof(TO) - 1)) / (int)sizeof(TO), padded);
  const int pieces = (padded - head) / N, tail = head + pieces * N;
  const int p0 = min(chunk * GRAD_PIECES, pieces), p1 = min(p0 + GRAD_PIECES, pieces);
  const bool last = chunk == chunks - 1;
  const TI* x = logits + (live ? row : 0) * ld;
  float g = 0.f, factor = 0.f, m = 0.f, log_rest = 0.f;
  if (live) {
    const float* info = k.info + 8 * row;
    g = up.row(row);
    m = info[RI_M];
    log_rest = info[RI_LOG];
    factor = row_factor(g, info[RI_FACTOR]);
  }
  const bool flat = factor == 0.f;  // nothing but the known tokens has a gradient
  auto gradient = [&](float v) { return factor * __builtin_amdgcn_exp2f((v - m) * c - log_rest); };
  const bool together = ((uintptr_t)(x + head) & 15) == 0;
#pragma unroll 2
  for (int p = p0 + threadIdx.x; p < p1; p += THREADS) {
    const int at = head + p * N;
    float v[N];
    if (flat) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.f;
    } else {
      if (together && at + N <= width) {
#pragma unroll
        for (int i = 0; i < N; i += Piece<TI>::N) Piece<TI>::load(x + at + i, v + i);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = at + i < width ? Elem<TI>::load(x, at + i) : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = at + i < width ? gradient(v[i]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; i += Piece<TO>::N) Piece<TO>::store(o + at + i, v + i);
    if (PARTS && live) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = left(v[i]);
#pragma unroll
      for (int i = 0; i < N; i += Piece<TO>::N) Piece<TO>::store(o2 + at + i, v + i);
    }
  }
  auto single = [&](int at) {
    const float v = flat || at >= width ? 0.f : gradient(Elem<TI>::load(x, at));
    Elem<TO>::store(o, at, v);
    if (PARTS && live) Elem<TO>::store(o2, at, left(v));
  };
  if (chunk == 0 && (int)threadIdx.x < head) single(threadIdx.x);
  if (last && tail + (int)threadIdx.x < padded) single(tail + threadIdx.x);
  if (!live) return;
  __syncthreads();
  const int lo = chunk == 0 ? 0 : head + p0 * N, hi = min(last ? padded : head + p1 * N, width);
  for (int i = threadIdx.x; i < k.known; i += THREADS) {
    const int id = k.ids[row * k.known + i];
    const int64_t at = (int64_t)id - first;
    if (id == VL_NONE || at < lo || at >= hi) continue;
    const float v = g == 0.f ? 0.f : g * k.weight[row * k.known + i];
    Elem<TO>::store(o, at, v);
    if (PARTS) Elem<TO>::store(o2, at, left(v));
  }
}

// Few rows, tokens first: a thread a token, which reads its logits of all rows.
constexpr int MAX_FEW = 32;

__global__ void __launch_bounds__(THREADS)
few_grads_kernel(const float* __restrict__ logits, int64_t ld, int rows, int width, int64_t first, KnownRows k,
                 float c, Upstream up, float* __restrict__ out, int pad) {
  __shared__ float s_m[MAX_FEW], s_log[MAX_FEW], s_factor[MAX_FEW], s_up[MAX_FEW];
  if ((int)threadIdx.x < rows) {
    const float* info = k.info + 8 * threadIdx.x;
    const float g = up.row(threadIdx.x);
    s_m[threadIdx.x] = info[RI_M];
    s_log[threadIdx.x] = info[RI_LOG];
    s_factor[threadIdx.x] = row_factor(g, info[RI_FACTOR]);
    s_up[threadIdx.x] = g;
  }
  __syncthreads();
  const int lo = blockIdx.x * THREADS, at = lo + threadIdx.x;
  if (at < width) {
    float* o = out + (int64_t)at * pad;
    for (int r = 0; r < pad; r += 4) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = r + e < rows ? s_factor[r + e] : 0.f;
        v[e] = 0.f;
        if (f != 0.f)  // (or NaN)
          v[e] = f * __builtin_amdgcn_exp2f((logits[(r + e) * ld + at] - s_m[r + e]) * c - s_log[r + e]);
      }
      *reinterpret_cast<float4*>(o + r) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  __syncthreads();
  // the known tokens' own
  for (int i = threadIdx.x; i < rows * k.known; i += THREADS) {
    const int r = i / k.known;
    const int64_t t = (int64_t)k.ids[i] - first - lo;
    if (k.ids[i] == VL_NONE || t < 0 || t >= THREADS || lo + t >= width) continue;
    out[(lo + t) * pad + r] = s_up[r] == 0.f ? 0.f : s_up[r] * k.weight[i];
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
void known_prepare_launch(const KnownRows& k, const GivenRows& given, int64_t rows, hipStream_t st) {
  known_prepare_kernel<<<ceil_div_u(rows, WAVES), THREADS, 0, st>>>(k, given, rows);
}

// Parts of a row: one where the rows alone give every compute unit two workgroups, else as
// many as make 256 workgroups (few rows) or 1024, of 2048 tokens at least.
int64_t row_stats_chunks(int64_t rows, int64_t width) {
  const int64_t least = (width + MAX_PART - 1) / MAX_PART;
  if (rows >= 512) return least;
  const int64_t want = ((rows < 32 ? 256 : 1024) + rows - 1) / rows;
  const int64_t most = width / 2048 > 1 ? width / 2048 : 1;
  const int64_t n = want < most ? want : most;
  return n > least ? n : least;
}

template <typename T>
void row_stats_launch(const T* logits, int64_t ld, int64_t rows, int64_t width, int64_t first,
                      const KnownRows& k, const GivenRows& given, bool prepared, float c, int64_t chunks,
                      Part* part, hipStream_t st) {
  const int64_t chunk_width = ((width + chunks - 1) / chunks + 63) / 64 * 64;
  const size_t lds = 4 * (size_t)((chunk_width + 2 * Piece<T>::N + 31) / 32 + 1);
  const unsigned grid = (unsigned)(rows * chunks);
  if (prepared)
    row_stats_kernel<T, true><<<grid, THREADS, lds, st>>>(logits, ld, rows, (int)width, first, k, given, c,
                                                          (int)chunks, (int)chunk_width, part);
  else
    row_stats_kernel<T, false><<<grid, THREADS, lds, st>>>(logits, ld, rows, (int)width, first, k, given, c,
                                                           (int)chunks, (int)chunk_width, part);
}
template void row_stats_launch<float>(const float*, int64_t, int64_t, int64_t, int64_t, const KnownRows&,
                                      const GivenRows&, bool, float, int64_t, Part*, hipStream_t);

template <typename T>
void known_finish_launch(const KnownRows& k, const GivenRows& given, const T* logits, int64_t ld,
                         const Part* part, int64_t parts, int64_t rows, float c, bool scaled,
                         int reduction, float* loss, hipStream_t st) {
  const unsigned grid = ceil_div_u(rows, FIN_ROWS), threads = FIN_ROWS * FIN_LANES;
  if (rows > 0 && logits)
    known_finish_kernel<T, true, false><<<grid, threads, 0, st>>>(k, given, logits, ld, part, parts, rows, c,
                                                                  reduction, loss);
  else if (rows > 0 && scaled)
    known_finish_kernel<T, false, true><<<grid, threads, 0, st>>>(k, given, nullptr, 0, part, parts, rows, c,
                                                                  reduction, loss);
  else if (rows > 0)
    known_finish_kernel<T, false, false><<<grid, threads, 0, st>>>(k, given, nullptr, 0, part, parts, rows, c,
                                                                  reduction, loss);
  if (reduction != VL_EACH && grid != 1)
    known_reduce_kernel<<<1, 1024, 0, st>>>(k, rows, reduction == VL_MEAN, loss);
}
template void known_finish_launch<float>(const KnownRows&, const GivenRows&, const float*, int64_t, const Part*,
                                         int64_t, int64_t, float, bool, int, float*, hipStream_t);

template <typename TI, typename TO>
void row_grads_launch(const TI* logits, int64_t ld, int64_t rows, int64_t width, int64_t first,
                      const KnownRows& k, float c, const Upstream& up, TO* out, int64_t ldo,
                      int64_t padded_rows, int64_t padded, hipStream_t st, bool parts) {
  const int64_t chunks = (padded / 8 + GRAD_PIECES) / GRAD_PIECES;
  if constexpr (!std::is_same<TI, TO>::value)
    if (parts) {
      row_grads_kernel<TI, TO, true><<<(unsigned)((padded_rows - rows) * chunks), THREADS, 0, st>>>(
          logits, ld, rows, (int)width, first, k, c, up, out, ldo, (int)padded, (int)chunks);
      return;
    }
  row_grads_kernel<TI, TO, false><<<(unsigned)(padded_rows * chunks), THREADS, 0, st>>>(
      logits, ld, rows, (int)width, first, k, c, up, out, ldo, (int)padded, (int)chunks);
}
template void row_grads_launch<float, float>(const float*, int64_t, int64_t, int64_t, int64_t, const KnownRows&,
                                             float, const Upstream&, float*, int64_t, int64_t, int64_t,
                                             hipStream_t, bool);
template void row_grads_launch<float, bf16_t>(const float*, int64_t, int64_t, int64_t, int64_t, const KnownRows&,
                                              float, const Upstream&, bf16_t*, int64_t, int64_t, int64_t,
                                              hipStream_t, bool);

void few_grads_launch(const float* logits, int64_t ld, int64_t rows, int64_t width, int64_t first,
                      const KnownRows& k, float c, const Upstream& up, float* out, int64_t pad,
                      hipStream_t st) {
  few_grads_kernel<<<ceil_div_u(width, THREADS), THREADS, 0, st>>>(logits, ld, (int)rows, (int)width, first, k, c,
                                                                  up, out, (int)pad);
}

// ---------------------------------------------------------------------------
// Distillation from logits
// ---------------------------------------------------------------------------
extern "C" int64_t alodlm_vocab_loss_state(int64_t rows, int64_t known) { return known_rows_floats(rows, known); }

extern "C" int64_t alodlm_distillation_workspace(int64_t rows, int64_t vocab) {
  return rows > 0 ? 2 * rows * row_stats_chunks(rows, vocab) : 0;
}

extern "C" int alodlm_distillation(const void* logits, int64_t ld, const int64_t* ids, const float* log_q,
                                   int64_t rows, int64_t vocab, int64_t known, float inv_temperature,
                                   int rest, int reduction, float* loss, float* state,
                                   float* workspace, int dtype, void* stream) {
  const int rc = check_vocab_loss("distillation", rows, vocab, known, inv_temperature, reduction);
  if (rc) return rc;
  ALODLM_CHECK_ARG(ld >= vocab, "distillation: rows overlap");
  if (rows == 0 && reduction == VL_EACH) return ALODLM_OK;
  ALODLM_CHECK_ARG(loss && state && (rows == 0 || (logits && ids && log_q && workspace)),
                   "distillation: the call lacks an array");
  ALODLM_CHECK_ARG((uintptr_t)workspace % 8 == 0, "distillation: workspace not 8-byte aligned");
  const int64_t chunks = rows > 0 ? row_stats_chunks(rows, vocab) : 0;
  ALODLM_CHECK_ARG(rows * chunks < VL_MOST_GROUPS, "distillation: too many rows in one call");
  const hipStream_t st = as_stream(stream);
  const KnownRows k = known_rows(state, rows, known);
  const GivenRows given = {nullptr, ids, log_q, 0, (int)known, (int)vocab, rest != 0};
  const float c = inv_temperature * VL_LOG2E;
  Part* part = reinterpret_cast<Part*>(workspace);
  ALODLM_DISPATCH(dtype, T, {
    if (rows > 0) row_stats_launch<T>((const T*)logits, ld, rows, vocab, 0, k, given, false, c, chunks, part, st);
    known_finish_launch<T>(k, given, rows > 0 ? (const T*)logits : nullptr, ld, part, chunks, rows, c, false,
                           reduction, loss, st);
  });
  ALODLM_CHECK_LAUNCH("distillation");
  return ALODLM_OK;
}

extern "C" int alodlm_distillation_bwd(const void* logits, int64_t ld, const float* state, const float* d_loss,
                                       int64_t rows, int64_t vocab, int64_t known,
                                       float inv_temperature, int reduction, void* dlogits, int dtype,
                                       void* stream) {
  const int rc = check_vocab_loss("distillation_bwd", rows, vocab, known, inv_temperature, reduction);
  if (rc) return rc;
  ALODLM_CHECK_ARG(ld >= vocab, "distillation_bwd: rows overlap");
  if (rows == 0) return ALODLM_OK;
  ALODLM_CHECK_ARG(logits && state && d_loss && dlogits, "distillation_bwd: the call lacks an array");
  ALODLM_CHECK_ARG(rows * ((vocab / 8 + GRAD_PIECES) / GRAD_PIECES) < VL_MOST_GROUPS,
                   "distillation_bwd: too many rows in one call");
  const KnownRows k = known_rows(const_cast<float*>(state), rows, known);  // read only
  const Upstream up = {k.call, d_loss, reduction, 0, inv_temperature};
  ALODLM_DISPATCH(dtype, T, {
    row_grads_launch<T, T>((const T*)logits, ld, rows, vocab, 0, k, inv_temperature * VL_LOG2E, up, (T*)dlogits,
                           vocab, rows, vocab, as_stream(stream), false);
  });
  ALODLM_CHECK_LAUNCH("distillation_bwd");
  return ALODLM_OK;
}
