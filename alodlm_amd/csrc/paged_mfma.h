// What the matrix-core kernels of the paged attention share: 64-key tiles against query
// columns of 16, in transposed products S^T = K Q^T and O^T = V^T P^T on 16x16x32.
//
// The lane that holds query column c = lane % 16 of S^T holds the same column of P^T, so
// the probabilities never leave their registers.  The order in which keys are given to
// the rows of S^T makes a lane's 16 scores 16 keys in a row, lane / 16 saying which 16
// of the 64: row r of subtile i is key (r / 4) * 16 + 4 i + r % 4.  The second product
// then takes a value row's tokens in their order, 8 a fragment; and since page sizes are
// multiples of 16, each lane's 16 keys lie in one page.
//
// 8-bit codes become bf16 times the page's power of two in one instruction a pair
// (v_cvt_scalef32_pk_bf16_fp8), exactly.  Scores, maxima, sums and outputs are float32.
// The second product takes the probabilities in bf16.  Where many columns share a tile
// that is one rounding (2^-8 of a probability, as much again as the output's own), and the
// sum is that of the rounded ones (one more product with ones), so that the weights add
// up to one.  Decoding steps and small windows, which wait for memory, multiply
// the rounding errors as well: the probabilities then have 16 bits, and only the
// output's rounding is left.  64 rows over 585 MB of codes take 118 us so; the values of
// 16-bit pages, which can be inf, are cleared of it for the low parts' products (see
// add_values), which costs a windows' kernel of one column tile 5 % (48 -> 50 us).
#pragma once

#include "paged.h"

#include <type_traits>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

#define PAGED_TILE 64   // keys of a tile
#define PAGED_WAVES 4   // waves of a workgroup

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight e4m3 codes times a power of two as bf16.
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi, float scale) {
  bf16x8 r;
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1];
  r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
  return r;
}

// inf and NaN in a word of codes (bf16 pairs): nonzero where there is any; without them.
template <bool EIGHT>
__device__ __forceinline__ uint32_t special_bits(uint32_t w) {
  return EIGHT ? ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u
               : ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
template <bool EIGHT>
__device__ __forceinline__ uint32_t without_special(uint32_t w) {
  const uint32_t z = special_bits<EIGHT>(w);
  return w & (EIGHT ? ~((z >> 7) * 0xffu) : ~((z >> 15) * 0xffffu));
}

// The sequence, head and keys that a workgroup (or a wave) works on.
struct Span {
  int b, h, slot;
  int held, n, given;    // tokens before the step; rows that take part; rows of the batch
  int sealed, reach;     // ends of the 8-bit pages and of the keys that are there
  int64_t row0;

  template <bool EIGHT>
  static __device__ __forceinline__ Span of(const PagedCache& c, const PagedBatch& bt, int b, int h) {
    Span s;
    s.b = b;
    s.h = h;
    s.given = given_rows(bt, b);
    const int held = bt.held(b, c.page);
    s.n = held < 0 ? 0 : bt.row_count(b, held, c.page);
    s.held = max(held, 0);
    const int end = s.held + s.n;
    s.sealed = EIGHT ? sealed_keys(c, bt, s.held, end, true) : end;
    s.reach = key_end(c, bt, s.sealed, end, EIGHT);
    s.slot = EIGHT ? bt.slot(b, c.slots) : 0;
    s.row0 = bt.first_row(b);
    return s;
  }
  // Keys that row i sees.
  __device__ __forceinline__ int limit(int i) const { return i < n ? min(held + i + 1, reach) : 0; }
  // The page (of the pool, or among all open ones) of the 16 keys from `key` on, as far as
  // [lo, hi) reaches into them; -1 for none.
  template <bool POOL>
  __device__ __forceinline__ int page(const PagedCache& c, const PagedBatch& bt, int key, int lo,
                                      int hi) const {
    if (key + 15 < lo || key >= hi) return -1;
    const int p = key >> c.shift;
    if (!POOL) return slot < 0 ? -1 : open_page(c, slot, p);
    return bt.page_of(b, p, c.pages);
  }
  // The same in two steps, so that no arithmetic waits for the table: its entry (any, for
  // keys past the table), and what page that is.
  __device__ __forceinline__ int entry(const PagedCache& c, const PagedBatch& bt, int key) const {
    return bt.table[(int64_t)b * bt.width + min(key >> c.shift, bt.width - 1)];
  }
  __device__ __forceinline__ int page_in(const PagedCache& c, int entry, int key, int lo, int hi) const {
    return key + 15 < lo || key >= hi || entry < 0 || entry >= c.pages ? -1 : entry;
  }
  // First value of a page's block for this head.
  __device__ __forceinline__ int64_t block(const PagedCache& c, int page, int head_block) const {
    return ((int64_t)page * c.kv_heads + h) * head_block;
  }
  // Exponent of a pool page's keys (side 0) or values (side 1).  Made a scale where that is
  // used: the arithmetic would wait for this load and all that went before it.
  __device__ __forceinline__ int exponent(const PagedCache& c, int page, int side) const {
    return c.exponents[((int64_t)page * 2 + side) * c.kv_heads + h];
  }
};

// Tiles in which some row sees a key that another does not are multiplied with zeros in
// the place of values that are inf or NaN: 0 times one of them would not be 0 for the
// rows that do not see it.  Those that do get them afterwards: the sum of dimension d's
// inf and NaN over keys [from, to) (a probability is positive, and inf times it is inf).
template <int DH, bool EIGHT, typename T>
__device__ __forceinline__ float special_sum(const PagedCache& c, const PagedBatch& bt, const Span& sp,
                                             int d, int from, int to) {
  float sum = 0.f;
  for (int key = from; key < to; ++key) {
    const bool pool = !EIGHT || key < sp.sealed;
    const int page = pool ? sp.page<true>(c, bt, key, key, key + 1) : sp.page<false>(c, bt, key, key, key + 1);
    if (page < 0) continue;
    const int64_t at = sp.block(c, page, c.page * DH) + (int64_t)d * c.page + (key & (c.page - 1));
    const float v = EIGHT && pool ? __builtin_amdgcn_cvt_f32_fp8(((const e4m3_t*)c.values)[at], 0)
                                  : Elem<T>::load((const T*)(EIGHT ? c.open_values : c.values), at);
    if (!(fabsf(v) < INFINITY)) sum += v;
  }
  return sum;
}

// CT times 16 query columns of one wave and what becomes of them.  Column x is row x /
// group and query head h * group + x % group.
template <int DH, int CT> struct Columns {
  static constexpr int FR = DH / 32, DT = DH / 16;  // query fragments, 16-row tiles of the output
  bf16x8 q[CT][FR];
  f32x4 o[CT][DT], l[CT];
  float m[CT];
  int limit[CT];

  // Lane group g holds dims dim(f, g) .. + 8 of fragment f.
  template <typename Dim>
  __device__ __forceinline__ void start(const AttendArgs& a, const Span& s, int first, Dim dim) {
    const int col = threadIdx.x & 15, grp = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const int x = first + t * 16 + col, i = x / a.group, head = s.h * a.group + x % a.group;
      limit[t] = s.limit(i);
      const bf16_t* p = (const bf16_t*)a.q + (s.row0 + i) * a.ldq + (int64_t)head * DH;
#pragma unroll
      for (int f = 0; f < FR; ++f) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (i < s.n) w = *reinterpret_cast<const uint4*>(p + dim(f, grp));
        q[t][f] = __builtin_bit_cast(bf16x8, w);
      }
      m[t] = -INFINITY;
      l[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  // key(i, f): the lane's part of subtile i's rows, dims of fragment f.
  template <typename Key>
  __device__ __forceinline__ void scores(f32x4 (&s)[CT][4], Key key) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int t = 0; t < CT; ++t) s[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < FR; ++f) {
        const bf16x8 k = key(i, f);
#pragma unroll
        for (int t = 0; t < CT; ++t) s[t][i] = mfma16(k, q[t][f], s[t][i]);
      }
    }
  }
  // The same with the next subtile's fragments read while this one's are multiplied (and
  // no further ahead: the registers are taken).
  template <typename Key>
  __device__ __forceinline__ void scores_ahead(f32x4 (&s)[CT][4], Key key) const {
    bf16x8 now[FR], next[FR];
#pragma unroll
    for (int f = 0; f < FR; ++f) now[f] = key(0, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i < 3)
#pragma unroll
        for (int f = 0; f < FR; ++f) next[f] = key(i + 1, f);
#pragma unroll
      for (int t = 0; t < CT; ++t) s[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < FR; ++f)
#pragma unroll
        for (int t = 0; t < CT; ++t) s[t][i] = mfma16(now[f], q[t][f], s[t][i]);
#pragma unroll
      for (int f = 0; f < FR; ++f) now[f] = next[f];
      if (i < 3) __builtin_amdgcn_sched_group_barrier(0x100, FR, 0);  // LDS reads first,
      __builtin_amdgcn_sched_group_barrier(0x8, FR * CT, 0);          // then the products
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // Keys outside [lo, hi), beyond a row's own, or in a page that is missing are hidden.
  __device__ __forceinline__ void hide(f32x4 (&s)[CT][4], int base, int lo, int hi, bool there) const {
    const int grp = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const int end = there ? min(hi, limit[t]) : 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = base + grp * 16 + i;
        if (!(key >= lo && key < end)) s[t][i / 4][i % 4] = -INFINITY;
      }
    }
  }
  // Scores -> probabilities in bf16.  The reference m that they are taken against is the
  // running maximum, but follows it only when that has grown by more than 2^8: until
  // then the probabilities stay below 2^8 of what they would be, which costs float32
  // sums and bf16 factors nothing, and no output is rescaled.
  // With `low` the rounding errors of the probabilities are kept as bf16 too.
  template <bool LOW>
  __device__ __forceinline__ void softmax(const f32x4 (&s)[CT][4], bf16x8 (&p)[CT][2], bf16x8 (&low)[CT][2],
                                          float scale2) {
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      float top = s[t][0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[t][i / 4][i % 4]);
      top *= scale2;
      if (__any(top > m[t] + 8.f)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));  // the four lanes of a column agree
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float to = fmaxf(m[t], top);
        const float f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[t] - to);
        m[t] = to;
        l[t] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] *= f;
      }
      const float base = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[t][i / 4][i % 4], scale2, -base));
        p[t][i / 8][i % 8] = (__bf16)e;
        if (LOW) low[t][i / 8][i % 8] = (__bf16)(e - (float)p[t][i / 8][i % 8]);
      }
    }
  }
  // value(d, j): dimension d * 16 + lane % 16, keys (lane / 16) * 16 + 8 j .. + 8.  PLAIN:
  // 16-bit values, which can be inf: a low part, which has either sign or is zero, would
  // make NaN of it, so the low parts are multiplied with zeros in the place of inf and NaN.
  template <bool PLAIN, typename Value>
  __device__ __forceinline__ void add_values(const bf16x8 (&p)[CT][2], const bf16x8 (&low)[CT][2], Value value) {
    bf16x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int t = 0; t < CT; ++t) l[t] = mfma16(ones, low[t][j], mfma16(ones, p[t][j], l[t]));
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const bf16x8 v = value(d, j);
        bf16x8 v_low = v;
        if constexpr (PLAIN) {
          uint4 w = __builtin_bit_cast(uint4, v);
          w = make_uint4(without_special<false>(w.x), without_special<false>(w.y), without_special<false>(w.z),
                         without_special<false>(w.w));
          v_low = __builtin_bit_cast(bf16x8, w);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) o[t][d] = mfma16(v_low, low[t][j], mfma16(v, p[t][j], o[t][d]));
      }
    }
  }
  // The same four fragments at a time, the next four read meanwhile.
  template <bool LOW, typename Value>
  __device__ __forceinline__ void add_values_ahead(const bf16x8 (&p)[CT][2], const bf16x8 (&low)[CT][2],
                                                   Value value) {
    bf16x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.f;
    constexpr int STEPS = 2 * DT / 4;
    bf16x8 now[4], next[4];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < 4; ++k) now[k] = value(k, 0);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      l[t] = mfma16(ones, p[t][1], mfma16(ones, p[t][0], l[t]));
      if (LOW) l[t] = mfma16(ones, low[t][1], mfma16(ones, low[t][0], l[t]));
    }
#pragma unroll
    for (int g = 0; g < STEPS; ++g) {
      __builtin_amdgcn_sched_barrier(0);
      if (g + 1 < STEPS)
#pragma unroll
        for (int k = 0; k < 4; ++k) next[k] = value((g + 1) * 4 % DT + k, (g + 1) * 4 / DT);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          f32x4& to = o[t][g * 4 % DT + k];
          to = mfma16(now[k], p[t][g * 4 / DT], to);
          if (LOW) to = mfma16(now[k], low[t][g * 4 / DT], to);
        }
#pragma unroll
      for (int k = 0; k < 4; ++k) now[k] = next[k];
      if (g + 1 < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, 4 * CT * (LOW ? 2 : 1), 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
};

// Four outputs in their type.
__device__ __forceinline__ void store_four(bf16_t* p, f32x4 x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
}
__device__ __forceinline__ void store_four(float* p, f32x4 x) { *reinterpret_cast<f32x4*>(p) = x; }

// Writes column x of a tile: its outputs `o` over dims d0 .. + 4 N in strides of `step`,
// maximum m and sum; the call's own or a chunk's part of them.  `whole`: where the keys
// begin that not every row of the tile sees, [whole, k1) holding inf or NaN if `special`.
template <int DH, bool EIGHT, typename T, int N>
__device__ __forceinline__ void write_column(const PagedCache& c, const PagedBatch& bt, const AttendArgs& a,
                                             const Span& sp, int x, int chunk, int k0, int k1, int whole,
                                             bool special, f32x4 (&o)[N], float m, float sum, int d0,
                                             int step, bool states) {
  const int i = x / a.group;
  if (i >= sp.given) return;
  const int limit = sp.limit(i);
  const int64_t T_heads = (int64_t)bt.rows * a.heads;
  const int64_t to = (sp.row0 + i) * a.heads + sp.h * a.group + x % a.group;
  if (special)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        o[n][k] += special_sum<DH, EIGHT, T>(c, bt, sp, d0 + n * step + k, whole, min(limit, k1));
  if (limit == 0) {  // a row that sees no key is zero
    m = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (a.chunks == 1) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int n = 0; n < N; ++n) store_four((T*)a.out + to * DH + d0 + n * step, o[n] * inv);
    return;
  }
  if (limit <= k0 && chunk > 0) return;  // the join knows which chunks a row has
#pragma unroll
  for (int n = 0; n < N; ++n) store_four(a.part + (chunk * T_heads + to) * DH + d0 + n * step, o[n]);
  if (states) a.stat[chunk * T_heads + to] = make_float2(m, sum);
}

// LDS in which the waves of a workgroup, each of which went over keys of its own, are
// joined 16 columns at a time.
template <int DH> struct WaveJoin {
  float o[PAGED_WAVES][16 * (DH + 4)], m[PAGED_WAVES][16], sum[PAGED_WAVES][16];
  int special[PAGED_WAVES];

  template <bool EIGHT, typename T, int CT, int DT>
  __device__ __forceinline__ void write(const PagedCache& c, const PagedBatch& bt, const AttendArgs& a,
                                        const Span& sp, int first, int chunk, int k0, int k1, int whole,
                                        bool odd, const f32x4 (&out)[CT][DT], const float (&top)[CT],
                                        const float (&total)[CT]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    if (lane == 0) special[wave] = odd;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      __syncthreads();
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&o[wave][col * (DH + 4) + d * 16 + grp * 4]) = out[t][d];
      if (grp == 0) {
        m[wave][col] = top[t];
        sum[wave][col] = total[t];
      }
      __syncthreads();
      const int x = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (DH / 16);
      float M = m[0][x];
#pragma unroll
      for (int w = 1; w < PAGED_WAVES; ++w) M = fmaxf(M, m[w][x]);
      const float base = M == -INFINITY ? 0.f : M;
      float all = 0.f;
      f32x4 r[DH / 64] = {};
#pragma unroll
      for (int w = 0; w < PAGED_WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(m[w][x] - base);
        all = fmaf(sum[w][x], f, all);
#pragma unroll
        for (int n = 0; n < DH / 64; ++n)
          r[n] += *reinterpret_cast<const f32x4*>(&o[w][x * (DH + 4) + d0 + n * 4]) * f;
      }
      write_column<DH, EIGHT, T>(c, bt, a, sp, first + t * 16 + x, chunk, k0, k1, whole,
                                 special[0] | special[1] | special[2] | special[3], r, M, all, d0, 4,
                                 (threadIdx.x & 15) == 0);
    }
  }
};
