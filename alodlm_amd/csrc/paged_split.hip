// Attention over paged keys on the matrix cores, the keys split over the waves: bf16,
// head_dim 64 and 128, few rows a sequence (decoding steps and windows).
//
// A decoding step reads every key and value once and does a few operations with each:
// it is bound by the bytes.  So nothing is staged: every wave takes 64-key tiles of its
// own straight from memory into the registers that the matrix instructions read, the
// next keys on their way during the products with the values and the next values during
// those with the keys, and no wave waits for another until the end.
//
// Transposed products keep the probabilities in registers: S^T = K Q^T and O^T = V^T
// P^T on 16x16x32 tiles.  The lane that holds query column c = lane % 16 of S^T holds the
// same column of P^T, and the order in which keys are given to the rows of S^T is
// chosen so that a lane's 16 scores are 16 keys in a row, lane / 16 saying which 16 of
// the 64:  row r of subtile t is key (r / 4) * 16 + 4 t + r % 4.  That is the order of
// the 16 bytes that the lane loads of a value row (tokens are contiguous there), and
// since page sizes are multiples of 16, each lane's 16 keys lie in one page.
//
// 8-bit codes become bf16 times the page's power of two in one instruction a pair
// (v_cvt_scalef32_pk_bf16_fp8), exactly.  Scores, maxima, sums and outputs are float32;
// the probabilities are rounded to bf16 for the second product, and the sum is that of
// the rounded ones (one more product with ones), so that the weights add up to one.
#include "paged.h"

#include <type_traits>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

#define SPLIT_WAVES 4
#define SPLIT_TILE 64

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

// A lane's part of one 64-key tile.  8 bits: k[t][c] 16 dims of a key, v[d] 16 keys of a
// dimension; 16 bits: the same in twice the registers.
template <int DH, bool EIGHT> struct KeyTile {
  static constexpr bool E = EIGHT;
  static constexpr int N = DH / (EIGHT ? 64 : 32);
  uint4 w[4][N];
  float scale;
};
template <int DH, bool EIGHT> struct ValueTile {
  static constexpr bool E = EIGHT;
  static constexpr int N = EIGHT ? 1 : 2;
  uint4 w[DH / 16][N];
  float scale;
  bool ok;
};

template <int DH, int CT, bool EIGHT>
__global__ void __launch_bounds__(64 * SPLIT_WAVES, CT == 1 ? 2 : 1)
paged_split_kernel(PagedCache c, PagedBatch bt, AttendArgs a) {
  constexpr int FR = DH / 32, DT = DH / 16;  // query fragments, output row tiles
  __shared__ __attribute__((aligned(16))) float buf[SPLIT_WAVES][16 * (DH + 4)];
  __shared__ float m_of[SPLIT_WAVES][16], l_of[SPLIT_WAVES][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  if (blockIdx.x >= gridDim.x - a.zero_blocks) {
    zero_rest(bt, (bf16_t*)a.out, (int64_t)a.heads * DH, gridDim.x - 1 - blockIdx.x, a.zero_blocks);
    return;
  }
  const int page = c.page, shift = 31 - __builtin_clz(page);
  // Neighbouring workgroups go to different dies.  Heads side by side, then sequences,
  // turned on by one per chunk, then chunks: every die gets long and short sequences, and
  // the chunks that few sequences reach come last.  Query tiles lie a multiple of all
  // that apart, so that they tend to meet on one die's cache.
  const int per_chunk = bt.sequences * c.kv_heads, per_tile = per_chunk * a.chunks;
  const int qt = blockIdx.x / per_tile, rest = blockIdx.x % per_tile;
  const int chunk = rest / per_chunk, h = rest % c.kv_heads;
  const int b = (rest % per_chunk / c.kv_heads + chunk) % bt.sequences;
  const int given = given_rows(bt, b), first_col = qt * 16 * CT;
  if (first_col >= given * a.group) return;
  const int held = bt.held(b, page);
  const int n = held < 0 ? 0 : bt.row_count(b, held, page);
  const int end = max(held, 0) + n, sealed = EIGHT ? sealed_keys(bt, max(held, 0), end, page, true) : 0;
  const int reach = EIGHT ? open_end(c, sealed, end) : end;  // keys that are there
  const int slot = EIGHT ? bt.slot(b, c.slots) : 0;
  const int64_t row0 = bt.first_row(b);
  // keys that the first and the last row of the tile see
  const int row_lo = first_col / a.group, row_hi = min((first_col + 16 * CT - 1) / a.group, n - 1);
  const int most = row_hi < row_lo ? 0 : min(held + row_hi + 1, reach);
  const int least = row_hi < row_lo ? 0 : min(held + row_lo + 1, reach);
  const int k0 = chunk * a.chunk_keys, k1 = min(most, k0 + a.chunk_keys);
  if (k1 <= k0 && chunk > 0) return;
  // this lane's columns: row first_col + ..., limit on its keys
  int limit[CT];
  bf16x8 q[CT][FR];
  int64_t at[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const int x = first_col + t * 16 + col, i = x / a.group, head = h * a.group + x % a.group;
    limit[t] = i < n ? min(held + i + 1, reach) : 0;
    at[t] = i < given ? (row0 + i) * a.heads + head : -1;
    const bf16_t* p = (const bf16_t*)a.q + (row0 + i) * a.ldq + (int64_t)head * DH + grp * 16;
#pragma unroll
    for (int f = 0; f < FR; ++f) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (i < n) w = *reinterpret_cast<const uint4*>(p + (f / 2) * 64 + (f % 2) * 8);
      q[t][f] = __builtin_bit_cast(bf16x8, w);
    }
  }
  f32x4 o[CT][DT], l[CT];
  float m[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    m[t] = -INFINITY;
    l[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  bf16x8 ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.f;

  const int64_t head_block = (int64_t)page * DH;
  // The page (of the pool, or open) of the 16 keys from `key` on, in blocks of one head.
  auto find = [&](int key, int lo, int hi, auto eight) -> int64_t {
    if (key + 15 < lo || key >= hi) return -1;
    const int p = key >> shift;
    if (EIGHT && !decltype(eight)::value)
      return slot < 0 ? -1 : open_page(c, slot, p) * c.kv_heads + h;
    const int64_t id = bt.page_of(b, p, c.pages);
    return id < 0 ? -1 : id * c.kv_heads + h;
  };
  // The keys: group (lane % 16) / 4 of the tile; a block of -1 gives zeros.
  auto load_keys = [&](auto& t, int base, int64_t block) {
    constexpr bool E = std::decay_t<decltype(t)>::E;
    typedef typename std::conditional<E, e4m3_t, bf16_t>::type S;
    t.scale = 1.f;
    const S* keys = (const S*)(EIGHT && !E ? c.open_keys : c.keys);
    const int in_page = (base + (col >> 2) * 16) & (page - 1);
    const S* p = keys + block * head_block + (int64_t)(in_page + (col & 3)) * DH + grp * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < KeyTile<DH, E>::N; ++j) {
        t.w[i][j] = make_uint4(0, 0, 0, 0);
        if (block >= 0)
          t.w[i][j] = *reinterpret_cast<const uint4*>(p + 4 * i * DH + (E ? j * 64 : (j / 2) * 64 + (j % 2) * 8));
      }
    if (E && block >= 0) t.scale = exp2_int(c.exponents[block / c.kv_heads * 2 * c.kv_heads + h]);
  };
  // The values: group lane / 16.
  auto load_values = [&](auto& t, int base, int64_t block) {
    constexpr bool E = std::decay_t<decltype(t)>::E;
    typedef typename std::conditional<E, e4m3_t, bf16_t>::type S;
    t.scale = 1.f;
    t.ok = block >= 0;
    const S* values = (const S*)(EIGHT && !E ? c.open_values : c.values);
    const int in_page = (base + grp * 16) & (page - 1);
    const S* p = values + block * head_block + (int64_t)col * page + in_page;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int j = 0; j < ValueTile<DH, E>::N; ++j) {
        t.w[d][j] = make_uint4(0, 0, 0, 0);
        if (block >= 0) t.w[d][j] = *reinterpret_cast<const uint4*>(p + d * 16 * page + j * 8);
      }
    if (E && block >= 0) t.scale = exp2_int(c.exponents[(block / c.kv_heads * 2 + 1) * c.kv_heads + h]);
  };
  // p * v of the values that are inf or NaN, one by one, for the rows that see them: in
  // the products they are zeros, since 0 times one of them would not be 0 for the rows
  // that do not.
  auto add_special = [&](int base, const bf16x8 (&p)[CT][2], int lo, int hi, auto eight) {
    constexpr bool E = decltype(eight)::value;
    float* mine = buf[wave];
    for (int t = 0; t < CT; ++t) {
      __builtin_amdgcn_wave_barrier();
      int lim = 0;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
        if (ct == t) {
          lim = limit[ct];
#pragma unroll
          for (int i = 0; i < 16; ++i) mine[(grp * 16 + i) * 16 + col] = (float)p[ct][i / 8][i % 8];
        }
      __builtin_amdgcn_wave_barrier();
      for (int k = 0; k < SPLIT_TILE; ++k) {
        const int key = base + k;
        if (key < lo || key >= hi) continue;
        const int64_t pl = find(key & ~15, lo, hi, eight);
        if (pl < 0) continue;
        const float w = mine[k * 16 + col];
        const int64_t v_at = pl * head_block + (key & (page - 1));
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t x = v_at + (int64_t)(d * 16 + grp * 4 + i) * page;
            const float v = E ? __builtin_amdgcn_cvt_f32_fp8(((const e4m3_t*)c.values)[x], 0)
                              : bf16_to_float(((const bf16_t*)(EIGHT ? c.open_values : c.values))[x]);
            if (key < lim && !(fabsf(v) < INFINITY)) {
#pragma unroll
              for (int ct = 0; ct < CT; ++ct)
                if (ct == t) o[ct][d][i] = fmaf(w, v, o[ct][d][i]);
            }
          }
      }
    }
  };
  auto scores = [&](const auto& keys, f32x4 (&s)[CT][4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int t = 0; t < CT; ++t) s[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < FR; ++f) {
        bf16x8 k;
        if constexpr (std::decay_t<decltype(keys)>::E) {
          const uint4 w = keys.w[i][f / 2];
          k = f % 2 ? widen(w.z, w.w, keys.scale) : widen(w.x, w.y, keys.scale);
        } else {
          k = __builtin_bit_cast(bf16x8, keys.w[i][f]);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) s[t][i] = mfma16(k, q[t][f], s[t][i]);
      }
    }
  };
  // Scores -> probabilities in bf16; the maximum and what goes with it move along.
  auto softmax = [&](const f32x4 (&s)[CT][4], bf16x8 (&p)[CT][2]) {
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      float top = s[t][0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[t][i / 4][i % 4]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64)) * a.scale2;
      if (__any(top > m[t])) {
        const float to = fmaxf(m[t], top);
        const float f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[t] - to);
        m[t] = to;
        l[t] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] *= f;
      }
      const float base_m = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        p[t][i / 8][i % 8] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[t][i / 4][i % 4], a.scale2, -base_m));
    }
  };
  auto add_values = [&](const auto& values, const bf16x8 (&p)[CT][2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int t = 0; t < CT; ++t) l[t] = mfma16(ones, p[t][j], l[t]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        bf16x8 v;
        if constexpr (std::decay_t<decltype(values)>::E) {
          const uint4 w = values.w[d][0];
          v = j ? widen(w.z, w.w, values.scale) : widen(w.x, w.y, values.scale);
        } else {
          v = __builtin_bit_cast(bf16x8, values.w[d][j]);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) o[t][d] = mfma16(v, p[t][j], o[t][d]);
      }
    }
  };
  // Keys outside [lo, hi), beyond a row's own, or in a page that is missing are hidden.
  auto hide = [&](f32x4 (&s)[CT][4], int base, int lo, int hi, bool there) {
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = base + grp * 16 + i;
        if (!(key >= lo && key < min(hi, limit[t]) && there)) s[t][i / 4][i % 4] = -INFINITY;
      }
  };
  // inf and NaN among a tile's values -> zero; whether there was any.
  auto clean = [&](auto& tile) -> bool {
    constexpr bool E = std::decay_t<decltype(tile)>::E;
    uint32_t odd = 0;
    auto word = [&](uint32_t& w, bool write) {  // bytes (halves) with all ones for an exponent
      const uint32_t z = E ? ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u
                           : ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
      odd |= z;
      if (write) w &= E ? ~((z >> 7) * 0xffu) : ~((z >> 15) * 0xffffu);
    };
    auto sweep = [&](bool write) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < ValueTile<DH, E>::N; ++j) {
          word(tile.w[d][j].x, write);
          word(tile.w[d][j].y, write);
          word(tile.w[d][j].z, write);
          word(tile.w[d][j].w, write);
        }
    };
    sweep(false);
    if (!__any(odd)) return false;
    sweep(true);
    return true;
  };

  constexpr int STEP = SPLIT_WAVES * SPLIT_TILE;
  // Tiles [from, to) of keys [lo, hi) that some row does not see whole.
  auto edge_tiles = [&](int from, int to, int lo, int hi, auto eight) {
    constexpr bool E = decltype(eight)::value;
    for (int base = from + ((wave - from / SPLIT_TILE) & (SPLIT_WAVES - 1)) * SPLIT_TILE; base < to;
         base += STEP) {
      KeyTile<DH, E> keys;
      ValueTile<DH, E> values;
      load_keys(keys, base, find(base + (col >> 2) * 16, lo, hi, eight));
      load_values(values, base, find(base + grp * 16, lo, hi, eight));
      f32x4 s[CT][4];
      bf16x8 p[CT][2];
      scores(keys, s);
      hide(s, base, lo, hi, values.ok);
      softmax(s, p);
      const bool special = clean(values);
      add_values(values, p);
      if (special) add_special(base, p, lo, hi, eight);
    }
  };
  // Whole tiles of keys [k0, to) that every row sees: the next tile's keys are on their
  // way while this one's values are used, and its values while those keys are.
  auto whole_tiles = [&](int to, auto eight) {
    constexpr bool E = decltype(eight)::value;
    int base = k0 + ((wave - k0 / SPLIT_TILE) & (SPLIT_WAVES - 1)) * SPLIT_TILE;
    if (base >= to) return;
    KeyTile<DH, E> keys;
    ValueTile<DH, E> values;
    load_keys(keys, base, find(base + (col >> 2) * 16, 0, to, eight));
    load_values(values, base, find(base + grp * 16, 0, to, eight));
    int64_t k_next = find(base + STEP + (col >> 2) * 16, 0, to, eight);
    int64_t v_next = find(base + STEP + grp * 16, 0, to, eight);
    while (true) {
      const bool more = base + STEP < to;
      f32x4 s[CT][4];
      bf16x8 p[CT][2];
      scores(keys, s);
      if (more) load_keys(keys, base + STEP, k_next);
      if (!__all(values.ok)) hide(s, base, 0, to, values.ok);
      softmax(s, p);
      add_values(values, p);
      if (!more) break;
      base += STEP;
      load_values(values, base, v_next);
      k_next = find(base + STEP + (col >> 2) * 16, 0, to, eight);
      v_next = find(base + STEP + grp * 16, 0, to, eight);
    }
  };
  // 8 bits: the sealed pages, then the open ones; 16 bits: the pool's
  const int hi = EIGHT ? min(k1, sealed) : k1;
  const int whole = max(min(hi, least) / SPLIT_TILE * SPLIT_TILE, k0);
  typedef std::integral_constant<bool, EIGHT> Pool;
  whole_tiles(whole, Pool());
  edge_tiles(whole, hi, k0, hi, Pool());
  if constexpr (EIGHT) {
    const int lo = max(k0, sealed);
    if (lo < k1) edge_tiles(lo / SPLIT_TILE * SPLIT_TILE, k1, lo, k1, std::false_type());
  }

  // join the waves, 16 columns at a time
  const int64_t T_heads = (int64_t)bt.rows * a.heads;
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<f32x4*>(&buf[wave][col * (DH + 4) + d * 16 + grp * 4]) = o[t][d];
    if (grp == 0) { m_of[wave][col] = m[t]; l_of[wave][col] = l[t][0]; }
    __syncthreads();
    const int x = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (DH / 16);
    float M = m_of[0][x];
#pragma unroll
    for (int w = 1; w < SPLIT_WAVES; ++w) M = fmaxf(M, m_of[w][x]);
    const float base_m = M == -INFINITY ? 0.f : M;
    float sum = 0.f, r[DH / 16] = {};
#pragma unroll
    for (int w = 0; w < SPLIT_WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(m_of[w][x] - base_m);
      sum = fmaf(l_of[w][x], f, sum);
#pragma unroll
      for (int i = 0; i < DH / 16; ++i) r[i] = fmaf(buf[w][x * (DH + 4) + d0 + i], f, r[i]);
    }
    const int y = first_col + t * 16 + x, i = y / a.group;
    if (i >= given) continue;
    const int64_t to = (row0 + i) * a.heads + h * a.group + y % a.group;
    if (a.chunks == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees no key is zero
      bf16_t* out = (bf16_t*)a.out + to * DH + d0;
#pragma unroll
      for (int k = 0; k < DH / 16; k += 4)
        *reinterpret_cast<uint2*>(out + k) = make_uint2(pack_bf16x2(r[k] * inv, r[k + 1] * inv),
                                                        pack_bf16x2(r[k + 2] * inv, r[k + 3] * inv));
      continue;
    }
    const int lim = i < n ? min(held + i + 1, reach) : 0;
    if (lim <= k0 && chunk > 0) continue;  // the join knows which chunks a row has
    float* part = a.part + (chunk * T_heads + to) * DH + d0;
#pragma unroll
    for (int k = 0; k < DH / 16; k += 4)
      *reinterpret_cast<f32x4*>(part + k) = f32x4{r[k], r[k + 1], r[k + 2], r[k + 3]};
    if ((threadIdx.x & 15) == 0) a.stat[chunk * T_heads + to] = make_float2(M, sum);
  }
}

bool paged_split_takes(const alodlm_paged_cache* c) {
  return c->dtype == ALODLM_BF16 && (c->head_dim == 64 || c->head_dim == 128);
}

template <int DH, int CT>
static void launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, const AttendArgs& a,
                   unsigned grid, hipStream_t st) {
  if (c->eight_bit)
    paged_split_kernel<DH, CT, true><<<grid, 64 * SPLIT_WAVES, 0, st>>>(paged_cache(c), paged_batch(b), a);
  else
    paged_split_kernel<DH, CT, false><<<grid, 64 * SPLIT_WAVES, 0, st>>>(paged_cache(c), paged_batch(b), a);
}

void paged_split_launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, const AttendArgs& a,
                        const AttendPlan& p, unsigned grid, hipStream_t st) {
  if (c->head_dim == 64) {
    if (p.column_tiles == 1) launch<64, 1>(c, b, a, grid, st);
    else launch<64, 2>(c, b, a, grid, st);
  } else {
    if (p.column_tiles == 1) launch<128, 1>(c, b, a, grid, st);
    else launch<128, 2>(c, b, a, grid, st);
  }
}
