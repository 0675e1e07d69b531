// Attention over paged keys on the matrix cores, the keys split over the waves: bf16,
// head_dim 64 and 128, few rows a sequence (decoding steps, small windows).
//
// A decoding step reads every key and value once and does a few operations with each:
// it is bound by the bytes.  So nothing is staged: every wave takes 64-key tiles of its
// own straight from memory into the registers that the matrix instructions read, the
// next keys on their way during the products with the values and the next values during
// those with the keys, and no wave waits for another until the end.
//
// Measured: 64 sequences of 200 to 8000 tokens, one row of 32 heads over 8 each, 585 MB:
// 120 us and 5 for the join (4.7 TB/s; a large copy runs at 5.08).  One sequence of 130001
// tokens, 16 heads over 8, 266 MB: 48 and 7 us.  One of 300 tokens: 11 us, a tile of codes
// a wave and behind one of them the open page.  Pages in bf16: the 64 sequences 235 us for
// 1.07 GB (4.5 TB/s), the long one 109.  16 windows of 16 rows, 16 heads over 8, behind 300 to
// 3100 tokens: 38 us; both of a window's column tiles in one wave made it 42 (one wave a
// SIMD instead of three).  On the way: spilled registers cost 2.4 times (their
// reloads wait for the tile on its way), chunk numbers that pick the die 1.4 (eight
// chunks, eight dies, and few sequences reach the last), a scale computed where its
// exponent is loaded, or a page number checked there, 1.1 (both wait for what was loaded
// before).
#include "paged_mfma.h"

// A lane's part of one 64-key tile of codes: 16 dims of a key, 16 keys of a dimension.
template <int DH> struct CodeTile {
  uint4 k[4][DH / 64], v[DH / 16];
  int k_exponent, v_exponent;
  bool there;
};

template <int DH, bool EIGHT>
__global__ void __launch_bounds__(64 * PAGED_WAVES, 3)
paged_split_kernel(PagedCache c, PagedBatch bt, AttendArgs a) {
  constexpr int DT = DH / 16, CT = 1;  // more columns: more workgroups
  __shared__ __attribute__((aligned(16))) WaveJoin<DH> join;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  if (blockIdx.x >= gridDim.x - a.zero_blocks) {
    zero_rest(bt, (bf16_t*)a.out, (int64_t)a.heads * DH, gridDim.x - 1 - blockIdx.x, a.zero_blocks);
    return;
  }
  const int page = c.page;
  // Neighbouring workgroups go to different dies.  Heads side by side, then a sequence's
  // query tiles (eight heads on, so that they tend to meet on one die's cache), then
  // sequences, turned on by one per chunk, then chunks: every die gets long and short
  // sequences, and the chunks that few sequences reach come last.
  const int per_chunk = bt.sequences * a.query_tiles * c.kv_heads;
  const int chunk = blockIdx.x / per_chunk, rest = blockIdx.x % per_chunk;
  const int qt = rest / c.kv_heads % a.query_tiles;
  const Span sp = Span::of<EIGHT>(c, bt, (rest / (c.kv_heads * a.query_tiles) + chunk) % bt.sequences,
                                  rest % c.kv_heads);
  const int first_col = qt * 16 * CT;
  if (first_col >= sp.given * a.group) return;
  // keys that the first and the last row of the tile see
  const int row_lo = first_col / a.group, row_hi = min((first_col + 16 * CT - 1) / a.group, sp.n - 1);
  const int least = sp.limit(row_lo), most = row_hi < row_lo ? 0 : sp.limit(row_hi);
  const int k0 = chunk * a.chunk_keys, k1 = min(most, k0 + a.chunk_keys);
  if (k1 <= k0 && chunk > 0) return;
  // the lane's 16 bytes of a code row are dims (f / 2) * 64 + grp * 16 of two fragments
  Columns<DH, CT> cols;
  cols.start(a, sp, first_col, [](int f, int g) { return (f / 2) * 64 + g * 16 + (f % 2) * 8; });

  const int head_block = page * DH;
  // Places of a tile: keys of group (lane % 16) / 4, values of group lane / 16
  // (of page `id`; not followed where that is -1).
  auto key_place = [&](int base, int id) {
    const int in_page = (base + (col >> 2) * 16) & (page - 1);
    return sp.block(c, id, head_block) + ((in_page + (col & 3)) * DH + grp * 16);
  };
  auto value_place = [&](int base, int id) {
    return sp.block(c, id, head_block) + (col * page + ((base + grp * 16) & (page - 1)));
  };
  // Codes are loaded whether or not there is a page (from page 0 where there is none):
  // branches between loads would wait for the ones before.  The scores of keys that are
  // not there are hidden, their values cleared.
  auto load_key_codes = [&](CodeTile<DH>& t, int base, int id) {
    id = max(id, 0);
    const e4m3_t* p = (const e4m3_t*)c.keys + key_place(base, id);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < DH / 64; ++j) t.k[i][j] = *reinterpret_cast<const uint4*>(p + 4 * i * DH + j * 64);
    t.k_exponent = sp.exponent(c, id, 0);
  };
  auto load_value_codes = [&](CodeTile<DH>& t, int base, int id) {
    t.there = id >= 0;
    id = max(id, 0);
    const e4m3_t* p = (const e4m3_t*)c.values + value_place(base, id);
#pragma unroll
    for (int d = 0; d < DT; ++d) t.v[d] = *reinterpret_cast<const uint4*>(p + d * 16 * page);
    t.v_exponent = sp.exponent(c, id, 1);
  };
  auto clear_values = [&](CodeTile<DH>& t) {
    if (!t.there)
#pragma unroll
      for (int d = 0; d < DT; ++d) t.v[d] = make_uint4(0, 0, 0, 0);
  };
  auto scores = [&](const CodeTile<DH>& t, f32x4 (&s)[CT][4]) {
    const float scale = exp2_int(t.k_exponent);
    cols.scores(s, [&](int i, int f) {
      const uint4 w = t.k[i][f / 2];
      return f % 2 ? widen(w.z, w.w, scale) : widen(w.x, w.y, scale);
    });
  };
  auto add_values = [&](const CodeTile<DH>& t, const bf16x8 (&p)[CT][2], const bf16x8 (&low)[CT][2]) {
    const float scale = exp2_int(t.v_exponent);
    cols.template add_values<false>(p, low, [&](int d, int j) {
      const uint4 w = t.v[d];
      return j ? widen(w.z, w.w, scale) : widen(w.x, w.y, scale);
    });
  };

  constexpr int STEP = PAGED_WAVES * PAGED_TILE;
  uint32_t odd = 0;  // inf or NaN among the values of a tile that not every row sees whole
  // tiles keep the waves' turns
  auto first_tile = [&](int from) {
    return from + ((wave - from / PAGED_TILE) & (PAGED_WAVES - 1)) * PAGED_TILE;
  };
  // Whole tiles of codes [k0, to), which every row sees: the next tile's keys are on
  // their way while this one's values are used, and its values while those keys are.
  auto whole_code_tiles = [&](int to) {
    int base = first_tile(k0);
    if (base >= to) return;
    CodeTile<DH> tile;
    load_key_codes(tile, base, sp.page<true>(c, bt, base + (col >> 2) * 16, 0, to));
    load_value_codes(tile, base, sp.page<true>(c, bt, base + grp * 16, 0, to));
    int k_next = sp.entry(c, bt, base + STEP + (col >> 2) * 16);
    int v_next = sp.entry(c, bt, base + STEP + grp * 16);
    while (true) {
      const bool more = base + STEP < to;
      f32x4 s[CT][4];
      bf16x8 p[CT][2], low[CT][2];
      scores(tile, s);
      if (more) load_key_codes(tile, base + STEP, sp.page_in(c, k_next, base + STEP, 0, to));
      if (!__all(tile.there)) {
        cols.hide(s, base, 0, to, tile.there);
        clear_values(tile);
      }
      cols.template softmax<true>(s, p, low, a.scale2);
      add_values(tile, p, low);
      if (!more) break;
      base += STEP;
      load_value_codes(tile, base, sp.page_in(c, v_next, base, 0, to));
      k_next = sp.entry(c, bt, base + STEP + (col >> 2) * 16);
      v_next = sp.entry(c, bt, base + STEP + grp * 16);
    }
  };
  // Tiles [from, to) of codes that some row does not see whole.
  auto edge_code_tiles = [&](int from, int to) {
    for (int base = first_tile(from); base < to; base += STEP) {
      CodeTile<DH> tile;
      load_key_codes(tile, base, sp.page<true>(c, bt, base + (col >> 2) * 16, k0, to));
      load_value_codes(tile, base, sp.page<true>(c, bt, base + grp * 16, k0, to));
      f32x4 s[CT][4];
      bf16x8 p[CT][2], low[CT][2];
      scores(tile, s);
      cols.hide(s, base, k0, to, tile.there);
      clear_values(tile);
      cols.template softmax<true>(s, p, low, a.scale2);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        uint32_t* w = &tile.v[d].x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          odd |= special_bits<true>(w[i]);
          w[i] = without_special<true>(w[i]);
        }
      }
      add_values(tile, p, low);
    }
  };
  // Tiles [from, to) of keys [lo, to) in 16 bits, loaded as the products take them
  // (keys and values of a tile at once do not fit the registers of three waves a SIMD).
  auto plain_tiles = [&](int from, int to, int lo, auto whole, auto pool) {
    constexpr bool WHOLE = decltype(whole)::value, POOL = decltype(pool)::value;
    const bf16_t* keys = (const bf16_t*)(POOL ? c.keys : c.open_keys);
    const bf16_t* values = (const bf16_t*)(POOL ? c.values : c.open_values);
    for (int base = first_tile(from); base < to; base += STEP) {
      const int k_page = sp.page<POOL>(c, bt, base + (col >> 2) * 16, lo, to);
      const int v_page = sp.page<POOL>(c, bt, base + grp * 16, lo, to);
      const bf16_t* kp = keys + key_place(base, max(k_page, 0));
      const bf16_t* vp = values + value_place(base, max(v_page, 0));
      f32x4 s[CT][4];
      bf16x8 p[CT][2], low[CT][2];
      cols.scores(s, [&](int i, int f) {
        return *reinterpret_cast<const bf16x8*>(kp + 4 * i * DH + (f / 2) * 64 + (f % 2) * 8);
      });
      if (!WHOLE || !__all(v_page >= 0)) cols.hide(s, base, lo, to, v_page >= 0);
      cols.template softmax<true>(s, p, low, a.scale2);
      cols.template add_values<WHOLE>(p, low, [&](int d, int j) {
        uint4 w = *reinterpret_cast<const uint4*>(vp + d * 16 * page + j * 8);
        if (v_page < 0) w = make_uint4(0, 0, 0, 0);
        if (!WHOLE) {
          odd |= special_bits<false>(w.x) | special_bits<false>(w.y) | special_bits<false>(w.z) |
                 special_bits<false>(w.w);
          w = make_uint4(without_special<false>(w.x), without_special<false>(w.y),
                         without_special<false>(w.z), without_special<false>(w.w));
        }
        return __builtin_bit_cast(bf16x8, w);
      });
    }
  };
  const int hi = EIGHT ? min(k1, sp.sealed) : k1;
  const int whole = max(min(hi, least) / PAGED_TILE * PAGED_TILE, k0);
  if constexpr (EIGHT) {  // the sealed pages, then the open ones
    whole_code_tiles(whole);
    edge_code_tiles(whole, hi);
    const int lo = max(k0, sp.sealed);
    if (lo < k1) plain_tiles(lo / PAGED_TILE * PAGED_TILE, k1, lo, std::false_type(), std::false_type());
  } else {
    plain_tiles(k0, whole, k0, std::true_type(), std::true_type());
    plain_tiles(whole, hi, k0, std::false_type(), std::true_type());
  }

  float sum[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) sum[t] = cols.l[t][0];
  join.template write<EIGHT, bf16_t>(c, bt, a, sp, first_col, chunk, k0, k1, whole, __any(odd), cols.o, cols.m, sum);
}

template <int DH>
static void launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, const AttendArgs& a,
                   unsigned grid, hipStream_t st) {
  if (c->eight_bit)
    paged_split_kernel<DH, true><<<grid, 64 * PAGED_WAVES, 0, st>>>(paged_cache(c), paged_batch(b), a);
  else
    paged_split_kernel<DH, false><<<grid, 64 * PAGED_WAVES, 0, st>>>(paged_cache(c), paged_batch(b), a);
}

void paged_split_launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, const AttendArgs& a,
                        const AttendPlan&, unsigned grid, hipStream_t st) {
  if (c->head_dim == 64) launch<64>(c, b, a, grid, st);
  else launch<128>(c, b, a, grid, st);
}
