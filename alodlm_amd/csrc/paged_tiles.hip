// Attention over paged keys on the matrix cores, the query rows split over the waves:
// bf16, head_dim 64 and 128, windows and prompts.
//
// A workgroup's four waves hold 64 CT query columns (rows times the heads that share a
// key/value head) against the same keys.  Each 64-key tile is fetched once, widened to
// bf16 once and laid into LDS, from where every wave takes its fragments; the next
// tile's bytes come in behind the products of the one before, into the other half of
// the buffer: one barrier a tile.  The limits are then the matrix instructions, the
// LDS reads (32 KB a wave and tile against 32 columns) and the exponentials, which
// two workgroups a compute unit overlap.
//
// Measured: four prompts of 700 to 4100 rows, 16 heads over 8 of 128: 178 to 208 us (the
// clock goes with the card), 675 to 790 TFLOP/s of 1198 for a large library product;
// matrix instructions busy 33 % of the cycles, vector instructions 48 %, LDS 27 %.  16
// windows of 16 to 27 rows behind 300 to 3100 tokens, 32 heads over 8: 39 us and 8 for the
// join, the time of a tile's instructions one after the other (2.7 us, in a cache or not)
// with too few workgroups to fill the gaps.  On the way: integer divisions per tile cost 10 %,
// page numbers checked and scales computed where they are loaded 18 %, outputs rescaled
// at every new maximum 7 %, LDS reads left behind the products before them 4 %; bank
// conflicts (27 % of the LDS cycles, none now) cost no time.
#include "paged_mfma.h"

template <int DH> struct TileBuffer {
  bf16_t k[PAGED_TILE * DH];
  bf16_t v[DH * PAGED_TILE];
};

// Places (in values) of 16-byte pieces.  A fragment's lanes read 16 rows of 4 pieces that
// lie together: keys in the order of a subtile's rows, 32 dims a block; dimensions, 8 of
// every group's 16 keys a block.  Within a row the pieces are XORed with the row (reads)
// and the block (writes of one key's blocks) so that no 16 lanes meet in a bank.
template <int DH>
__device__ __forceinline__ int key_piece(int key, int piece) {
  const int f = piece >> 2, r = ((key >> 2) & 3) * 16 + (key >> 4) * 4 + (key & 3);
  return (f * PAGED_TILE + r) * 32 + (((piece ^ (r >> 1) ^ f) & 3) << 3);
}
template <int DH>
__device__ __forceinline__ int value_piece(int d, int group, int j) {
  return (j * DH + d) * 32 + (((group ^ (d >> 1)) & 3) << 3);
}

template <int DH, int CT, bool EIGHT>
__global__ void __launch_bounds__(64 * PAGED_WAVES, 2)
paged_tiles_kernel(PagedCache c, PagedBatch bt, AttendArgs a) {
  constexpr int DT = DH / 16, COLS = 16 * CT * PAGED_WAVES;
  constexpr bool LOW = CT == 1;
  __shared__ __attribute__((aligned(16))) TileBuffer<DH> tiles[2];
  __shared__ int there[2][4], special_of[PAGED_WAVES], low_special[2][PAGED_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  if (blockIdx.x >= gridDim.x - a.zero_blocks) {
    zero_rest(bt, (bf16_t*)a.out, (int64_t)a.heads * DH, gridDim.x - 1 - blockIdx.x, a.zero_blocks);
    return;
  }
  const int page = c.page;
  // heads, sequences (turned on by one per chunk and query tile), chunks, query tiles,
  // the last of which see the most keys and go first
  const int per_chunk = bt.sequences * c.kv_heads, per_tile = per_chunk * a.chunks;
  const int qt = a.query_tiles - 1 - blockIdx.x / per_tile, rest = blockIdx.x % per_tile;
  const int chunk = rest / per_chunk;
  const Span sp = Span::of<EIGHT>(c, bt, (rest % per_chunk / c.kv_heads + chunk + qt) % bt.sequences,
                                  rest % c.kv_heads);
  const int first_col = qt * COLS;
  if (first_col >= sp.given * a.group) return;
  const int row_lo = first_col / a.group, row_hi = min((first_col + COLS - 1) / a.group, sp.n - 1);
  const int least = sp.limit(row_lo), most = row_hi < row_lo ? 0 : sp.limit(row_hi);
  const int k0 = chunk * a.chunk_keys, k1 = min(most, k0 + a.chunk_keys);
  if (k1 <= k0 && chunk > 0) return;
  // this wave's columns
  const int my_col = first_col + wave * 16 * CT;
  const int my_lo = my_col / a.group, my_hi = min((my_col + 16 * CT - 1) / a.group, sp.n - 1);
  const int my_least = sp.limit(my_lo), my_most = my_hi < my_lo ? 0 : sp.limit(my_hi);
  Columns<DH, CT> cols;
  cols.start(a, sp, my_col, [](int f, int g) { return f * 32 + g * 8; });

  // Tiles in order: the sealed pages' (or all of a 16-bit pool's), then the open pages'.
  const int hi = EIGHT ? min(k1, sp.sealed) : k1;
  const int lo_open = EIGHT ? max(k0, sp.sealed) : k1, start_open = lo_open / PAGED_TILE * PAGED_TILE;
  const int pool_tiles = hi > k0 ? (hi - k0 + PAGED_TILE - 1) / PAGED_TILE : 0;
  const int count = pool_tiles + (k1 > lo_open ? (k1 - start_open + PAGED_TILE - 1) / PAGED_TILE : 0);
  auto base_of = [&](int i) {
    return i < pool_tiles ? k0 + i * PAGED_TILE : start_open + (i - pool_tiles) * PAGED_TILE;
  };

  // A thread's part of a tile.  Keys: key tid / 4, a quarter of its row.  Values:
  // dimensions tid / 4 + 64 r, 16 keys (group tid % 4).
  constexpr int KW = DH / 64, KW16 = DH / 32, VR = DH / 64;  // 16-byte words of codes, of bf16
  const int head_block = page * DH, t_key = tid >> 2, t_part = tid & 3, t_dim = tid >> 2;
  struct Pages {
    int k, v;
  };
  auto entries_of = [&](int i) {
    const int base = base_of(min(i, max(pool_tiles - 1, 0)));
    return Pages{sp.entry(c, bt, base + (t_key & ~15)), sp.entry(c, bt, base + t_part * 16)};
  };
  // the thread's first value in its pages
  auto key_at = [&](int i, int id) {
    return sp.block(c, id, head_block) + (((base_of(i) + t_key) & (page - 1)) * DH + t_part * (DH / 4));
  };
  auto value_at = [&](int i, int id) {
    return sp.block(c, id, head_block) + (t_dim * page + ((base_of(i) + t_part * 16) & (page - 1)));
  };
  // What comes in behind the products: codes, or the keys of a 16-bit pool (its values
  // as well would not fit the registers of two waves a SIMD).  `next` runs a tile ahead
  // of that, so that nothing waits for the table.
  uint4 raw_k[EIGHT ? KW : KW16], raw_v[VR];
  int k_exponent = 0, v_exponent = 0;
  Pages ahead, next;
  auto fetch = [&](int i) {
    const int k_at = base_of(i) + (t_key & ~15), v_at = base_of(i) + t_part * 16;
    if (EIGHT && i >= pool_tiles) {
      ahead = Pages{sp.page<false>(c, bt, k_at, lo_open, k1), sp.page<false>(c, bt, v_at, lo_open, k1)};
      return;
    }
    ahead = Pages{sp.page_in(c, next.k, k_at, k0, hi), sp.page_in(c, next.v, v_at, k0, hi)};
    next = entries_of(i + 1);
    // from page 0 where there is none: branches between loads would wait for the ones before
    const int64_t kp = key_at(i, max(ahead.k, 0)), vp = value_at(i, max(ahead.v, 0));
#pragma unroll
    for (int j = 0; j < (EIGHT ? KW : KW16); ++j) {
      raw_k[j] = EIGHT ? *reinterpret_cast<const uint4*>((const e4m3_t*)c.keys + kp + j * 16)
                       : *reinterpret_cast<const uint4*>((const bf16_t*)c.keys + kp + j * 8);
    }
    if constexpr (EIGHT) {
#pragma unroll
      for (int r = 0; r < VR; ++r)
        raw_v[r] = *reinterpret_cast<const uint4*>((const e4m3_t*)c.values + vp + r * 64 * page);
      k_exponent = sp.exponent(c, max(ahead.k, 0), 0);
      v_exponent = sp.exponent(c, max(ahead.v, 0), 1);
    }
  };
  // Tile i -> bf16 in LDS.  In tiles that some row does not see whole, values that are
  // inf or NaN become zeros.
  uint32_t odd = 0;
  auto stage_codes = [&](int i) {
    TileBuffer<DH>& t = tiles[i & 1];
    const bool edge = base_of(i) + PAGED_TILE > min(hi, least);
    const float k_scale = exp2_int(k_exponent), v_scale = exp2_int(v_exponent);
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const uint4 w = raw_k[j];
      const int piece = t_part * (DH / 32) + 2 * j;
      *reinterpret_cast<bf16x8*>(t.k + key_piece<DH>(t_key, piece)) = widen(w.x, w.y, k_scale);
      *reinterpret_cast<bf16x8*>(t.k + key_piece<DH>(t_key, piece + 1)) = widen(w.z, w.w, k_scale);
    }
#pragma unroll
    for (int r = 0; r < VR; ++r) {
      uint4 w = raw_v[r];
      if (ahead.v < 0) w = make_uint4(0, 0, 0, 0);
      if (edge) {
        odd |= special_bits<true>(w.x) | special_bits<true>(w.y) | special_bits<true>(w.z) | special_bits<true>(w.w);
        w = make_uint4(without_special<true>(w.x), without_special<true>(w.y), without_special<true>(w.z),
                       without_special<true>(w.w));
      }
      *reinterpret_cast<bf16x8*>(t.v + value_piece<DH>(t_dim + 64 * r, t_part, 0)) = widen(w.x, w.y, v_scale);
      *reinterpret_cast<bf16x8*>(t.v + value_piece<DH>(t_dim + 64 * r, t_part, 1)) = widen(w.z, w.w, v_scale);
    }
    if (tid < 4) there[i & 1][tid] = ahead.v >= 0;  // thread t holds group t
  };
  auto stage_plain = [&](int i) {
    TileBuffer<DH>& t = tiles[i & 1];
    const bool pool = i < pool_tiles, edge = !pool || base_of(i) + PAGED_TILE > min(hi, least);
    const int64_t kp = key_at(i, max(ahead.k, 0)), vp = value_at(i, max(ahead.v, 0));
    const bf16_t* values = (const bf16_t*)(EIGHT ? c.open_values : c.values);
    uint32_t seen = 0;  // inf or NaN that stays
    uint4 wv[VR][2];
#pragma unroll
    for (int r = 0; r < VR; ++r)
#pragma unroll
      for (int j = 0; j < 2; ++j) wv[r][j] = *reinterpret_cast<const uint4*>(values + vp + r * 64 * page + j * 8);
#pragma unroll
    for (int j = 0; j < KW16; ++j) {
      uint4 w;
      if constexpr (!EIGHT) w = raw_k[j];
      else w = *reinterpret_cast<const uint4*>((const bf16_t*)c.open_keys + kp + j * 8);
      *reinterpret_cast<uint4*>(t.k + key_piece<DH>(t_key, t_part * (DH / 32) + j)) = w;
    }
#pragma unroll
    for (int r = 0; r < VR; ++r)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint4 w = wv[r][j];
        if (ahead.v < 0) w = make_uint4(0, 0, 0, 0);
        if (edge) {
          odd |= special_bits<false>(w.x) | special_bits<false>(w.y) | special_bits<false>(w.z) | special_bits<false>(w.w);
          w = make_uint4(without_special<false>(w.x), without_special<false>(w.y), without_special<false>(w.z),
                         without_special<false>(w.w));
        } else if (LOW) {
          seen |= special_bits<false>(w.x) | special_bits<false>(w.y) | special_bits<false>(w.z) | special_bits<false>(w.w);
        }
        *reinterpret_cast<uint4*>(t.v + value_piece<DH>(t_dim + 64 * r, t_part, j)) = w;
      }
    if (tid < 4) there[i & 1][tid] = ahead.v >= 0;
    if (LOW && !EIGHT) {
      const bool any = __any(seen);
      if (lane == 0) low_special[i & 1][wave] = any;
    }
  };
  auto stage = [&](int i) {
    if (EIGHT && i < pool_tiles) stage_codes(i);
    else stage_plain(i);
  };

  if (count > 0) {
    next = entries_of(0);
    fetch(0);
    stage(0);
  }
  __syncthreads();
  for (int i = 0; i < count; ++i) {
    const bool more = i + 1 < count;
    if (more) fetch(i + 1);
    const int base = base_of(i);
    const bool pool = i < pool_tiles;
    const int lo = pool ? k0 : lo_open, end = pool ? hi : k1;
    if (base < my_most) {
      const TileBuffer<DH>& t = tiles[i & 1];
      f32x4 s[CT][4];
      bf16x8 p[CT][2], low[CT][2];
      cols.scores_ahead(s, [&](int sub, int f) {
        const int key = (col >> 2) * 16 + 4 * sub + (col & 3);
        return *reinterpret_cast<const bf16x8*>(t.k + key_piece<DH>(key, f * 4 + grp));
      });
      const bool mine = there[i & 1][grp];
      if (base < lo || base + PAGED_TILE > min(end, my_least) || !__all(mine)) cols.hide(s, base, lo, end, mine);
      cols.template softmax<LOW>(s, p, low, a.scale2);
      auto value = [&](int d, int j) {
        return *reinterpret_cast<const bf16x8*>(t.v + value_piece<DH>(d * 16 + col, grp, j));
      };
      bool special = false;
      if constexpr (LOW && !EIGHT) {
        const int* w = low_special[i & 1];
        // a scalar: matrix instructions run whatever lanes a branch leaves on
        special = __builtin_amdgcn_readfirstlane(w[0] | w[1] | w[2] | w[3]);
        if (special) cols.template add_values<true>(p, low, value);
      }
      if (!special) cols.template add_values_ahead<LOW>(p, low, value);
    }
    if (more) stage(i + 1);
    __syncthreads();
  }

  // every wave writes its own columns
  const bool any = __any(odd);
  if (lane == 0) special_of[wave] = any;
  __syncthreads();
  const int whole = max(min(hi, least) / PAGED_TILE * PAGED_TILE, k0);
  const bool special = special_of[0] | special_of[1] | special_of[2] | special_of[3];
#pragma unroll
  for (int t = 0; t < CT; ++t)
    write_column<DH, EIGHT, bf16_t>(c, bt, a, sp, my_col + t * 16 + col, chunk, k0, k1, whole, special, cols.o[t],
                                    cols.m[t], cols.l[t][0], grp * 4, 16, grp == 0);
}

template <int DH, int CT>
static void launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, const AttendArgs& a,
                   unsigned grid, hipStream_t st) {
  if (c->eight_bit)
    paged_tiles_kernel<DH, CT, true><<<grid, 64 * PAGED_WAVES, 0, st>>>(paged_cache(c), paged_batch(b), a);
  else
    paged_tiles_kernel<DH, CT, false><<<grid, 64 * PAGED_WAVES, 0, st>>>(paged_cache(c), paged_batch(b), a);
}

void paged_tiles_launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, const AttendArgs& a,
                        const AttendPlan& p, unsigned grid, hipStream_t st) {
  if (c->head_dim == 64) {
    if (p.column_tiles == 1) launch<64, 1>(c, b, a, grid, st);
    else launch<64, 2>(c, b, a, grid, st);
  } else {
    if (p.column_tiles == 1) launch<128, 1>(c, b, a, grid, st);
    else launch<128, 2>(c, b, a, grid, st);
  }
}
