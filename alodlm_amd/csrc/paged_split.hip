// Attention over paged keys on the matrix cores, the keys split over the waves: bf16,
// head_dim 64 and 128, few rows a sequence (decoding steps and windows).
//
// A decoding step reads every key and value once and does a few operations with each:
// it is bound by the bytes.  So nothing is staged: every wave takes 64-key tiles of its
// own straight from memory into the registers that the matrix instructions read, one
// tile ahead, and no wave waits for another until the end.
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

// A lane's places in the pages of one tile: for the keys (16-key group (lane % 16) / 4)
// and for the values (group lane / 16); -1 where a page is missing.
struct Places {
  int64_t k, v;
};

// One 64-key tile in registers.  8 bits: k[t][c] 16 dims of a key, v[d] 16 keys of a
// dimension; 16 bits: the same in twice the registers.
template <int DH, bool EIGHT> struct Tile {
  static constexpr int KC = DH / (EIGHT ? 64 : 32), VC = EIGHT ? 1 : 2;
  uint4 k[4][KC];
  uint4 v[DH / 16][VC];
  float k_scale, v_scale;
  bool k_ok, v_ok;
};

template <int DH, int CT, bool EIGHT>
__global__ void __launch_bounds__(64 * SPLIT_WAVES, CT == 1 ? 2 : 1)
paged_split_kernel(PagedCache c, PagedBatch bt, AttendArgs a) {
  constexpr int FR = DH / 32, DT = DH / 16;  // query fragments, output row tiles
  __shared__ __attribute__((aligned(16))) float buf[SPLIT_WAVES][16 * (DH + 4)];
  __shared__ float m_of[SPLIT_WAVES][16], l_of[SPLIT_WAVES][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int page = c.page, shift = 31 - __builtin_clz(page);
  // query tiles of one (sequence, head, chunk) lie a multiple of the others apart, so
  // that they tend to meet on one die's cache
  const int per_tile = bt.sequences * c.kv_heads * a.chunks;
  const int qt = blockIdx.x / per_tile, rest = blockIdx.x % per_tile;
  const int chunk = rest % a.chunks, h = rest / a.chunks % c.kv_heads;
  const int b = rest / a.chunks / c.kv_heads;
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
  auto places = [&](int base, int lo, int hi, auto eight) {
    return Places{find(base + (col >> 2) * 16, lo, hi, eight), find(base + grp * 16, lo, hi, eight)};
  };
  auto load = [&](int base, const Places& pl, auto eight) {
    constexpr bool E = decltype(eight)::value;
    typedef typename std::conditional<E, e4m3_t, bf16_t>::type S;
    Tile<DH, E> t;
    const S* keys = (const S*)(EIGHT && !E ? c.open_keys : c.keys);
    const S* values = (const S*)(EIGHT && !E ? c.open_values : c.values);
    t.k_ok = pl.k >= 0;
    t.v_ok = pl.v >= 0;
    t.k_scale = t.v_scale = 1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < Tile<DH, E>::KC; ++j) t.k[i][j] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int j = 0; j < Tile<DH, E>::VC; ++j) t.v[d][j] = make_uint4(0, 0, 0, 0);
    if (t.k_ok) {
      const int in_page = (base + (col >> 2) * 16) & (page - 1);
      const S* p = keys + pl.k * head_block + (int64_t)(in_page + (col & 3)) * DH + grp * 16;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < Tile<DH, E>::KC; ++j)
          t.k[i][j] = *reinterpret_cast<const uint4*>(
              p + 4 * i * DH + (E ? j * 64 : (j / 2) * 64 + (j % 2) * 8));
      if (E) t.k_scale = exp2_int(c.exponents[pl.k / c.kv_heads * 2 * c.kv_heads + h]);
    }
    if (t.v_ok) {
      const int in_page = (base + grp * 16) & (page - 1);
      const S* p = values + pl.v * head_block + (int64_t)col * page + in_page;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < Tile<DH, E>::VC; ++j)
          t.v[d][j] = *reinterpret_cast<const uint4*>(p + d * 16 * page + j * 8);
      if (E) t.v_scale = exp2_int(c.exponents[(pl.v / c.kv_heads * 2 + 1) * c.kv_heads + h]);
    }
    return t;
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
  auto compute = [&](Tile<DH, true>* t8, Tile<DH, false>* t16, int base, int lo, int hi, auto eight) {
    constexpr bool E = decltype(eight)::value;
    f32x4 s[CT][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int t = 0; t < CT; ++t) s[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < FR; ++f) {
        bf16x8 k;
        if constexpr (E) {
          const uint4 w = t8->k[i][f / 2];
          k = f % 2 ? widen(w.z, w.w, t8->k_scale) : widen(w.x, w.y, t8->k_scale);
        } else {
          k = __builtin_bit_cast(bf16x8, t16->k[i][f]);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) s[t][i] = mfma16(k, q[t][f], s[t][i]);
      }
    }
    const bool v_ok = E ? t8->v_ok : t16->v_ok;
    // tiles that every row sees whole need no mask
    const bool masked = base < lo || base + SPLIT_TILE > min(hi, least) || !__all(v_ok);
    if (masked) {
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = base + grp * 16 + i;
          if (!(key >= lo && key < min(hi, limit[t]) && v_ok)) s[t][i / 4][i % 4] = -INFINITY;
        }
    }
    bf16x8 p[CT][2];
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
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[t][i / 4][i % 4], a.scale2, -base_m));
        p[t][i / 8][i % 8] = (__bf16)e;
      }
    }
    bool special = false;  // a value that is inf or NaN, in a tile that not all rows see whole
    if (masked) {
      uint32_t odd = 0;
      auto clean = [&](uint32_t& w, bool write) {  // bytes (halves) of all ones in the exponent -> 0
        if constexpr (E) {
          const uint32_t z = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          odd |= z;
          if (write) w &= ~((z >> 7) * 0xffu);
        } else {
          const uint32_t z = ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
          odd |= z;
          if (write) w &= ~((z >> 15) * 0xffffu);
        }
      };
      auto sweep = [&](bool write) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int j = 0; j < (E ? 1 : 2); ++j) {
            uint4& w = E ? t8->v[d][0] : t16->v[d][j];
            clean(w.x, write);
            clean(w.y, write);
            clean(w.z, write);
            clean(w.w, write);
          }
      };
      sweep(false);
      special = __any(odd);
      if (special) sweep(true);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int t = 0; t < CT; ++t) l[t] = mfma16(ones, p[t][j], l[t]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        bf16x8 v;
        if constexpr (E) {
          const uint4 w = t8->v[d][0];
          v = j ? widen(w.z, w.w, t8->v_scale) : widen(w.x, w.y, t8->v_scale);
        } else {
          v = __builtin_bit_cast(bf16x8, t16->v[d][j]);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) o[t][d] = mfma16(v, p[t][j], o[t][d]);
      }
    }
    if (special) add_special(base, p, lo, hi, eight);
  };

  constexpr int STEP = SPLIT_WAVES * SPLIT_TILE;
  if constexpr (EIGHT) {  // sealed pages, one tile ahead
    const int hi = min(k1, sealed);
    int base = k0 + wave * SPLIT_TILE;
    if (base < hi) {
      Places pl = places(base, 0, hi, std::true_type());
      Tile<DH, true> tile = load(base, pl, std::true_type());
      pl = places(base + STEP, 0, hi, std::true_type());
      while (true) {
        Tile<DH, true> now = tile;
        const bool more = base + STEP < hi;
        if (more) {
          tile = load(base + STEP, pl, std::true_type());
          pl = places(base + 2 * STEP, 0, hi, std::true_type());
        }
        compute(&now, nullptr, base, 0, hi, std::true_type());
        if (!more) break;
        base += STEP;
      }
    }
  }
  {  // 16-bit pages: the pool's, or the open ones behind the sealed
    const int lo = EIGHT ? max(k0, sealed) : k0;
    const int start = lo / SPLIT_TILE * SPLIT_TILE;
    // tiles keep the waves' turns
    for (int base = start + ((wave - start / SPLIT_TILE) & (SPLIT_WAVES - 1)) * SPLIT_TILE; base < k1;
         base += STEP) {
      const Places pl = places(base, lo, k1, std::false_type());
      Tile<DH, false> tile = load(base, pl, std::false_type());
      compute(nullptr, &tile, base, lo, k1, std::false_type());
    }
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
                        const AttendPlan& p, hipStream_t st) {
  const unsigned grid = (unsigned)(b->sequences * c->kv_heads * p.query_tiles * a.chunks);
  if (c->head_dim == 64) {
    if (p.column_tiles == 1) launch<64, 1>(c, b, a, grid, st);
    else launch<64, 2>(c, b, a, grid, st);
  } else {
    if (p.column_tiles == 1) launch<128, 1>(c, b, a, grid, st);
    else launch<128, 2>(c, b, a, grid, st);
  }
}
