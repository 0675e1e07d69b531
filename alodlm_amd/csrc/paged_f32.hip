// Attention over paged keys for float32 models on the float32 matrix instructions
// (v_mfma_f32_16x16x4_f32): head_dim 64 and 128, pages in float32 or 8 bits.
//
// The same transposed products as in bf16, 16 query columns a wave, in float32
// throughout.  A lane's 4 scores of a 16-key subtile are keys 4 (lane / 16) .. + 4: as an
// operand of the second product they are the probabilities of one key in each lane
// group, and a lane's 16 bytes of a value row (4 bytes of codes) the values of those four.
// A subtile lies in one page, whose number and scales are therefore the wave's.
//
// Every value that a wave reads feeds 16 columns at the float32 rate, 32 cycles for 64
// bytes a lane group: the caches keep up, so nothing is staged.  With few columns the
// keys are split over the waves, else the columns.
//
// Measured: five sequences of 1 to 3 rows over 30 to 903 float32 tokens, 16 heads over 8,
// 23 MB: 14 us and 4 for the join: chunks of 256 keys, one tile a wave, whose 256 matrix
// instructions (3.4 us) and loads follow each other.  64 rows of 16 heads over 200 to 8000
// tokens, 2.1 GB: 510 us (4.2 TB/s); over 8-bit pages, a quarter of the bytes, 363.
#include "paged_mfma.h"

__device__ __forceinline__ f32x4 mfma16_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Four values of a row.
__device__ __forceinline__ f32x4 load_four(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
__device__ __forceinline__ f32x4 load_four(const e4m3_t* p) {
  const int w = *reinterpret_cast<const int*>(p);
  return f32x4{__builtin_amdgcn_cvt_f32_fp8(w, 0), __builtin_amdgcn_cvt_f32_fp8(w, 1),
               __builtin_amdgcn_cvt_f32_fp8(w, 2), __builtin_amdgcn_cvt_f32_fp8(w, 3)};
}

template <int DH, bool EIGHT, bool SPLIT_KEYS>
__global__ void __launch_bounds__(64 * PAGED_WAVES)
paged_f32_kernel(PagedCache c, PagedBatch bt, AttendArgs a) {
  constexpr int DT = DH / 16, COLS = SPLIT_KEYS ? 16 : 16 * PAGED_WAVES;
  __shared__ __attribute__((aligned(16))) WaveJoin<SPLIT_KEYS ? DH : 16> join;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  if (blockIdx.x >= gridDim.x - a.zero_blocks) {
    zero_rest(bt, (float*)a.out, (int64_t)a.heads * DH, gridDim.x - 1 - blockIdx.x, a.zero_blocks);
    return;
  }
  const int page = c.page, head_block = page * DH;
  // heads, sequences (turned on by one per chunk), chunks, query tiles, the last first
  const int per_chunk = bt.sequences * c.kv_heads, per_tile = per_chunk * a.chunks;
  const int qt = a.query_tiles - 1 - blockIdx.x / per_tile, rest = blockIdx.x % per_tile;
  const int chunk = rest / per_chunk;
  const Span sp = Span::of<EIGHT>(c, bt, (rest % per_chunk / c.kv_heads + chunk + qt) % bt.sequences,
                                  rest % c.kv_heads);
  if (qt * COLS >= sp.given * a.group) return;
  const int first = qt * COLS + (SPLIT_KEYS ? 0 : wave * 16);
  const int row_lo = first / a.group, row_hi = min((first + 15) / a.group, sp.n - 1);
  const int least = sp.limit(row_lo), most = row_hi < row_lo ? 0 : sp.limit(row_hi);
  const int k0 = chunk * a.chunk_keys, k1 = min(most, k0 + a.chunk_keys);
  if (SPLIT_KEYS && k1 <= k0 && chunk > 0) return;

  const int x = first + col, row = x / a.group, limit = sp.limit(row);
  f32x4 q[DT], o[DT];
  float m = -INFINITY, sum = 0.f;  // the sum over this lane's keys
  const float* qp = (const float*)a.q + (sp.row0 + row) * a.ldq + (int64_t)(sp.h * a.group + x % a.group) * DH;
#pragma unroll
  for (int j = 0; j < DT; ++j) {
    q[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (row < sp.n) q[j] = load_four(qp + j * 16 + grp * 4);
    o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  uint32_t odd = 0;
  // Tiles [from, to) of keys [lo, to); whole: every column sees all of them.
  auto tiles = [&](int from, int to, int lo, bool whole, auto pool) {
    constexpr bool POOL = decltype(pool)::value, E = EIGHT && POOL;
    typedef typename std::conditional<E, e4m3_t, float>::type S;
    const S* keys = (const S*)(EIGHT && !POOL ? c.open_keys : c.keys);
    const S* values = (const S*)(EIGHT && !POOL ? c.open_values : c.values);
    const int step = SPLIT_KEYS ? PAGED_WAVES * PAGED_TILE : PAGED_TILE;
    int base = from;
    if (SPLIT_KEYS) base += ((wave - from / PAGED_TILE) & (PAGED_WAVES - 1)) * PAGED_TILE;
    for (; base < to; base += step) {
      int id[4];
      const S *kp[4], *vp[4];
      f32x4 s[4], s_odd[4];  // two sums each: half the roundings in a row
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = base + 16 * i;
        id[i] = __builtin_amdgcn_readfirstlane(sp.page<POOL>(c, bt, key, lo, to));
        const int64_t block = sp.block(c, max(id[i], 0), head_block);
        kp[i] = keys + block + (((key & (page - 1)) + col) * DH + grp * 4);
        vp[i] = values + block + (col * page + (key & (page - 1)) + grp * 4);
        s[i] = s_odd[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        f32x4 k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = load_four(kp[i] + j * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f32x4& to = j % 2 ? s_odd[i] : s[i];
            to = mfma16_f32(k[i][e], q[j][e], to);
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += s_odd[i];
      float k_scale[4], v_scale[4] = {1.f, 1.f, 1.f, 1.f};
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k_scale[i] = a.scale2;
        if (E && id[i] >= 0) {
          k_scale[i] *= exp2_int(sp.exponent(c, id[i], 0));
          v_scale[i] = exp2_int(sp.exponent(c, id[i], 1));
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = base + 16 * i + 4 * grp + r;
          if (id[i] < 0 || (!whole && !(key >= lo && key < min(to, limit)))) s[i][r] = -INFINITY;
          top = fmaxf(top, s[i][r] * k_scale[i]);
        }
      }
      if (__any(top > m + 8.f)) {  // the reference follows the maximum in steps
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float to_m = fmaxf(m, top);
        const float f = to_m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to_m);
        m = to_m;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
      }
      const float base_m = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 p;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], k_scale[i], -base_m));
          sum += p[r];
        }
        if (id[i] < 0) continue;
        p *= v_scale[i];
        f32x4 v[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) v[d] = load_four(vp[i] + d * 16 * page);
        if (!whole)
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool fine = fabsf(v[d][r]) < INFINITY;
              odd |= !fine;
              v[d][r] = fine ? v[d][r] : 0.f;
            }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d] = mfma16_f32(v[d][r], p[r], o[d]);
      }
    }
  };
  const int hi = EIGHT ? min(k1, sp.sealed) : k1;
  const int whole = max(min(hi, least) / PAGED_TILE * PAGED_TILE, k0);
  tiles(k0, whole, k0, true, std::true_type());
  tiles(whole, hi, k0, false, std::true_type());
  if constexpr (EIGHT) {
    const int lo = max(k0, sp.sealed);
    if (lo < k1) tiles(lo / PAGED_TILE * PAGED_TILE, k1, lo, false, std::false_type());
  }
  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  if constexpr (SPLIT_KEYS) {
    f32x4 out[1][DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) out[0][d] = o[d];
    const float top[1] = {m}, total[1] = {sum};
    join.template write<EIGHT, float>(c, bt, a, sp, first, chunk, k0, k1, whole, __any(odd), out, top, total);
  } else {
    write_column<DH, EIGHT, float>(c, bt, a, sp, x, chunk, k0, k1, whole, __any(odd), o, m, sum, grp * 4, 16,
                                   grp == 0);
  }
}

template <int DH, bool EIGHT>
static void launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, const AttendArgs& a,
                   const AttendPlan& p, unsigned grid, hipStream_t st) {
  if (p.kernel == PAGED_F32_COLUMNS)
    paged_f32_kernel<DH, EIGHT, false><<<grid, 64 * PAGED_WAVES, 0, st>>>(paged_cache(c), paged_batch(b), a);
  else
    paged_f32_kernel<DH, EIGHT, true><<<grid, 64 * PAGED_WAVES, 0, st>>>(paged_cache(c), paged_batch(b), a);
}

void paged_f32_launch(const alodlm_paged_cache* c, const alodlm_paged_batch* b, const AttendArgs& a,
                      const AttendPlan& p, unsigned grid, hipStream_t st) {
  if (c->head_dim == 64) {
    if (c->eight_bit) launch<64, true>(c, b, a, p, grid, st);
    else launch<64, false>(c, b, a, p, grid, st);
  } else {
    if (c->eight_bit) launch<128, true>(c, b, a, p, grid, st);
    else launch<128, false>(c, b, a, p, grid, st);
  }
}
