// Losses over the vocabulary from hidden states [rows, width] and the output projection
// [vocab, width], without the logits, and their gradients (vocab_loss.h has the
// mathematics).
//
// Forward: the logits leave the matrix cores tile by tile (256 rows x 256 tokens, the
// two-stage kernel of gemm_dl_tile.h) and are summed where they are, in the epilogue: a
// tile leaves one part (largest logit, sum) a row, 8 bytes for 256 logits.  Backward: a piece
// of the vocabulary at a time, the tiles are computed once more and leave the piece's gradient
// D = dloss / dlogits in bf16, from which two products give its share of d_hidden (D W, in
// float32 planes that one pass adds up; where the planes would pass 1 GiB the pieces add to one
// in their epilogues, at the same speed: 16384 rows of width 4096 59.5 -> 59.1 ms, 2.97 -> 0.72
// GiB) and its rows of d_weight (D^T hidden, written once).  Four products of 2 rows vocab width
// operations in all, of which the second computation of the logits is what not keeping them
// costs.
//
// Logits of at most 2^25 values are cheaper to keep, in float32, than to compute again (and
// the products of few rows read the weight, which a tile of 256 rows would wait for): they
// go through memory and the row kernels of vocab_loss.hip, as those of float32 models and
// of 64 rows or fewer do, piece by piece where they are more.
//
// D is rounded to bf16 (half a step, 2^-8 of a value at most), as a bf16 model's logits'
// gradient is anywhere: it is an operand of the bf16 matrix cores.  A reduced loss's upstream
// gradient is applied to the products, not to D: of a row far from its target, D is then -1
// there, which is exact.  Of few rows, whose D's rounding does not average out (13 rows: 1.5
// times the error of the result's own), D is two bf16 parts that the products take as rows of
// their own, waiting for the weight as before: 16 rows of width 4096 against 151936 tokens 782 ->
// 793 us, 64 of width 2048 516 -> 587.
#include "few_bf16.h"
#include "few_f32.h"
#include "gemm_dl_tile.h"
#include "gemm_mid.h"
#include "vocab_loss.h"

namespace {

// max / sum over the four lanes that share a tile row (lane % 16)
__device__ __forceinline__ float quad_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The known tokens of a tile's rows, in LDS: a bit a column, and how many of a row's known
// tokens come before the tile.  A row's tokens ascend, so a marked column's place among
// them is that count plus the marks before it.
struct TileMarks {
  static constexpr int BYTES = TB * 32 + TB * 2;
  // thread t: row t of the tile
  static __device__ __forceinline__ void fill(char* lds, const KnownRows& k, int64_t row, int64_t rows,
                                              int64_t token0) {
    uint32_t* bits = reinterpret_cast<uint32_t*>(lds) + 8 * threadIdx.x;
    *reinterpret_cast<uint4*>(bits) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(bits + 4) = make_uint4(0, 0, 0, 0);
    int before = 0;
    if (row < rows) {
      const int K = k.known, token = (int)token0;
      const int* ids = k.ids + row * K;
      // the first that is not before the tile: eight parts of what is left, seven loads at once
      // (2048 rows of width 2048 against 151936 tokens, 64 known a row: 4.51 -> 4.34 ms, 256: 5.61 ->
      // 4.43).
      // Every loaded id is used, or the main loop would wait for those that are not.
      for (int n = K; n > 8;) {
        n = (n + 7) >> 3;
        int parts = 0;
#pragma unroll
        for (int j = 1; j < 8; ++j) {
          const int at = before + j * n - 1;
          parts += (int)(ids[at < K ? at : K - 1] < token) & (int)(at < K);
        }
        before += parts * n;
      }
      bool more = true;
      for (int i = before; more && i < K; i += 8) {
        int id[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) id[e] = ids[i + e < K ? i + e : K - 1];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = (i + e < K ? id[e] : VL_NONE) - token;
          before += at < 0;
          if ((unsigned)at < (unsigned)TB) bits[at >> 5] |= 1u << (at & 31);
          more = at < TB;
        }
      }
    }
    reinterpret_cast<uint16_t*>(lds + TB * 32)[threadIdx.x] = (uint16_t)before;
  }
  static __device__ __forceinline__ uint4 half(const char* lds, int row, int wn) {
    return reinterpret_cast<const uint4*>(lds)[2 * row + wn];
  }
  static __device__ __forceinline__ uint32_t nibble(const uint4& b, int j, int g) {
    const uint32_t w = j < 2 ? b.x : j < 4 ? b.y : j < 6 ? b.z : b.w;
    return w >> (16 * (j & 1) + 4 * g) & 15u;
  }
  static __device__ __forceinline__ int before(const char* lds, int row) {
    return reinterpret_cast<const uint16_t*>(lds + TB * 32)[row];
  }
  // place of tile column col (marked) among the row's known tokens
  static __device__ __forceinline__ int place(const char* lds, int row, int col) {
    const uint32_t* bits = reinterpret_cast<const uint32_t*>(lds) + 8 * row;
    int n = before(lds, row);
    for (int w = 0; w < col >> 5; ++w) n += __popc(bits[w]);
    return n + __popc(bits[col >> 5] & ((1u << (col & 31)) - 1u));
  }
};

// Tile rows that are swept together: all of them up to six, else three, as gemm_dl.hip's
// products (a lone fourth row took the weight once more: 777 rows 1.62 -> 1.59 ms, 1000 rows of
// width 4096 4.41 -> 4.30; of 16 tile rows, three together take 7.92 ms, four 7.96, 16 8.04).
__device__ __forceinline__ int swept_rows(int tiles_m) { return tiles_m <= 6 ? tiles_m : 3; }

// Forward tiles: parts of the rows' sums, and the known tokens' logits.  The parts' reference
// is the largest exponent z c rounded up to a whole number K: 2^(z c - K) is one multiply-add
// and one exponential, K is exact, and parts are joined by whole powers of two.  The values
// of 16 rows that hold a known token, or columns past the vocabulary, go through LDS, where
// single ones can be reached (a lane's own 32 values, so nothing waits for another lane);
// selecting them in registers made the compiler spill 52 of them, 5 % of the kernel's time.
struct SumHooks {
  static constexpr bool Epilogue = true;
  static constexpr int EXTRA_LDS = TileMarks::BYTES + 2 * TB * (int)sizeof(Part);
  static __device__ int group(int tiles_m) { return swept_rows(tiles_m); }
  KnownRows k;
  float c;
  Part* part;     // [tiles][rows], of the piece
  int64_t first;  // the piece's first token

  __device__ __forceinline__ void before(char* extra, int64_t M, int64_t m0, int64_t n0) const {
    TileMarks::fill(extra, k, m0 + threadIdx.x, M, first + n0);
  }
  template <typename Quad>
  __device__ __forceinline__ void after(char* lds, char* extra, Quad quad, void*, int64_t, int64_t M,
                                        int64_t N, int64_t m0, int64_t n0) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = wave & 1, g = lane >> 4;
    Part* red = reinterpret_cast<Part*>(extra + TileMarks::BYTES);
    // this lane's values: 16 bytes at own + 1024 j
    char* own = lds + 8192 * wave + 16 * lane;
    const bool edge = n0 + TB > N;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the stages are free
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v[8][4];
      int row = 0, col = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) quad(8 * i + j, row, col, v[j]);
      const uint4 b = TileMarks::half(extra, row, wn);
      if (edge || __any((b.x | b.y | b.z | b.w) != 0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<float4*>(own + 1024 * j) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
        uint32_t mine = 0;  // a bit a column of this lane
#pragma unroll
        for (int j = 0; j < 8; ++j) mine |= TileMarks::nibble(b, j, g) << (4 * j);
        for (; mine; mine &= mine - 1) {
          const int at = __builtin_ctz(mine), tile_col = wn * 128 + 16 * (at >> 2) + 4 * g + (at & 3);
          float* z = reinterpret_cast<float*>(own + 1024 * (at >> 2)) + (at & 3);
          k.logit[(m0 + row) * k.known + TileMarks::place(extra, row, tile_col)] = *z;
          *z = -INFINITY;
        }
        if (edge)
#pragma unroll 1
          for (int at = 0; at < 32; ++at)
            if (n0 + wn * 128 + 16 * (at >> 2) + 4 * g + (at & 3) >= N)
              *(reinterpret_cast<float*>(own + 1024 * (at >> 2)) + (at & 3)) = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 x = *reinterpret_cast<const float4*>(own + 1024 * j);
          v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
        }
      }
      float m = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        m = fmaxf(m, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
      m = part_ref(quad_max(m), c);
      const float minus = m == -INFINITY ? 0.f : -m;
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += __builtin_amdgcn_exp2f(fmaf(v[j][e], c, minus));
      const float sum = quad_sum((s[0] + s[1]) + (s[2] + s[3]));
      if (g == 0) red[wn * TB + row] = {m, sum};
    }
    __syncthreads();
    const int t = threadIdx.x;
    if (m0 + t < M) part[n0 / TB * M + m0 + t] = part_join(red[t], red[TB + t], 1.f);
  }
};

// Backward tiles: D of a piece of the vocabulary, bf16, zero in the padding.
struct GradHooks {
  static constexpr bool Epilogue = true;
  static constexpr int EXTRA_LDS = TileMarks::BYTES + TB * 16;
  static __device__ int group(int tiles_m) { return swept_rows(tiles_m); }
  KnownRows k;
  float c;
  Upstream up;
  int64_t first;          // the piece's first token
  int64_t rows, columns;  // of D, padding included

  __device__ __forceinline__ void before(char* extra, int64_t M, int64_t m0, int64_t n0) const {
    const int64_t row = m0 + threadIdx.x;
    float4 r = make_float4(0.f, 1e30f, 0.f, 0.f);  // 2^-1e30: nothing
    if (row < M) {
      const float* info = k.info + 8 * row;
      const float g = up.row(row);
      const float f = info[RI_FACTOR];
      r.z = g;
      if (g != 0.f && f != 0.f) {
        // the whole part of the exponent joins the whole reference, where it is exact
        const float whole = floorf(info[RI_LOG]);
        r.x = g * f * __builtin_amdgcn_exp2f(whole - info[RI_LOG]);
        r.y = info[RI_M] + whole;
      } else if (!(info[RI_LOG] < INFINITY)) {
        r.w = 1.f;  // NaN that takes no part
      }
    }
    reinterpret_cast<float4*>(extra + TileMarks::BYTES)[threadIdx.x] = r;
    TileMarks::fill(extra, k, row, M, first + n0);
  }
  template <typename Quad>
  __device__ __forceinline__ void after(char* lds, char* extra, Quad quad, void* D, int64_t ldd,
                                        int64_t M, int64_t N, int64_t m0, int64_t n0) const {
    const int lane = threadIdx.x & 63, wm = threadIdx.x >> 7;
    const float4* consts = reinterpret_cast<const float4*>(extra + TileMarks::BYTES);
    float factor[8], log_rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 r = consts[wm * 128 + 16 * i + (lane & 15)];
      factor[i] = r.x;
      log_rest[i] = r.y;
    }
    auto grad = [&](int t, int& row, int& col, float* v) {
      const int i = t >> 3;
      quad(t, row, col, v);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = factor[i] * __builtin_amdgcn_exp2f(fmaf(v[e], c, -log_rest[i]));
    };
    tile_epilogue<ALODLM_EPI_STORE, 256, false>(lds, grad, D, ldd, nullptr, 0, rows, columns, m0, n0,
                                                1.f, nullptr, 0);
    // the known tokens' own and the padding, behind the tile's stores
    __syncthreads();
    const int64_t row = m0 + threadIdx.x;
    if (n0 + TB > N && row < rows)
      for (int64_t at = N; at < columns; ++at) reinterpret_cast<bf16_t*>(D)[row * ldd + at] = 0;
    if (row >= M) return;
    const float own_up = consts[threadIdx.x].z;
    if (consts[threadIdx.x].w != 0.f)
      for (int64_t at = n0; at < N && at < n0 + TB; ++at) reinterpret_cast<bf16_t*>(D)[row * ldd + at] = 0;
    const uint32_t* bits = reinterpret_cast<const uint32_t*>(extra) + 8 * threadIdx.x;
    const float* own = k.weight + row * k.known + TileMarks::before(extra, threadIdx.x);
    for (int w = 0; w < 8; ++w)
      for (uint32_t b = bits[w]; b; b &= b - 1, ++own)
        reinterpret_cast<bf16_t*>(D)[row * ldd + n0 + 32 * w + __builtin_ctz(b)] =
            float_to_bf16(own_up == 0.f ? 0.f : own_up * *own);
  }
};

template <typename Hooks>
void tiles_launch(const bf16_t* hidden, int64_t ldh, const bf16_t* weight, int64_t ldw, int64_t rows,
                  int64_t tokens, int64_t width, void* out, int64_t ldo, const Hooks& hooks,
                  hipStream_t st) {
  const int64_t tiles = ((rows + TB - 1) / TB) * ((tokens + TB - 1) / TB);
  gemm_dl2_kernel<true, true, ALODLM_EPI_STORE, false, Hooks><<<dim3((unsigned)tiles, 1), 256, 0, st>>>(
      hidden, ldh, weight, ldw, out, ldo, nullptr, 0, rows, tokens, width, 1.f, width, nullptr, 0, hooks);
}

// Rows of d_weight straight from the tiles: times the upstream gradient, rounded once.
struct ScaleHooks {
  static constexpr bool Epilogue = true;
  Upstream up;
  template <typename Quad>
  __device__ __forceinline__ void after(char* lds, Quad quad, void* C, int64_t ldc, int64_t M, int64_t N,
                                        int64_t m0, int64_t n0) const {
    tile_epilogue<ALODLM_EPI_STORE, 256, true>(lds, quad, C, ldc, nullptr, 0, M, N, m0, n0, up.all(),
                                               nullptr, 0);
  }
};

// dst [padded, padded_width] = src [rows, width] `times` below each other, zeros around them, 16
// bytes a thread.
template <typename T>
__global__ void __launch_bounds__(256)
copy_rows_kernel(const T* __restrict__ src, int64_t lds, int64_t rows, int64_t width, T* __restrict__ dst,
                 int64_t padded, int64_t padded_width, int times) {
  constexpr int N = 16 / (int)sizeof(T);
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N;
  if (at >= padded_width) return;
  for (int64_t row = blockIdx.y; row < padded; row += gridDim.y) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows * times && at < width)
      v = *reinterpret_cast<const uint4*>(src + (row < rows ? row : row - rows) * lds + at);
    *reinterpret_cast<uint4*>(dst + row * padded_width + at) = v;
  }
}

// out [rows, width] = up.all() * (the planes' sum + the last `rest` columns of D's parts times the
// weight's last `rest` rows, which no product took), rounded once.  GROUPS of threads take
// every GROUPS-th plane each (many planes of few rows: a thread would wait for one after the
// other), their sums are added in order.
template <typename T, int GROUPS>
__global__ void __launch_bounds__(256)
finish_product_kernel(const float* __restrict__ planes, int64_t count, int64_t rows, int64_t width,
                      Upstream up, const T* __restrict__ D, int64_t ldd, const T* __restrict__ weight,
                      int64_t ldw, int rest, int parts, T* __restrict__ out) {
  constexpr int LANES = 256 / GROUPS, VEC = 4;
  __shared__ float shared[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? LANES * VEC : 1];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int64_t at = ((int64_t)blockIdx.x * LANES + lane) * VEC;
  const bool inside = at < width;
  const float scale = up.all();
  const int64_t plane = rows * width;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float* src = planes + row * width + at;
    float s[VEC] = {};
    if (inside)
#pragma unroll 8
      for (int64_t p = group; p < count; p += GROUPS) {
        const float4 x = *reinterpret_cast<const float4*>(src + p * plane);
        s[0] += x.x; s[1] += x.y; s[2] += x.z; s[3] += x.w;
      }
    if constexpr (GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VEC; ++e) shared[group][lane * VEC + e] = s[e];
      __syncthreads();
      if (group) continue;
      for (int n = 1; n < GROUPS; ++n)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] += shared[n][lane * VEC + e];
    }
    if (!inside) continue;
    for (int t = 0; t < rest; ++t) {
      float d = Elem<T>::load(D, row * ldd + t);
      if (parts > 1) d += Elem<T>::load(D, (rows + row) * ldd + t);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e] = fmaf(d, Elem<T>::load(weight, t * ldw + at + e), s[e]);
    }
    T* dst = out + row * width + at;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(scale * s[0], scale * s[1]),
                                                  pack_bf16x2(scale * s[2], scale * s[3]));
    else
      *reinterpret_cast<float4*>(dst) = make_float4(scale * s[0], scale * s[1], scale * s[2], scale * s[3]);
  }
}

int64_t ceil_div(int64_t x, int64_t by) { return (x + by - 1) / by; }
int64_t up_to(int64_t x, int64_t to) { return ceil_div(x, to) * to; }
dim3 row_grid(int64_t width, int64_t rows) {
  return dim3((unsigned)ceil_div(width, 256), (unsigned)(rows < 65535 ? rows : 65535));
}

template <typename T>
void finish_product(const float* planes, int64_t count, int64_t rows, int64_t width, const Upstream& up,
                    const T* D, int64_t ldd, const T* weight, int64_t ldw, int rest, int parts, T* out,
                    hipStream_t st) {
  if (count >= 16)
    finish_product_kernel<T, 16><<<row_grid(width / 4 * 16, rows), 256, 0, st>>>(
        planes, count, rows, width, up, D, ldd, weight, ldw, rest, parts, out);
  else
    finish_product_kernel<T, 1><<<row_grid(width / 4, rows), 256, 0, st>>>(
        planes, count, rows, width, up, D, ldd, weight, ldw, rest, parts, out);
}

// Which bf16 tiles a product [M, N] over K runs on and how its K is split: the least of
// the times that gemm.hip's rule is made of (a 32-deep step of a round of 256 workgroups:
// 0.58 to 0.78 us on 256x256 tiles, 0.28 us on 128x128 ones and 0.3 on 32 or 64 rows), and
// the float planes, written and read at 5.5 TB/s; `direct`: 256x256 tiles need none; `whole`: K is
// not split.
struct Split {
  bool large;
  int64_t planes;
};
Split split_product(int64_t M, int64_t N, int64_t K, bool large_ok, bool direct, bool few, bool whole = false) {
  const int64_t steps = ceil_div(K, 32);
  Split best = {true, 1};
  double least = 1e30;
  auto offer = [&](bool large, int64_t s, int64_t tiles, double each) {
    double t = (double)ceil_div(tiles * s, 256) * (double)ceil_div(steps, s) * each;
    if (!(large && direct)) t += 4.0 + 4e-6 / 5.5 * (double)(2 * s) * (double)M * (double)N;
    if (t < least) {
      least = t;
      best = {large, s};
    }
  };
  if (large_ok) {
    const int64_t tiles = ceil_div(M, 256) * ceil_div(N, 256);
    for (int64_t s = 1; s <= (direct || whole ? 1 : 32) && (s == 1 || steps / s >= 16); ++s) {
      const double fill = tiles * s < 256 ? (double)(tiles * s) / 256.0 : 1.0;
      offer(true, s, tiles, 0.58 + 0.2 * fill);
    }
  }
  const int64_t rows = !few ? 128 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  const int64_t tiles = ceil_div(M, rows) * ceil_div(N, 128);
  for (int64_t s = 1; s <= (whole ? 1 : 64) && (s == 1 || steps / s >= 8); ++s)
    offer(false, s, tiles, rows == 128 ? 0.28 : 0.3);
  return best;
}

constexpr int64_t KEPT = 1 << 25;                // logits that a forward keeps for its backward (128 MiB)
// of what is held of the vocabulary at a time: the logits, their gradient and copied rows of the
// weight, each
constexpr int64_t PIECE_BYTES = 512ll << 20;
// of d_hidden's planes; where they would be more, all pieces add to one (the pieces get smaller
// with the rows, so that their number times a plane's size grows with the square of the rows)
constexpr int64_t PLANE_BYTES = 1ll << 30;
constexpr int64_t FEW = ALODLM_FEW_ROWS;

// How a call runs, from its sizes alone.
struct Plan {
  bool half;              // bf16
  bool small, keep, tiles;  // few enough logits to keep; kept; never in memory
  bool few;                 // float32 products of few rows (few_f32.hip)
  int64_t piece, pieces;  // tokens of a piece (a multiple of 256), pieces
  int64_t deep, deep_rows;  // width and rows of D as the tile kernels take them
  int parts;                // of D, each of as many rows as there are
  bool copy_hidden, copy_weight;
  int64_t chunks, sum_parts;  // of a piece's rows, of all
  int64_t planes;           // of d_hidden, most
  bool add;                 // one, which the pieces add to
  bool direct;              // d_hidden needs no planes
  Split hidden_split, last_split;
  // workspace, in floats
  int64_t part, logits, D, hidden, weight, sums, rows, gemm, total;
};

// Row stride of a piece's logits in memory (a forward's and its backward's pieces differ, the
// logits between them do not).
int64_t logits_stride(const Plan& p, int64_t V, int64_t n) { return up_to(p.small ? V : n, 8); }

Plan make_plan(int64_t R, int64_t V, int64_t H, int dtype, bool keep, bool backward, bool d_hidden,
               bool d_weight) {
  Plan p = {};
  p.half = dtype == ALODLM_BF16;
  // (a loss has the same bits whether or not a backward will want the logits)
  p.small = R * up_to(V, 8) <= KEPT;
  p.keep = keep && p.small;
  p.tiles = p.half && !p.small && R > FEW;
  p.few = !p.half && R <= FEW_F32_ROWS && V * H >= (1 << 20);
  p.deep = p.half ? up_to(H, 64) : H;
  p.parts = backward && p.half && R <= FEW ? 2 : 1;
  const int64_t d_rows = p.parts * R;
  p.deep_rows = p.half ? up_to(d_rows, 32) : R;
  const int64_t es = p.half ? 2 : 4;
  const bool computes = !(backward && p.keep);  // the logits
  p.copy_weight = p.half && computes && p.deep != H;
  p.copy_hidden = p.copy_weight;
  // bytes of a token
  int64_t most = V;
  auto limit = [&](int64_t bytes) {
    const int64_t n = PIECE_BYTES / bytes / 256 * 256;
    most = n < most ? (n > 256 ? n : 256) : most;
  };
  if (backward && p.half) limit(2 * p.deep_rows);
  if (computes && !p.tiles && !p.small) limit(4 * R);
  if (backward && p.few) limit(4 * few_f32_pad(R));
  if (p.copy_weight) limit(2 * p.deep);
  if (p.half) {  // a piece of a weight without gaps stays in one launch of 128x128 tiles
    const int64_t n = (1ll << 30) / up_to(H, 64) / 256 * 256;
    most = n < most ? n : most;
  }
  p.pieces = ceil_div(V, most);
  p.piece = up_to(ceil_div(V, p.pieces), 256);
  p.pieces = ceil_div(V, p.piece);
  const int64_t last = V - (p.pieces - 1) * p.piece, whole = last / 32 * 32, rest = last - whole;
  int64_t at = 0, gemm = 0;
  auto room = [&](int64_t floats) {
    const int64_t here = at;
    at += up_to(floats, 64);
    return here;
  };
  auto product = [&](int64_t M, int64_t N, int64_t K, int epi) {
    if (M < 1 || K < 1) return;
    const int64_t n = alodlm_gemm_workspace(M, N, K, epi, dtype);
    gemm = n > gemm ? n : gemm;
  };
  const int f32_out = p.half ? ALODLM_EPI_STORE_F32 : ALODLM_EPI_STORE;
  // whole 32 rows for the large tiles; a row for each part of D
  p.copy_hidden |= backward && d_weight && p.parts > 1;
  if (backward && d_weight && p.half && p.deep_rows != R)
    for (const int64_t n : {p.piece, up_to(last, 32)})
      p.copy_hidden |= split_product(n, H, d_rows, true, true, false).large;
  if (p.copy_hidden) p.hidden = room(ceil_div(p.deep_rows * p.deep * es, 4));
  if (p.copy_weight) p.weight = room(ceil_div(p.piece * p.deep * es, 4));
  if (computes && !p.tiles) {
    if (!p.keep) p.logits = room(R * up_to(p.small ? V : p.piece, 8));
    if (p.pieces > 1) product(R, p.piece, p.deep, f32_out);
    product(R, last, p.deep, f32_out);
  }
  if (!backward) {
    p.chunks = p.tiles ? p.piece / TB : row_stats_chunks(R, p.piece);
    p.sum_parts = p.tiles ? ceil_div(V, TB) : p.chunks * p.pieces;
    p.part = room(2 * R * p.sum_parts);
  } else {
    // float32: D takes the place of logits that are not kept
    if (p.few) p.D = room(p.piece * few_f32_pad(R));
    else if (p.half || p.keep) p.D = room(ceil_div(p.deep_rows * p.piece * es, 4));
    else p.D = p.logits;
    if (p.few) {
      p.planes = (p.pieces - 1) * few_f32_planes(p.piece, H) + few_f32_planes(last, H);
      if (d_hidden) p.sums = room(p.planes * R * H);
    } else if (d_hidden) {
      const bool large = H >= 256;
      auto split = [&](int64_t K) {
        return p.half && K ? split_product(d_rows, H, K, large, false, true, p.add) : Split{true, 1};
      };
      p.hidden_split = split(p.piece);
      p.last_split = split(whole);
      p.planes = (p.pieces - 1) * p.hidden_split.planes + (whole ? p.last_split.planes : 0);
      if (p.planes > 1 && p.planes * d_rows * H * 4 > PLANE_BYTES) {
        p.add = true;
        p.hidden_split = split(p.piece);
        p.last_split = split(whole);
        p.planes = 1;
      }
      p.direct = !p.half && p.planes == 1 && rest == 0;
      if (!p.direct) p.sums = room(p.planes * d_rows * H);
      if (!p.half) {
        if (p.pieces > 1) product(d_rows, H, p.piece, f32_out);
        product(d_rows, H, whole, f32_out);
      }
    }
    if (d_weight && !p.few) {
      int64_t floats = 0;
      for (const int64_t n : {p.piece, up_to(last, 32)}) {
        if (p.half) {
          const Split s = split_product(n, H, d_rows, true, true, false);
          if (!s.large && s.planes * n * H > floats) floats = s.planes * n * H;
        } else {
          product(up_to(n == p.piece ? n : last, 8), H, R, f32_out);
        }
      }
      p.rows = room(floats);
    }
  }
  p.gemm = room(gemm);
  p.total = at;
  if (!gemm) p.gemm = -1;
  return p;
}

int check_linear(const char* what, const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                 int64_t R, int64_t V, int64_t H, int64_t known, float inv_t, int reduction, int dtype) {
  const int rc = check_vocab_loss(what, R, V, known, inv_t, reduction);
  if (rc) return rc;
  ALODLM_CHECK_ARG(dtype == ALODLM_F32 || dtype == ALODLM_BF16, "%s: unknown dtype %d", what, dtype);
  ALODLM_CHECK_ARG(H >= 1 && H < (1ll << 20), "%s: width out of range", what);
  ALODLM_CHECK_ARG(ldh >= H && ldw >= H && ldh < (1ll << 22) && ldw < (1ll << 22),
                   "%s: row strides out of range", what);
  if (R > 0)
    ALODLM_CHECK_ARG(hidden && weight, "%s: the call lacks an array", what);
  ALODLM_CHECK_ARG((R + 255) / 256 * ((V + 255) / 256) < VL_MOST_GROUPS, "%s: too many rows in one call", what);
  const int64_t step = dtype == ALODLM_BF16 ? 8 : 4;  // elements of 16 bytes
  ALODLM_CHECK_ARG(H % step == 0, "%s: rows must be whole 16 bytes", what);
  if (R > 0)
    ALODLM_CHECK_ARG((((uintptr_t)hidden | (uintptr_t)weight) & 15) == 0 && ldh % step == 0 && ldw % step == 0,
                     "%s: rows must be 16-byte aligned", what);
  return ALODLM_OK;
}

#define LL_CALL(expr)            \
  do {                           \
    const int _rc = (expr);      \
    if (_rc) return _rc;         \
  } while (0)

// What the calls below take of the plan and the caller's arrays.
template <typename T> struct Call {
  Plan p;
  const T* hidden;
  int64_t ldh;
  const T* weight;
  int64_t ldw;
  int64_t R, V, H;
  float* ws;
  int dtype;
  hipStream_t st;
  const T* deep_hidden;  // as the tile kernels take it
  int64_t deep_ldh;

  float* gemm() const { return p.gemm < 0 ? nullptr : ws + p.gemm; }
  void copy_hidden() {
    deep_hidden = hidden;
    deep_ldh = ldh;
    if (!p.copy_hidden) return;
    T* to = reinterpret_cast<T*>(ws + p.hidden);
    copy_rows_kernel<T><<<row_grid(p.deep / 8, p.deep_rows), 256, 0, st>>>(hidden, ldh, R, H, to, p.deep_rows, p.deep,
                                                                          p.parts);
    deep_hidden = to;
    deep_ldh = p.deep;
  }
  // the piece's rows of the weight for the products that compute logits
  const T* piece_weight(int64_t first, int64_t n, int64_t& ld) const {
    const T* w = weight + first * ldw;
    ld = ldw;
    if (!p.copy_weight) return w;
    T* to = reinterpret_cast<T*>(ws + p.weight);
    copy_rows_kernel<T><<<row_grid(p.deep / 8, n), 256, 0, st>>>(w, ldw, n, H, to, n, p.deep, 1);
    ld = p.deep;
    return to;
  }
  int64_t logits_ld(int64_t n) const { return logits_stride(p, V, n); }
  // float logits of a piece, row stride logits_ld(n)
  int logits(int64_t first, int64_t n, float* out) const {
    int64_t ld;
    const T* w = piece_weight(first, n, ld);
    const int64_t to = logits_ld(n);
    if constexpr (sizeof(T) == 2)
      if (R <= FEW && n >= 128 * 256) {
        few_bf16_logits(deep_hidden, deep_ldh, w, ld, R, n, p.deep, out, to, st);
        ALODLM_CHECK_LAUNCH("linear_loss_logits");
        return ALODLM_OK;
      }
    if constexpr (sizeof(T) == 2)
      // 256 rows of tiles at once, where the dispatch would take two of 128
      if (R > 128 && R < 256 && n >= 256 * 128) {
        int64_t count = 1;
        gemm_dl_launch(deep_hidden, deep_ldh, 1, w, ld, 1, out, to, nullptr, 0, R, n, p.deep, 1.f,
                       ALODLM_EPI_STORE_F32, nullptr, 1, &count, 0, st);
        ALODLM_CHECK_LAUNCH("linear_loss_logits");
        return ALODLM_OK;
      }
    return alodlm_gemm(deep_hidden, deep_ldh, 1, w, ld, 1, out, to, nullptr, 0, R, n, p.deep, 1.f,
                       p.half ? ALODLM_EPI_STORE_F32 : ALODLM_EPI_STORE, dtype, gemm(), st);
  }
};

template <typename T>
int forward(Call<T>& a, const KnownRows& k, const GivenRows& given, float c, int reduction, float* loss,
            float* kept) {
  const Plan& p = a.p;
  Part* part = reinterpret_cast<Part*>(a.ws + p.part);
  a.copy_hidden();
  // whole logits in memory need no prepared tokens
  const bool whole = !p.tiles && p.pieces == 1;
  if (!whole) known_prepare_launch(k, given, a.R, a.st);
  float* logits = p.keep ? kept : a.ws + p.logits;
  int64_t ld = 0;
  for (int64_t first = 0, i = 0; first < a.V; first += p.piece, ++i) {
    const int64_t n = a.V - first < p.piece ? a.V - first : p.piece;
    if (p.tiles) {
      if constexpr (sizeof(T) == 2) {
        const SumHooks hooks = {k, c, part + i * p.chunks * a.R, first};
        int64_t ldw;
        const T* w = a.piece_weight(first, n, ldw);
        tiles_launch(a.deep_hidden, a.deep_ldh, w, ldw, a.R, n, p.deep, nullptr, 0, hooks, a.st);
      }
    } else {
      float* to = p.keep ? logits + first : logits;
      LL_CALL(a.logits(first, n, to));
      ld = a.logits_ld(n);
      row_stats_launch<float>(to, ld, a.R, n, first, k, given, !whole, c, p.chunks,
                              part + i * p.chunks * a.R, a.st);
    }
    ALODLM_CHECK_LAUNCH("linear_loss");
  }
  known_finish_launch<float>(k, given, whole ? logits : nullptr, ld, part, p.sum_parts, a.R, c, p.tiles,
                             reduction, loss, a.st);
  ALODLM_CHECK_LAUNCH("linear_loss");
  return ALODLM_OK;
}

template <typename T>
int backward(Call<T>& a, const KnownRows& k, float c, const Upstream& up, const float* kept, T* d_hidden,
             T* d_weight) {
  const Plan& p = a.p;
  constexpr bool half = sizeof(T) == 2;
  const int64_t R = a.R, V = a.V, H = a.H, d_rows = p.parts * R;
  T* D = reinterpret_cast<T*>(a.ws + p.D);
  float* sums = a.ws + p.sums;
  int64_t planes = 0, rest = 0;
  const T* rest_weight = nullptr;
  a.copy_hidden();
  for (int64_t first = 0; first < V; first += p.piece) {
    const int64_t n = V - first < p.piece ? V - first : p.piece, padded = up_to(n, 32);
    const bool last = first + n == V;
    // D of the piece; zeros from column n to `columns`
    const bool own = half || p.keep;  // D has a place of its own
    const int64_t ldd = own ? p.piece : a.logits_ld(n), columns = own ? padded : ldd;
    if (p.tiles) {
      if constexpr (half) {
        const GradHooks hooks = {k, c, up, first, p.deep_rows, columns};
        int64_t ldw;
        const T* w = a.piece_weight(first, n, ldw);
        tiles_launch(a.deep_hidden, a.deep_ldh, w, ldw, R, n, p.deep, D, p.piece, hooks, a.st);
      }
    } else {
      const float* logits = p.keep ? kept + first : a.ws + p.logits;
      if (!p.keep) LL_CALL(a.logits(first, n, a.ws + p.logits));
      if constexpr (!half)
        if (p.few) {
          const T* w = a.weight + first * a.ldw;
          few_grads_launch(logits, a.logits_ld(n), R, n, first, k, c, up, D, few_f32_pad(R), a.st);
          if (d_hidden) {
            few_f32_hidden(D, w, a.ldw, R, n, H, sums + planes * R * H, a.st);
            planes += few_f32_planes(n, H);
            if (last) finish_product<T>(sums, planes, R, H, up, nullptr, 0, nullptr, 0, 0, 1, d_hidden, a.st);
          }
          if (d_weight) few_f32_weight(D, a.hidden, a.ldh, R, n, H, d_weight + first * H, a.st);
          ALODLM_CHECK_LAUNCH("linear_loss_bwd");
          continue;
        }
      row_grads_launch<float, T>(logits, a.logits_ld(n), R, n, first, k, c, up, D, ldd, p.deep_rows, columns,
                                 a.st, p.parts > 1);
    }
    ALODLM_CHECK_LAUNCH("linear_loss_bwd");
    const T* w = a.weight + first * a.ldw;
    if (d_hidden) {
      const int64_t take = n / 32 * 32;
      rest = n - take;  // 0 but in the last piece
      rest_weight = w + take * a.ldw;
      if (take) {
        const Split s = last ? p.last_split : p.hidden_split;
        const bool more = p.add && planes > 0;
        float* to = p.direct ? reinterpret_cast<float*>(d_hidden) : sums + (more ? 0 : planes) * d_rows * H;
        int64_t count = 1;
        if constexpr (half) {
          if (s.large)
            gemm_dl_launch(D, ldd, 1, w, a.ldw, 0, to, H, nullptr, 0, d_rows, H, take, 1.f,
                           more ? ALODLM_EPI_ACCUM : ALODLM_EPI_STORE_F32, to, s.planes, &count, more, a.st);
          else
            count = gemm_mid_planes(D, ldd, 1, w, a.ldw, d_rows, H, take, s.planes, to, more, a.st);
        } else {
          LL_CALL(alodlm_gemm(D, ldd, 1, w, a.ldw, 0, to, H, nullptr, 0, d_rows, H, take, 1.f,
                              more ? ALODLM_EPI_ACCUM : ALODLM_EPI_STORE, a.dtype, a.gemm(), a.st));
        }
        if (!more) planes += count;
        ALODLM_CHECK_LAUNCH("linear_loss_bwd");
      }
      if (last && !p.direct)
        // (a plane has the parts' rows one after the other: planes of their own)
        finish_product<T>(sums, p.parts * planes, R, H, up, D + take, ldd, rest_weight, a.ldw, (int)rest, p.parts,
                          d_hidden, a.st);
    }
    if (d_weight) {
      T* to = d_weight + first * H;  // (up to 31 rows behind the last: the caller's room)
      if constexpr (half) {
        float* rows = a.ws + p.rows;
        const Split s = split_product(padded, H, d_rows, true, true, false);
        if (s.large) {
          const int64_t tiles = ceil_div(padded, TB) * ceil_div(H, TB);
          gemm_dl_kernel<false, false, ALODLM_EPI_STORE, 4, true, false, ScaleHooks>
              <<<dim3((unsigned)tiles, 1), 256, 0, a.st>>>(D, ldd, a.deep_hidden, a.deep_ldh, to, H, nullptr, 0,
                                                           padded, H, p.deep_rows, 1.f, p.deep_rows, nullptr, 0,
                                                           KSegs{}, ScaleHooks{up});
        } else {
          const int64_t count =
              gemm_mid_planes(D, ldd, 0, a.deep_hidden, a.deep_ldh, padded, H, d_rows, s.planes, rows, false, a.st);
          finish_product<T>(rows, count, padded, H, up, nullptr, 0, nullptr, 0, 0, 1, to, a.st);
        }
      } else {
        LL_CALL(alodlm_gemm(D, ldd, 0, a.hidden, a.ldh, 0, to, H, nullptr, 0, up_to(n, 8), H, R, 1.f, ALODLM_EPI_STORE,
                            a.dtype, a.gemm(), a.st));
      }
      ALODLM_CHECK_LAUNCH("linear_loss_bwd");
    }
  }
  ALODLM_CHECK_LAUNCH("linear_loss_bwd");
  return ALODLM_OK;
}

}  // namespace

extern "C" int64_t alodlm_linear_loss_kept(int64_t rows, int64_t vocab, int64_t width, int dtype) {
  if (rows < 1 || vocab < 1 || width < 1) return 0;
  return make_plan(rows, vocab, width, dtype, true, false, false, false).keep ? rows * up_to(vocab, 8) : 0;
}

extern "C" int64_t alodlm_linear_loss_workspace(int64_t rows, int64_t vocab, int64_t width, int keep,
                                                int dtype) {
  if (rows < 1 || vocab < 1 || width < 1) return 0;
  return make_plan(rows, vocab, width, dtype, keep != 0, false, false, false).total;
}

extern "C" int64_t alodlm_linear_loss_bwd_workspace(int64_t rows, int64_t vocab, int64_t width, int keep,
                                                    int d_hidden, int d_weight, int dtype) {
  if (rows < 1 || vocab < 1 || width < 1) return 0;
  return make_plan(rows, vocab, width, dtype, keep != 0, true, d_hidden != 0, d_weight != 0).total;
}

extern "C" int alodlm_linear_loss(const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                                  const int64_t* targets, const int64_t* ids, const float* log_q,
                                  int64_t rows, int64_t vocab, int64_t width, int64_t known,
                                  float inv_temperature, int64_t ignore, int rest, int reduction,
                                  float* loss, float* state, float* kept, float* workspace, int dtype,
                                  void* stream) {
  LL_CALL(check_linear("linear_loss", hidden, ldh, weight, ldw, rows, vocab, width, known, inv_temperature,
                       reduction, dtype));
  ALODLM_CHECK_ARG(!targets || (known == 1 && !rest), "linear_loss: a target is one known token");
  if (rows == 0 && reduction == VL_EACH) return ALODLM_OK;
  ALODLM_CHECK_ARG(loss && state && (rows == 0 || (workspace && (targets || (ids && log_q)))),
                   "linear_loss: the call lacks an array");
  ALODLM_CHECK_ARG((((uintptr_t)workspace | (uintptr_t)kept) & 15) == 0, "linear_loss: workspace not 16-byte aligned");
  const hipStream_t st = as_stream(stream);
  const KnownRows k = known_rows(state, rows, known);
  const GivenRows given = {targets, ids, log_q, ignore, (int)known, (int)vocab, rest != 0};
  const float c = inv_temperature * VL_LOG2E;
  if (rows == 0) {
    known_finish_launch<float>(k, given, nullptr, 0, nullptr, 0, 0, c, false, reduction, loss, st);
    ALODLM_CHECK_LAUNCH("linear_loss");
    return ALODLM_OK;
  }
  const Plan p = make_plan(rows, vocab, width, dtype, kept != nullptr, false, false, false);
  ALODLM_CHECK_ARG(!kept || p.keep, "linear_loss: logits of this size are not kept");
  ALODLM_CHECK_ARG(p.tiles || rows * p.chunks < VL_MOST_GROUPS, "linear_loss: too many rows in one call");
  if (dtype == ALODLM_BF16) {
    Call<bf16_t> a = {p, (const bf16_t*)hidden, ldh, (const bf16_t*)weight, ldw, rows, vocab, width, workspace,
                      dtype, st};
    return forward(a, k, given, c, reduction, loss, kept);
  }
  Call<float> a = {p, (const float*)hidden, ldh, (const float*)weight, ldw, rows, vocab, width, workspace, dtype, st};
  return forward(a, k, given, c, reduction, loss, kept);
}

extern "C" int alodlm_linear_loss_bwd(const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                                      const float* state, const float* kept, const float* d_loss, int64_t rows,
                                      int64_t vocab, int64_t width, int64_t known, float inv_temperature,
                                      int reduction, void* d_hidden, void* d_weight, float* workspace, int dtype,
                                      void* stream) {
  LL_CALL(check_linear("linear_loss_bwd", hidden, ldh, weight, ldw, rows, vocab, width, known,
                       inv_temperature, reduction, dtype));
  if (rows == 0 || (!d_hidden && !d_weight)) return ALODLM_OK;
  ALODLM_CHECK_ARG(state && d_loss && workspace, "linear_loss_bwd: the call lacks an array");
  ALODLM_CHECK_ARG((((uintptr_t)workspace | (uintptr_t)kept | (uintptr_t)d_hidden | (uintptr_t)d_weight) & 15) == 0,
                   "linear_loss_bwd: an array is not 16-byte aligned");
  const hipStream_t st = as_stream(stream);
  const KnownRows k = known_rows(const_cast<float*>(state), rows, known);  // read only
  const float c = inv_temperature * VL_LOG2E;
  const Plan p = make_plan(rows, vocab, width, dtype, kept != nullptr, true, d_hidden != nullptr, d_weight != nullptr);
  ALODLM_CHECK_ARG(!kept || p.keep, "linear_loss_bwd: logits of this size are not kept");
  const Upstream up = {k.call, d_loss, reduction, p.half, inv_temperature};
  if (dtype == ALODLM_BF16) {
    Call<bf16_t> a = {p, (const bf16_t*)hidden, ldh, (const bf16_t*)weight, ldw, rows, vocab, width, workspace,
                      dtype, st};
    return backward(a, k, c, up, kept, (bf16_t*)d_hidden, (bf16_t*)d_weight);
  }
  Call<float> a = {p, (const float*)hidden, ldh, (const float*)weight, ldw, rows, vocab, width, workspace, dtype, st};
  return backward(a, k, c, up, kept, (float*)d_hidden, (float*)d_weight);
}
