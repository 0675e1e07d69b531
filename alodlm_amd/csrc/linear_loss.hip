// Losses over the vocabulary from hidden states [rows, width] and the output projection
// [vocab, width], without the logits, and their gradients (vocab_loss.h has the
// mathematics).
//
// Forward: the logits leave the matrix cores tile by tile (256 rows x 256 tokens, the
// two-stage kernel of gemm_dl_tile.h) and are summed where they are, in the epilogue: a
// tile leaves one part (largest logit, sum) a row.  Nothing of the size of the logits is
// written.  Backward: a piece of the vocabulary at a time, the tiles are computed once more
// and leave the piece's gradient D = dloss / dlogits in bf16, from which two products give
// its share of d_hidden (D W, summed in float32 over the pieces) and its rows of d_weight
// (D^T hidden, written once).  Four products of 2 rows vocab width operations in all, of
// which the second computation of the logits is what not keeping them costs.
//
// D is rounded to bf16 (half a step, 2^-9 of a value at most), as a bf16 model's logits'
// gradient is anywhere: it is an operand of the bf16 matrix cores.  Float32 models, and
// widths that are no multiple of 64, take a piece's logits in float32 through memory.
#include "gemm_dl_tile.h"
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
      const int* ids = k.ids + row * k.known;
#pragma unroll 8
      for (int i = 0; i < k.known; ++i) {
        const int at = ids[i] - (int)token0;
        before += at < 0;
        if ((unsigned)at < (unsigned)TB) bits[at >> 5] |= 1u << (at & 31);
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

// Forward tiles: parts of the rows' sums, and the known tokens' logits.
struct SumHooks {
  static constexpr bool Epilogue = true;
  static constexpr int EXTRA_LDS = TileMarks::BYTES + 2 * TB * (int)sizeof(Part);
  KnownRows k;
  float c;
  Part* part;  // [tiles][rows]

  __device__ __forceinline__ void before(char* extra, int64_t M, int64_t m0, int64_t n0) const {
    TileMarks::fill(extra, k, m0 + threadIdx.x, M, n0);
  }
  template <typename Quad>
  __device__ __forceinline__ void after(char*, char* extra, Quad quad, void*, int64_t, int64_t M,
                                        int64_t N, int64_t m0, int64_t n0) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = wave & 1, g = lane >> 4;
    Part* red = reinterpret_cast<Part*>(extra + TileMarks::BYTES);
    const bool edge = n0 + TB > N;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v[8][4];
      int row = 0, col = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        quad(8 * i + j, row, col, v[j]);
        if (edge)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = n0 + col + e < N ? v[j][e] : -INFINITY;
      }
      const uint4 b = TileMarks::half(extra, row, wn);
      if (__any((b.x | b.y | b.z | b.w) != 0)) {
        // this lane's 32 columns, a bit each
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mine |= TileMarks::nibble(b, j, g) << (4 * j);
        for (uint32_t left = mine; left; left &= left - 1) {
          const int at = __builtin_ctz(left);
          float z = v[0][0];
#pragma unroll
          for (int n = 1; n < 32; ++n) z = at == n ? v[n >> 2][n & 3] : z;
          const int tile_col = wn * 128 + 16 * (at >> 2) + 4 * g + (at & 3);
          k.logit[(m0 + row) * k.known + TileMarks::place(extra, row, tile_col)] = z;
        }
#pragma unroll
        for (int n = 0; n < 32; ++n) v[n >> 2][n & 3] = mine >> n & 1 ? -INFINITY : v[n >> 2][n & 3];
      }
      float m = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        m = fmaxf(m, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
      m = quad_max(m);
      const float base = m == -INFINITY ? 0.f : m;
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += __builtin_amdgcn_exp2f((v[j][e] - base) * c);
      const float sum = quad_sum((s[0] + s[1]) + (s[2] + s[3]));
      if (g == 0) red[wn * TB + row] = {m, sum};
    }
    __syncthreads();
    const int t = threadIdx.x;
    if (m0 + t < M) part[n0 / TB * M + m0 + t] = part_join(red[t], red[TB + t], c);
  }
};

// Backward tiles: D of a piece of the vocabulary, bf16, zero in the padding.
struct GradHooks {
  static constexpr bool Epilogue = true;
  static constexpr int EXTRA_LDS = TileMarks::BYTES + TB * 16;
  KnownRows k;
  float c, inv_t;
  const float* d_loss;
  int reduction;
  int64_t first;          // the piece's first token
  int64_t rows, columns;  // of D, padding included

  __device__ __forceinline__ void before(char* extra, int64_t M, int64_t m0, int64_t n0) const {
    const int64_t row = m0 + threadIdx.x;
    float4 r = make_float4(0.f, 1e30f, 0.f, 0.f);  // 2^-1e30: nothing
    if (row < M) {
      const float* info = k.info + 8 * row;
      const float g = row_upstream(k.call, d_loss, reduction, row, inv_t);
      const float f = info[RI_FACTOR];
      r.z = g;
      if (g != 0.f && f != 0.f) {
        r.x = g * f;
        r.y = fmaf(info[RI_M], c, info[RI_LOG]);
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
    const bool edge = n0 + TB > N;
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
      if (edge)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = n0 + col + e < N ? v[e] : 0.f;
    };
    tile_epilogue<ALODLM_EPI_STORE, 256, false>(lds, grad, D, ldd, nullptr, 0, rows, columns, m0, n0,
                                                1.f, nullptr, 0);
    // the known tokens' own, behind the tile's stores
    __syncthreads();
    const int64_t row = m0 + threadIdx.x;
    if (row >= M) return;
    const float up = consts[threadIdx.x].z;
    const uint32_t* bits = reinterpret_cast<const uint32_t*>(extra) + 8 * threadIdx.x;
    const float* own = k.weight + row * k.known + TileMarks::before(extra, threadIdx.x);
    for (int w = 0; w < 8; ++w)
      for (uint32_t b = bits[w]; b; b &= b - 1, ++own)
        reinterpret_cast<bf16_t*>(D)[row * ldd + n0 + 32 * w + __builtin_ctz(b)] =
            float_to_bf16(up == 0.f ? 0.f : up * *own);
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

// dst [padded, width] = src's first `rows` rows, zeros behind them.
template <typename T>
__global__ void __launch_bounds__(256)
copy_rows_kernel(const T* __restrict__ src, int64_t lds, int64_t rows, T* __restrict__ dst, int64_t ldd,
                 int64_t width) {
  const int64_t row = blockIdx.y, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at < width) dst[row * ldd + at] = row < rows ? src[row * lds + at] : T(0);
}
template <typename T>
void copy_rows(const T* src, int64_t lds, int64_t rows, T* dst, int64_t ldd, int64_t padded, int64_t width,
               hipStream_t st) {
  for (int64_t r = 0; r < padded; r += 65535) {  // rows of a launch
    const int64_t n = padded - r < 65535 ? padded - r : 65535;
    copy_rows_kernel<T><<<dim3(ceil_div_u(width, 256), (unsigned)n), 256, 0, st>>>(
        src + r * lds, lds, rows - r, dst + r * ldd, ldd, width);
  }
}

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Bytes of a piece: what is held of the vocabulary at a time.
constexpr int64_t PIECE_BYTES = 512ll << 20;

struct Plan {
  bool tiles;             // logits stay on chip
  int64_t piece, pieces;  // tokens of a piece (a multiple of 256), pieces
  int64_t parts, part_chunks;
  int64_t padded_rows, contributions;
  bool pad, accumulate;
  // workspace, in floats
  int64_t part, logits, D, hidden, sums, tail, d_tail, gemm, total;
};

Plan make_plan(int64_t R, int64_t V, int64_t H, int dtype, bool backward, bool d_hidden, bool d_weight) {
  Plan p = {};
  const int64_t es = dtype == ALODLM_BF16 ? 2 : 4;
  p.tiles = dtype == ALODLM_BF16 && H % 64 == 0;
  p.padded_rows = dtype == ALODLM_BF16 ? up(R, 32) : R;
  const int64_t token = p.padded_rows * (p.tiles ? 2 : 4);  // bytes
  const int64_t most = PIECE_BYTES / token / 256 * 256 > 256 ? PIECE_BYTES / token / 256 * 256 : 256;
  p.pieces = (V + most - 1) / most;
  p.piece = up((V + p.pieces - 1) / p.pieces, 256);
  p.pieces = (V + p.piece - 1) / p.piece;
  int64_t at = 0;
  auto room = [&](int64_t floats) {
    const int64_t here = at;
    at += up(floats, 64);
    return here;
  };
  int64_t gemm = 0;
  auto product = [&](int64_t M, int64_t N, int64_t K, int epi) {
    if (M < 1 || K < 1) return;
    const int64_t n = alodlm_gemm_workspace(M, N, K, epi, dtype);
    gemm = n > gemm ? n : gemm;
  };
  const int store_f32 = dtype == ALODLM_F32 ? ALODLM_EPI_STORE : ALODLM_EPI_STORE_F32;
  const int64_t last = V - (p.pieces - 1) * p.piece;
  if (!p.tiles) {
    p.logits = room(R * p.piece);
    if (p.pieces > 1) product(R, p.piece, H, store_f32);
    product(R, last, H, store_f32);
  }
  if (!backward) {
    p.part_chunks = p.tiles ? 0 : row_stats_chunks(R, p.piece);
    p.parts = p.tiles ? (V + TB - 1) / TB : p.part_chunks * p.pieces;
    p.part = room(2 * R * p.parts);
  } else {
    // float32: D takes the logits' place
    if (dtype == ALODLM_BF16) p.D = room((p.padded_rows * p.piece * es + 3) / 4);
    else p.D = p.logits;
    const int64_t whole = last / 32 * 32, rest = last - whole;
    p.pad = d_weight && p.padded_rows != R;
    if (p.pad) p.hidden = room((p.padded_rows * H * es + 3) / 4);
    if (rest) {
      p.tail = room((32 * H * es + 3) / 4);
      p.d_tail = room((32 * H * es + 3) / 4);
    }
    p.contributions = p.pieces - 1 + (whole > 0) + (rest > 0);
    p.accumulate = d_hidden && p.contributions > 1;
    if (p.accumulate && dtype == ALODLM_BF16) p.sums = room(R * H);
    if (d_hidden) {
      if (p.accumulate) {
        for (int epi : {store_f32, (int)ALODLM_EPI_ACCUM}) {
          if (p.pieces > 1) product(R, H, p.piece, epi);
          product(R, H, whole, epi);
          if (rest) product(R, H, 32, epi);
        }
      } else {
        product(R, H, whole ? whole : 32, ALODLM_EPI_STORE);
      }
    }
    if (d_weight) {
      if (p.pieces > 1) product(p.piece, H, p.padded_rows, ALODLM_EPI_STORE);
      product(whole, H, p.padded_rows, ALODLM_EPI_STORE);
      if (rest) product(32, H, p.padded_rows, ALODLM_EPI_STORE);
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
  if (R > 0 && dtype == ALODLM_BF16 && H % 64 == 0)
    ALODLM_CHECK_ARG((((uintptr_t)hidden | (uintptr_t)weight) & 15) == 0 && ldh % 8 == 0 && ldw % 8 == 0,
                     "%s: rows must be 16-byte aligned", what);
  return ALODLM_OK;
}

#define LL_CALL(expr)            \
  do {                           \
    const int _rc = (expr);      \
    if (_rc) return _rc;         \
  } while (0)

template <typename T>
int backward(const T* hidden, int64_t ldh, const T* weight, int64_t ldw, const KnownRows& k,
             const float* d_loss, int64_t R, int64_t V, int64_t H, float inv_t, int reduction,
             T* d_hidden, T* d_weight, float* ws, int dtype, hipStream_t st) {
  const Plan p = make_plan(R, V, H, dtype, true, d_hidden != nullptr, d_weight != nullptr);
  constexpr bool half = sizeof(T) == 2;
  const float c = inv_t * VL_LOG2E;
  float* gemm = p.gemm < 0 ? nullptr : ws + p.gemm;
  T* D = reinterpret_cast<T*>(ws + p.D);
  T* tail = reinterpret_cast<T*>(ws + p.tail);
  T* d_tail = reinterpret_cast<T*>(ws + p.d_tail);
  const T* h = hidden;
  int64_t ldp = ldh;
  if (p.pad) {
    T* padded = reinterpret_cast<T*>(ws + p.hidden);
    copy_rows(hidden, ldh, R, padded, H, p.padded_rows, H, st);
    h = padded;
    ldp = H;
  }
  float* sums = half ? ws + p.sums : reinterpret_cast<float*>(d_hidden);
  bool begun = false;
  auto to_hidden = [&](const T* d, const T* w, int64_t ld, int64_t tokens) {
    if (!p.accumulate)
      return alodlm_gemm(d, p.piece, 1, w, ld, 0, d_hidden, H, nullptr, 0, R, H, tokens, 1.f,
                         ALODLM_EPI_STORE, dtype, gemm, st);
    const int epi = begun ? ALODLM_EPI_ACCUM : half ? ALODLM_EPI_STORE_F32 : ALODLM_EPI_STORE;
    begun = true;
    return alodlm_gemm(d, p.piece, 1, w, ld, 0, sums, H, nullptr, 0, R, H, tokens, 1.f, epi, dtype, gemm,
                       st);
  };
  for (int64_t first = 0; first < V; first += p.piece) {
    const int64_t n = V - first < p.piece ? V - first : p.piece;
    const int64_t whole = n / 32 * 32, rest = n - whole, padded = up(n, 32);
    const T* w = weight + first * ldw;
    if (p.tiles) {
      if constexpr (half) {
        const GradHooks hooks = {k, c, inv_t, d_loss, reduction, first, p.padded_rows, padded};
        tiles_launch(hidden, ldh, w, ldw, R, n, H, D, p.piece, hooks, st);
      }
    } else {
      float* logits = ws + p.logits;
      LL_CALL(alodlm_gemm(hidden, ldh, 1, w, ldw, 1, logits, p.piece, nullptr, 0, R, n, H, 1.f,
                          half ? ALODLM_EPI_STORE_F32 : ALODLM_EPI_STORE, dtype, gemm, st));
      row_grads_launch<float, T>(logits, p.piece, R, n, first, k, c, inv_t, d_loss, reduction, D, p.piece,
                                 p.padded_rows, padded, st);
    }
    ALODLM_CHECK_LAUNCH("linear_loss_bwd");
    if (rest) copy_rows(w + whole * ldw, ldw, rest, tail, H, 32, H, st);
    if (d_hidden) {
      if (whole) LL_CALL(to_hidden(D, w, ldw, whole));
      if (rest) LL_CALL(to_hidden(D + whole, tail, H, 32));
    }
    if (d_weight) {
      if (whole)
        LL_CALL(alodlm_gemm(D, p.piece, 0, h, ldp, 0, d_weight + first * H, H, nullptr, 0, whole, H,
                            p.padded_rows, 1.f, ALODLM_EPI_STORE, dtype, gemm, st));
      if (rest) {
        LL_CALL(alodlm_gemm(D + whole, p.piece, 0, h, ldp, 0, d_tail, H, nullptr, 0, 32, H, p.padded_rows,
                            1.f, ALODLM_EPI_STORE, dtype, gemm, st));
        copy_rows(d_tail, H, rest, d_weight + (first + whole) * H, H, rest, H, st);
      }
    }
    ALODLM_CHECK_LAUNCH("linear_loss_bwd");
  }
  if (p.accumulate && half) LL_CALL(alodlm_cast_f32(sums, nullptr, d_hidden, R * H, dtype, st));
  return ALODLM_OK;
}

}  // namespace

extern "C" int64_t alodlm_linear_loss_workspace(int64_t rows, int64_t vocab, int64_t width, int dtype) {
  if (rows < 1 || vocab < 1 || width < 1) return 0;
  return make_plan(rows, vocab, width, dtype, false, false, false).total;
}

extern "C" int64_t alodlm_linear_loss_bwd_workspace(int64_t rows, int64_t vocab, int64_t width,
                                                    int d_hidden, int d_weight, int dtype) {
  if (rows < 1 || vocab < 1 || width < 1) return 0;
  return make_plan(rows, vocab, width, dtype, true, d_hidden != 0, d_weight != 0).total;
}

extern "C" int alodlm_linear_loss(const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                                  const int64_t* targets, const int64_t* ids, const float* log_q,
                                  int64_t rows, int64_t vocab, int64_t width, int64_t known,
                                  float inv_temperature, int64_t ignore, int rest, int reduction,
                                  float* loss, float* state, float* workspace, int dtype, void* stream) {
  LL_CALL(check_linear("linear_loss", hidden, ldh, weight, ldw, rows, vocab, width, known, inv_temperature,
                       reduction, dtype));
  ALODLM_CHECK_ARG(!targets || (known == 1 && !rest), "linear_loss: a target is one known token");
  if (rows == 0 && reduction == VL_NONE_REDUCED) return ALODLM_OK;
  ALODLM_CHECK_ARG(loss && state && (rows == 0 || (workspace && (targets || (ids && log_q)))),
                   "linear_loss: the call lacks an array");
  ALODLM_CHECK_ARG((uintptr_t)workspace % 16 == 0, "linear_loss: workspace not 16-byte aligned");
  const hipStream_t st = as_stream(stream);
  const KnownRows k = known_rows(state, rows, known);
  if (rows == 0) {
    known_finish_launch(k, nullptr, 0, 0, 1.f, false, reduction, loss, st);
    ALODLM_CHECK_LAUNCH("linear_loss");
    return ALODLM_OK;
  }
  const Plan p = make_plan(rows, vocab, width, dtype, false, false, false);
  const float c = inv_temperature * VL_LOG2E;
  Part* part = reinterpret_cast<Part*>(workspace + p.part);
  known_prepare_launch(k, targets, ids, log_q, rows, vocab, ignore, rest != 0, st);
  if (p.tiles) {
    const SumHooks hooks = {k, c, part};
    tiles_launch((const bf16_t*)hidden, ldh, (const bf16_t*)weight, ldw, rows, vocab, width, nullptr, 0,
                 hooks, st);
  } else {
    float* logits = workspace + p.logits;
    const int64_t es = dtype == ALODLM_BF16 ? 2 : 4;
    ALODLM_CHECK_ARG(rows * p.part_chunks < (1ll << 31), "linear_loss: too many rows in one call");
    for (int64_t first = 0, i = 0; first < vocab; first += p.piece, ++i) {
      const int64_t n = vocab - first < p.piece ? vocab - first : p.piece;
      LL_CALL(alodlm_gemm(hidden, ldh, 1, (const char*)weight + first * ldw * es, ldw, 1, logits, p.piece,
                          nullptr, 0, rows, n, width, 1.f,
                          dtype == ALODLM_F32 ? ALODLM_EPI_STORE : ALODLM_EPI_STORE_F32, dtype,
                          p.gemm < 0 ? nullptr : workspace + p.gemm, stream));
      row_stats_launch<float>(logits, p.piece, rows, n, first, k, c, p.part_chunks,
                              part + i * p.part_chunks * rows, st);
    }
  }
  known_finish_launch(k, part, p.parts, rows, c, targets != nullptr, reduction, loss, st);
  ALODLM_CHECK_LAUNCH("linear_loss");
  return ALODLM_OK;
}

extern "C" int alodlm_linear_loss_bwd(const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                                      const float* state, const float* d_loss, int64_t rows, int64_t vocab,
                                      int64_t width, int64_t known, float inv_temperature, int reduction,
                                      void* d_hidden, void* d_weight, float* workspace, int dtype,
                                      void* stream) {
  LL_CALL(check_linear("linear_loss_bwd", hidden, ldh, weight, ldw, rows, vocab, width, known,
                       inv_temperature, reduction, dtype));
  if (rows == 0 || (!d_hidden && !d_weight)) return ALODLM_OK;
  ALODLM_CHECK_ARG(state && d_loss && workspace, "linear_loss_bwd: the call lacks an array");
  ALODLM_CHECK_ARG((uintptr_t)workspace % 16 == 0, "linear_loss_bwd: workspace not 16-byte aligned");
  const KnownRows k = known_rows(const_cast<float*>(state), rows, known);  // read only
  if (dtype == ALODLM_BF16)
    return backward((const bf16_t*)hidden, ldh, (const bf16_t*)weight, ldw, k, d_loss, rows, vocab, width,
                    inv_temperature, reduction, (bf16_t*)d_hidden, (bf16_t*)d_weight, workspace, dtype,
                    as_stream(stream));
  return backward((const float*)hidden, ldh, (const float*)weight, ldw, k, d_loss, rows, vocab, width,
                  inv_temperature, reduction, (float*)d_hidden, (float*)d_weight, workspace, dtype,
                  as_stream(stream));
}
