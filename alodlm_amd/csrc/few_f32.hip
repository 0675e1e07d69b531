// Float32 products of at most 32 rows with a weight over the vocabulary:
//   d_hidden[r][h] = sum_v D[v][r] weight[v][h],   d_weight[v][h] = sum_r D[v][r] hidden[r][h].
//
// Bound: the weight's bytes, read or written once.  A thread owns four neighbouring columns,
// so a wave moves a whole KB of a weight row at a time, and keeps every row's sums (or hidden
// values) of them in registers; D lies token by token, its values are the same for all
// threads of a workgroup and come through scalar loads.  The float32 matrix cores would
// multiply 64-row tiles of which few rows are used: 5 rows of width 4096 against 151936
// tokens took 1.02 ms on them for d_hidden and 0.84 ms for d_weight.  Up to 32 rows, 128
// multiply-adds a KB and wave keep up with memory.
#include <type_traits>

#include "few_f32.h"

namespace {

constexpr int THREADS = 256, COLUMNS = 4 * THREADS;

// The rows in registers: a multiple of four, at most 32.
template <int ROWS>
__global__ void __launch_bounds__(THREADS)
few_hidden_kernel(const float* __restrict__ D, const float* __restrict__ weight, int64_t ldw, int rows,
                  int64_t tokens, int64_t per_part, int64_t width, float* __restrict__ planes) {
  const int64_t at = (int64_t)blockIdx.x * COLUMNS + 4 * threadIdx.x;
  const int64_t first = (int64_t)blockIdx.y * per_part;
  const int64_t last = first + per_part < tokens ? first + per_part : tokens;
  // (threads past the width take the last columns again and store nothing)
  const float* w = weight + (at < width ? at : width - 4);
  float4 acc[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) acc[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& x, int64_t v) {
    const float* d = D + v * ROWS;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float s = d[r];
      acc[r].x = fmaf(s, x.x, acc[r].x);
      acc[r].y = fmaf(s, x.y, acc[r].y);
      acc[r].z = fmaf(s, x.z, acc[r].z);
      acc[r].w = fmaf(s, x.w, acc[r].w);
    }
  };
  constexpr int AHEAD = 8;
  int64_t v = first;
  if (v + AHEAD <= last) {
    float4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = *reinterpret_cast<const float4*>(w + (v + i) * ldw);
    for (; v + 2 * AHEAD <= last; v += AHEAD) {
      float4 y[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) y[i] = *reinterpret_cast<const float4*>(w + (v + AHEAD + i) * ldw);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) add(x[i], v + i);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) x[i] = y[i];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) add(x[i], v + i);
    v += AHEAD;
  }
  for (; v < last; ++v) add(*reinterpret_cast<const float4*>(w + v * ldw), v);
  if (at >= width) return;
  float* out = planes + (int64_t)blockIdx.y * rows * width + at;
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
    if (r < rows) *reinterpret_cast<float4*>(out + r * width) = acc[r];
}

template <int ROWS>
__global__ void __launch_bounds__(THREADS)
few_weight_kernel(const float* __restrict__ D, const float* __restrict__ hidden, int64_t ldh, int rows,
                  int64_t tokens, int64_t per_part, int64_t width, float* __restrict__ out) {
  const int64_t at = (int64_t)blockIdx.x * COLUMNS + 4 * threadIdx.x;
  if (at >= width) return;
  const int64_t first = (int64_t)blockIdx.y * per_part;
  const int64_t last = first + per_part < tokens ? first + per_part : tokens;
  float4 h[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    h[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) h[r] = *reinterpret_cast<const float4*>(hidden + r * ldh + at);
  }
#pragma unroll 4
  for (int64_t v = first; v < last; ++v) {
    const float* d = D + v * ROWS;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float x = d[r];
      s.x = fmaf(x, h[r].x, s.x);
      s.y = fmaf(x, h[r].y, s.y);
      s.z = fmaf(x, h[r].z, s.z);
      s.w = fmaf(x, h[r].w, s.w);
    }
    __builtin_nontemporal_store(nt_f32x4_t{s.x, s.y, s.z, s.w}, reinterpret_cast<nt_f32x4_t*>(out + v * width + at));
  }
}

int64_t ceil_div(int64_t x, int64_t by) { return (x + by - 1) / by; }

// Parts of the tokens: four workgroups a compute unit, 64 tokens at least.
int64_t token_parts(int64_t tokens, int64_t width) {
  const int64_t want = ceil_div(1024, ceil_div(width, COLUMNS)), most = tokens / 64 > 1 ? tokens / 64 : 1;
  const int64_t n = want < most ? want : most;
  return ceil_div(tokens, ceil_div(tokens, n));
}

template <typename F> void with_rows(int64_t rows, F f) {
  switch (few_f32_pad(rows)) {
    case 4: f(std::integral_constant<int, 4>()); break;
    case 8: f(std::integral_constant<int, 8>()); break;
    case 16: f(std::integral_constant<int, 16>()); break;
    case 24: f(std::integral_constant<int, 24>()); break;
    default: f(std::integral_constant<int, 32>());
  }
}

}  // namespace

int64_t few_f32_pad(int64_t rows) { return rows <= 4 ? 4 : (rows + 7) / 8 * 8; }

int64_t few_f32_planes(int64_t tokens, int64_t width) { return token_parts(tokens, width); }

void few_f32_hidden(const float* D, const float* weight, int64_t ldw, int64_t rows, int64_t tokens,
                    int64_t width, float* planes, hipStream_t st) {
  const int64_t parts = token_parts(tokens, width);
  const dim3 grid((unsigned)ceil_div(width, COLUMNS), (unsigned)parts);
  with_rows(rows, [&](auto n) {
    few_hidden_kernel<decltype(n)::value><<<grid, THREADS, 0, st>>>(D, weight, ldw, (int)rows, tokens,
                                                                    ceil_div(tokens, parts), width, planes);
  });
}

void few_f32_weight(const float* D, const float* hidden, int64_t ldh, int64_t rows, int64_t tokens,
                    int64_t width, float* out, hipStream_t st) {
  const int64_t parts = token_parts(tokens, width);
  const dim3 grid((unsigned)ceil_div(width, COLUMNS), (unsigned)parts);
  with_rows(rows, [&](auto n) {
    few_weight_kernel<decltype(n)::value><<<grid, THREADS, 0, st>>>(D, hidden, ldh, (int)rows, tokens,
                                                                    ceil_div(tokens, parts), width, out);
  });
}
