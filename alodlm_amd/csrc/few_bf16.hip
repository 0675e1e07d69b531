// Float logits of at most 64 bf16 rows over the vocabulary:  out[r][v] = hidden[r] . weight[v].
//
// Bound: the weight's bytes, and how memory is asked for them: every workgroup goes down the
// rows of its tokens, and the longer the piece of a row that it takes at a time, the better.
// 4 rows of width 2048 against 151936 tokens, the weight not in a cache: 152 us with 64-byte
// pieces (gemm_mid.hip's stages), 146 with 128, 138 with 256 and 133 with 512; 8 rows scored
// again and again 119 (5.2 TB/s).  So a stage is 16 KB of
// the weight: 64 KH deep for 128 / KH tokens, KH as large as the width divides and the hidden
// states' part of a stage stays below the weight's.  Two workgroups a compute unit, each with
// two or three stages under way, filled by direct loads to LDS; a wave has 16 or 32 tokens
// and all rows.  LDS layout and instruction as in gemm_dl_tile.h: blocks of eight rows,
// 64-byte halves, chunk ^ ((row / 2) % 4), free of bank conflicts; weight rows are the first
// operand, so a lane has 4 neighbouring tokens of one row.
//
// A workgroup has as many tokens as there are for each, in tiles one after the other: the
// loads of the next tile follow the last ones of a tile.
#include "few_bf16.h"
#include "lds_dma.h"

typedef __attribute__((__vector_size__(8 * sizeof(short)))) short bf16x8_t;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4_t;

namespace {

__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 3; }

// 16 bytes a lane from the wave-uniform origin plus the lane's offset into LDS slot lane of m0v.
__device__ __forceinline__ void load_slot(const char* origin, uint32_t off, uint32_t m0v) {
  asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(origin), "{m0}"(m0v) : "memory");
}

// MB: blocks of 16 rows; KH: 64-deep parts of a stage, which has 128 / KH tokens.
template <int MB, int KH>
__global__ void __launch_bounds__(KH == 4 ? 128 : 256, 2)
few_logits_kernel(const bf16_t* __restrict__ hidden, int64_t ldh, const bf16_t* __restrict__ weight,
                  int64_t ldw, int rows, int64_t tokens, int64_t share, int width, float* __restrict__ out,
                  int64_t ldo) {
  // 1 KB blocks of a stage: the weight's, then the hidden states'
  constexpr int TOKENS = 128 / KH, DEEP = 64 * KH, NW = KH == 4 ? 2 : 4;
  constexpr int WT = TOKENS / 16 / NW;  // 16-token blocks a wave
  constexpr int W_BLOCKS = TOKENS / 8 * KH, H_BLOCKS = 2 * MB * KH, STAGE = (W_BLOCKS + H_BLOCKS) * 1024;
  constexpr int STAGES = MB * KH >= 4 ? 3 : 4;  // two workgroups a compute unit
  // loads of a wave and stage (two blocks of hidden states: two waves load each, the same bytes)
  constexpr int W_LOADS = W_BLOCKS / NW, H_LOADS = H_BLOCKS < NW ? 1 : H_BLOCKS / NW, LOADS = W_LOADS + H_LOADS;
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * STAGE];
  int64_t first = (int64_t)blockIdx.x * share;  // of the tile that is computed
  const int64_t last = first + share < tokens ? first + share : tokens;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // rows past the operand re-read its last one: they feed outputs that are never stored
  uint32_t w_off[W_LOADS], h_off[H_LOADS], h_slot[H_LOADS];
  auto offset = [&](int block, int64_t ld, int64_t left) {
    const int row = 8 * (block / KH) + ((lane & 31) >> 2), chunk = (lane & 3) ^ swizzle(row);
    return (uint32_t)(((row < left ? row : left - 1) * ld + 64 * (block % KH) + 32 * (lane >> 5) + 8 * chunk) * 2);
  };
#pragma unroll
  for (int i = 0; i < W_LOADS; ++i) w_off[i] = offset(W_LOADS * wave + i, ldw, last - first);
#pragma unroll
  for (int i = 0; i < H_LOADS; ++i) {
    const int block = (wave + NW * i) % H_BLOCKS;
    h_off[i] = offset(block, ldh, rows);
    h_slot[i] = (uint32_t)(W_BLOCKS + block) * 1024u;
  }
  const char* w = reinterpret_cast<const char*>(weight + first * ldw);
  const char* h = reinterpret_cast<const char*>(hidden);
  const int steps = width / DEEP, tiles = (int)((last - first + TOKENS - 1) / TOKENS);
  const uint32_t base = lds_addr(lds);
  int64_t next = first;  // the tile that is loaded, and its step
  int loaded = 0;
  auto load = [&](int stage) {
    const uint32_t to = base + (uint32_t)(stage * STAGE);
#pragma unroll
    for (int i = 0; i < W_LOADS; ++i) load_slot(w, w_off[i], to + (uint32_t)(W_LOADS * wave + i) * 1024u);
#pragma unroll
    for (int i = 0; i < H_LOADS; ++i) load_slot(h, h_off[i], to + h_slot[i]);
    if (++loaded < steps) {
      w += 2 * DEEP;
      h += 2 * DEEP;
    } else if (next + TOKENS < last) {
      loaded = 0;
      next += TOKENS;
      w = reinterpret_cast<const char*>(weight + next * ldw);
      h = reinterpret_cast<const char*>(hidden);
      if (last - next < TOKENS)
#pragma unroll
        for (int i = 0; i < W_LOADS; ++i) w_off[i] = offset(W_LOADS * wave + i, ldw, last - next);
    }  // past the last step it is loaded again
  };
  // a fragment: row lane % 16 of a block pair, k 8 (lane / 16) .. + 7 of a 32-deep half
  auto at_row = [&](int row) {
    return (uint32_t)((row >> 3) * KH * 1024 + (row & 7) * 64 + (((lane >> 4) ^ swizzle(row)) << 4));
  };
  const uint32_t wf = at_row(16 * WT * wave + (lane & 15)), hf = W_BLOCKS * 1024u + at_row(lane & 15);
  f32x4_t acc[MB][WT];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < WT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  };
  // lane: row 16 i + lane % 16, tokens 16 (WT wave + j) + 4 (lane / 16) .. + 3
  auto store = [&]() {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < WT; ++j) {
        const int64_t row = 16 * i + (lane & 15), token = first + 16 * WT * wave + 16 * j + 4 * (lane >> 4);
        if (row >= rows) continue;
        float* o = out + row * ldo + token;
        if (token + 4 <= last)
          *reinterpret_cast<float4*>(o) = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        else
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (token + e < last) o[e] = acc[i][j][e];
      }
  };
  clear();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load(s);
  int cur = 0, step = 0;
  for (int t = 0; t < steps * tiles; ++t) {
    // step t has come once at most the STAGES - 2 newest are under way; every wave has read
    // step t - 1, whose stage is filled next
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 2) * LOADS) : "memory");
    load(cur == 0 ? STAGES - 1 : cur - 1);
    const char* p = lds + cur * STAGE;
    cur = cur + 1 < STAGES ? cur + 1 : 0;
#pragma unroll
    for (int ks = 0; ks < 2 * KH; ++ks) {
      bf16x8_t a[WT], b[MB];
      const uint32_t part = 1024 * (ks >> 1) + 512 * (ks & 1);
#pragma unroll
      for (int j = 0; j < WT; ++j) a[j] = *reinterpret_cast<const bf16x8_t*>(p + wf + 2048 * KH * j + part);
#pragma unroll
      for (int i = 0; i < MB; ++i) b[i] = *reinterpret_cast<const bf16x8_t*>(p + hf + 2048 * KH * i + part);
#pragma unroll
      for (int j = 0; j < WT; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j], b[i], acc[i][j], 0, 0, 0);
    }
    if (++step == steps) {
      store();
      clear();
      step = 0;
      first += TOKENS;
    }
  }
  // no load may land in LDS after the workgroup has gone
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

}  // namespace

void few_bf16_logits(const bf16_t* hidden, int64_t ldh, const bf16_t* weight, int64_t ldw, int64_t rows,
                     int64_t tokens, int64_t width, float* out, int64_t ldo, hipStream_t st) {
  const int kh = rows <= 16 && width % 256 == 0 ? 4 : width % 128 == 0 ? 2 : 1;
  const int64_t tiles = (tokens + 128 / kh - 1) / (128 / kh), most = 2 * device_cus();
  const int64_t units = (tokens + 15) / 16, groups = tiles < most ? tiles : most;
  const int64_t share = 16 * ((units + groups - 1) / groups);
  const unsigned grid = (unsigned)((tokens + share - 1) / share);
  auto launch = [&](auto kernel) {
    kernel<<<grid, kh == 4 ? 128 : 256, 0, st>>>(hidden, ldh, weight, ldw, (int)rows, tokens, share, (int)width, out,
                                               ldo);
  };
  if (rows <= 16) launch(kh == 4 ? few_logits_kernel<1, 4> : kh == 2 ? few_logits_kernel<1, 2> : few_logits_kernel<1, 1>);
  else if (rows <= 32) launch(kh == 2 ? few_logits_kernel<2, 2> : few_logits_kernel<2, 1>);
  else launch(few_logits_kernel<4, 1>);
}
