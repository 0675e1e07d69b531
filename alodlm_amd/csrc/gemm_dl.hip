// bf16 GEMM with direct global->LDS staging for the large products of the
// step:  C[m, n] = alpha * sum_k A(m, k) B(n, k), operands k-contiguous or
// m/n-contiguous in any combination.
//
// 256x256 block tile, 32-deep k stages in a ring of STAGES LDS buffers.  Each
// stage is filled by global_load_lds_dwordx4 (lane i of an instruction
// writes the i-th 16-byte slot after the instruction's LDS base), issued
// STAGES-1 tiles ahead; there are no staging registers and no VALU copies.
// Loads address a wave-uniform tile origin plus a 32-bit lane offset; rows and
// columns past the operand's edge are clamped to its last valid row / chunk.
//
// Waves: 4 (2 x 2, 128x128 each, one per SIMD), v_mfma_f32_16x16x32_bf16 with
// the operands swapped (B rows as the MFMA's A operand), so each lane owns 4
// consecutive output columns of one row.  One 32-deep stage is one k step of
// 8 x 8 MFMAs per wave (256 accumulation registers).  The step is power-bound
// on MI355X (the chip holds its 1400 W limit by lowering the clock): with the
// same LDS bytes and direct loads, the 16x16x32 instruction runs the products
// at a 10-15 % higher clock than v_mfma_f32_32x32x16_bf16 (measured per
// kernel from GRBM_GUI_ACTIVE over its duration), which outweighs the few
// percent more cycles it takes; the 1.7B step ran 2.2 % faster with it.
//
// LDS layouts (16-byte-chunk XOR swizzles, chosen by the source chunk of each
// direct-load lane; measured free of bank conflicts for these fragment reads):
//  * k-contiguous operand: [256 rows][32 k], 64-byte rows,
//    chunk' = chunk ^ ((row >> 1) & 3); a fragment read takes rows
//    r + lane % 16, chunk lane / 16 (ds_read_b128);
//  * m/n-contiguous operand: [32 k][256], 512-byte rows,
//    chunk' = chunk ^ (4*(k & 3) ^ 2*((k >> 3) & 1)); fragments come from
//    ds_read_b64_tr_b16 (per 16 lanes: 4 k rows x 16 columns, result lane i =
//    column i), k rows 8 (lane / 16) + 0..3 and + 4..7.
// Both give the MFMA operand "row i = lane % 16, k = 8*(lane / 16) + 0..7".
//
// With one wave per SIMD every instruction of the loop takes an issue slot
// beside the MFMAs, and a 16x16x32 MFMA leaves room for about three: the loop
// carries no address arithmetic (the tile loop is unrolled over the STAGES
// stages of the ring, every fragment read is a per-lane base register plus an
// immediate, every direct load sets M0 with one scalar add from a per-wave
// base, the two tile origins advance by one 64-bit add per stage), and the
// memory instructions are spread one group per MFMA: with the 8 direct loads
// bunched into the first 8 MFMAs and 3 LDS reads after some, the same kernel
// ran 12 % slower.
//
// Workgroup -> tile order: consecutive workgroups land on different XCDs, so
// the tile sequence is dealt out in contiguous chunks per XCD, then swept in
// groups of 3 tile rows (down a group, then across).
#include "common.h"
#include "gemm_dl.h"
#include "gemm_dl_tile.h"
#include "lds_dma.h"

// The direct-load kernel needs whole 32-deep k stages, 16-byte-aligned rows and,
// for m/n-contiguous operands, dimensions in whole 16-byte chunks.
bool gemm_dl_eligible(int64_t lda, int a_kmajor, int64_t ldb, int b_kmajor, int64_t M, int64_t N,
                      int64_t K) {
  if (M < TB || N < TB || K < KMIN || K % KMIN != 0) return false;
  if (lda % 8 != 0 || ldb % 8 != 0) return false;
  if (!a_kmajor && M % 8 != 0) return false;
  if (!b_kmajor && N % 8 != 0) return false;
  return true;
}

// Splits of K for ALODLM_EPI_ACCUM products with few output tiles: the
// fewest (powers of two up to 8, each split keeping >= 32 k stages) whose
// rounds of 256 workgroups (one per CU) cost the least per unit of work.
// Splits that only add rounds cost float partials and their reduction: the
// 1.7B step's dW of the QKV and O projections take 2 and 4 splits (one
// round), 22 us faster each than at 4 and 8.
int64_t gemm_dl_splits(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ((M + TB - 1) / TB) * ((N + TB - 1) / TB);
  const int64_t ksteps = K / KMIN;
  const int64_t cus = 256;
  auto cost = [&](int64_t s) { return (double)((tiles * s + cus - 1) / cus) / (double)s; };
  int64_t best = 1;
  for (int64_t s = 2; s <= 8 && ksteps / s >= 32; s *= 2)
    if (cost(s) < 0.98 * cost(best)) best = s;
  return best;
}

// Splits of a bf16-output (STORE) product: the fewest that bring the rounds
// of 256 workgroups (one per CU) within 8 % of the split-free work, so that a
// long-K product with few output tiles (the LM head's dX) does not leave CUs
// idle in its last round; only K >= 16384 (the partials' traffic is then
// small next to the product) and every split keeps >= 2048 of K.  1 when the
// tiles already fill the rounds.
int64_t gemm_dl_store_splits(int64_t M, int64_t N, int64_t K) {
  if (K < 16384) return 1;
  const int64_t tiles = ((M + TB - 1) / TB) * ((N + TB - 1) / TB);
  const int64_t cus = 256;
  auto cost = [&](int64_t s) { return (double)((tiles * s + cus - 1) / cus) / (double)s; };
  const double ideal = (double)tiles / (double)cus;
  if (cost(1) <= 1.08 * ideal) return 1;
  int64_t best = 1;
  for (int64_t s = 2; s <= 8 && K / s >= 2048; ++s)
    if (cost(s) < cost(best) && cost(best) - cost(s) > 0.02 * cost(1)) best = s;
  return best;
}

template <bool AK, bool BK, bool SCALE>
static void launch_scaled(const bf16_t* A, int64_t lda, const bf16_t* B, int64_t ldb, void* C,
                          int64_t ldc, const bf16_t* R, int64_t ldr, int64_t M, int64_t N,
                          int64_t K, float alpha, int epi, float* part, int64_t kps,
                          int64_t nsplit, int first_into_c, const KSegs* segs, hipStream_t st) {
  const int64_t tiles = ((M + TB - 1) / TB) * ((N + TB - 1) / TB);
  dim3 grid((unsigned)tiles, (unsigned)nsplit);
  // K over separate segments: the dW layout with float outputs only
  if constexpr (!AK && !BK && SCALE) {
    if (segs != nullptr) {
      if (epi == ALODLM_EPI_STORE_F32 && part == nullptr)
        gemm_dl_kernel<false, false, ALODLM_EPI_STORE_F32, 4, true, true><<<grid, 256, 0, st>>>(
            A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, *segs, NoHooks{});
      else
        gemm_dl_kernel<false, false, ALODLM_EPI_ACCUM, 4, true, true><<<grid, 256, 0, st>>>(
            A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, *segs, NoHooks{});
      return;
    }
  }
  // both operands k-contiguous: two 64-deep stages (128-byte row pieces per
  // direct load; 3-7 % faster than the 32-deep ring on every such product of
  // the step, and the same results: the k order of every sum is unchanged)
  if constexpr (AK && BK) {
    if (K % 64 == 0 && kps % 64 == 0) {
      if (epi == ALODLM_EPI_STORE)
        gemm_dl2_kernel<AK, BK, ALODLM_EPI_STORE, SCALE><<<grid, 256, 0, st>>>(
            A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, NoHooks{});
      else if (epi == ALODLM_EPI_RESIDUAL)  // (without the multiply it spills)
        gemm_dl2_kernel<AK, BK, ALODLM_EPI_RESIDUAL, true><<<grid, 256, 0, st>>>(
            A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, NoHooks{});
      else if constexpr (SCALE) {
        if (epi == ALODLM_EPI_STORE_F32 && part == nullptr)
          gemm_dl2_kernel<AK, BK, ALODLM_EPI_STORE_F32, true><<<grid, 256, 0, st>>>(
              A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, NoHooks{});
        else
          gemm_dl2_kernel<AK, BK, ALODLM_EPI_ACCUM, true><<<grid, 256, 0, st>>>(
              A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, NoHooks{});
      }
      return;
    }
  }
  // 4 waves, 32-deep k stages in a ring of 4 (128 KB of LDS)
  constexpr int ST = 4;
  if (epi == ALODLM_EPI_STORE)
    gemm_dl_kernel<AK, BK, ALODLM_EPI_STORE, ST, SCALE><<<grid, 256, 0, st>>>(
        A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, KSegs{}, NoHooks{});
  else if (epi == ALODLM_EPI_RESIDUAL)
    gemm_dl_kernel<AK, BK, ALODLM_EPI_RESIDUAL, ST, SCALE><<<grid, 256, 0, st>>>(
        A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, KSegs{}, NoHooks{});
  else if constexpr (SCALE) {
    if (epi == ALODLM_EPI_STORE_F32 && part == nullptr)
      gemm_dl_kernel<AK, BK, ALODLM_EPI_STORE_F32, ST, true><<<grid, 256, 0, st>>>(
          A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, KSegs{}, NoHooks{});
    else
      gemm_dl_kernel<AK, BK, ALODLM_EPI_ACCUM, ST, true><<<grid, 256, 0, st>>>(
          A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, kps, part, first_into_c, KSegs{}, NoHooks{});
  }
}

template <bool AK, bool BK>
static void launch_layout(const bf16_t* A, int64_t lda, const bf16_t* B, int64_t ldb, void* C,
                          int64_t ldc, const bf16_t* R, int64_t ldr, int64_t M, int64_t N,
                          int64_t K, float alpha, int epi, float* part, int64_t kps,
                          int64_t nsplit, int first_into_c, const KSegs* segs, hipStream_t st) {
  // the float-output epilogues keep the multiply: without it the compiler
  // hoists their loads of C and spills
  if (alpha == 1.f && (epi == ALODLM_EPI_STORE || epi == ALODLM_EPI_RESIDUAL))
    launch_scaled<AK, BK, false>(A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, epi, part, kps,
                                 nsplit, first_into_c, segs, st);
  else
    launch_scaled<AK, BK, true>(A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, epi, part, kps,
                                nsplit, first_into_c, segs, st);
}

// Launch the direct-load kernel; `part` (splits*M*N floats) is used when
// splits > 1 (float-output epilogues only), the caller reduces it.  With
// `first_into_c` (an accumulated float product) split 0 adds its result into
// C itself and its partial plane is left unwritten: the caller then adds
// planes 1.. only.
void gemm_dl_launch(const bf16_t* A, int64_t lda, int a_kmajor, const bf16_t* B, int64_t ldb,
                    int b_kmajor, void* C, int64_t ldc, const bf16_t* R, int64_t ldr, int64_t M,
                    int64_t N, int64_t K, float alpha, int epi, float* part, int64_t splits,
                    int64_t* nsplit_out, int first_into_c, hipStream_t st, const KSegs* segs) {
  int64_t kps = K;
  if (splits > 1) kps = (((K + splits - 1) / splits) + KMIN - 1) / KMIN * KMIN;
  const int64_t nsplit = (K + kps - 1) / kps;
  *nsplit_out = nsplit;
  float* p = ((epi == ALODLM_EPI_ACCUM || epi == ALODLM_EPI_STORE_F32) && nsplit > 1) ? part : nullptr;
  if (a_kmajor && b_kmajor) launch_layout<true, true>(A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, epi, p, kps, nsplit, first_into_c, segs, st);
  else if (a_kmajor) launch_layout<true, false>(A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, epi, p, kps, nsplit, first_into_c, segs, st);
  else if (b_kmajor) launch_layout<false, true>(A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, epi, p, kps, nsplit, first_into_c, segs, st);
  else launch_layout<false, false>(A, lda, B, ldb, C, ldc, R, ldr, M, N, K, alpha, epi, p, kps, nsplit, first_into_c, segs, st);
}
