// Losses over a large vocabulary against a few known tokens a row.
//
// A row knows tokens id_k with probabilities q_k: one of probability 1 (cross entropy) or
// a teacher's most likely ones.  With z the row's logits over T, p = softmax(z),
//   loss = sum_k q_k (ln q_k - ln p[id_k])  [+ q_r (ln q_r - ln p_r)],
// q_r = max(0, 1 - sum_k q_k) and p_r the probability of all tokens that are not known.  Where
// none of these can be, q_r counts as 0: of a vocabulary that teacher and student mask alike it is
// what rounding leaves of 1, and would make the loss infinite.
// The known tokens are kept out of the sum over the vocabulary and joined to it at the
// end, so p_r is a sum of its own and never a difference from 1.  With Q = sum_k q_k [+ q_r]
// and s_r the softmax over the other tokens,
//   dloss / dz = Q p - [q at the known] - [q_r s_r elsewhere]
//              = (Q p_r - q_r) s_r   at a token that is not known: one factor a row,
//                Q p - q             at a known one: one value a row and known token.
// Sums are in base 2 with c = log2 e / T: 2^((z - m) c) of raw logits z relative to the largest
// m, or, where logits come from the matrix cores, 2^(z c - K) relative to a whole number K.
#pragma once

#include "common.h"

#define VL_MAX_KNOWN 256
#define VL_LOG2E 1.44269504088896341f
#define VL_LN2 0.69314718055994531f
#define VL_NONE 0x7fffffff  // no known token
#define VL_MOST_GROUPS (1ll << 24)  // workgroups of 256 threads in a launch: fewer than 2^32 threads

// What is kept of a call for its backward, in floats: 4 of the call, 8 of a row, and per
// row and place its known tokens, each id once (VL_NONE elsewhere).  known_prepare puts
// them in ascending order.
struct KnownRows {
  float* call;    // [0]: what an upstream gradient of the reduced loss is times
  float* info;    // [rows][8]
  int* ids;       // [rows][known]
  float* weight;  // [rows][known]: q, then Q p - q
  float* log_q;   // [rows][known]: the mean of ln q over an id's occurrences
  float* logit;   // [rows][known]: raw logits
  int known;
};
enum { RI_MASS = 0, RI_REST = 1, RI_BAD = 2, RI_COUNTED = 3, RI_M = 4, RI_LOG = 5, RI_FACTOR = 6, RI_LOSS = 7 };

static inline int64_t known_rows_floats(int64_t rows, int64_t known) { return 4 + rows * (8 + 4 * known); }
static inline KnownRows known_rows(float* state, int64_t rows, int64_t known) {
  KnownRows r;
  r.call = state;
  r.info = state + 4;
  r.ids = reinterpret_cast<int*>(r.info + 8 * rows);
  r.weight = reinterpret_cast<float*>(r.ids + rows * known);
  r.log_q = r.weight + rows * known;
  r.logit = r.log_q + rows * known;
  r.known = (int)known;
  return r;
}

// The known tokens as the caller has them: targets [rows] (one token of probability 1,
// `ignore` none), or ids and log_q [rows][known].
struct GivenRows {
  const int64_t* targets;
  const int64_t* ids;
  const float* log_q;
  int64_t ignore;
  int known, vocab, rest;
};

// A part of a row's sum over the tokens that are not known: its largest raw logit m and
// sum 2^((z - m) c), or K (in m) and sum 2^(z c - K); -inf and 0 where no token can be (or
// none is there).  Joined with c, or 1 for the latter.
struct Part {
  float m, sum;
};
__device__ __forceinline__ float part_ref(float largest, float c) { return ceilf(largest * c); }
__device__ __forceinline__ Part part_join(const Part& a, const Part& b, float c) {
  const float to = fmaxf(a.m, b.m), base = to == -INFINITY ? 0.f : to;
  // what is -inf weighs 0 (NaN stays)
  return {to, a.sum * __builtin_amdgcn_exp2f((a.m - base) * c) + b.sum * __builtin_amdgcn_exp2f((b.m - base) * c)};
}

enum { VL_EACH = 0, VL_SUM = 1, VL_MEAN = 2 };

// The upstream gradient over the temperature.  `apart`: a reduced loss's, which all rows
// share, is left to the end (all()), so that a row's gradient is Q p - q itself and loses
// nothing to another factor's mantissa when it is rounded; a row's is then 1, or 0 where
// the whole is.  (One that is NaN or infinite stays with the rows: at the end it would meet
// the zeros of rows that have no gradient.)
struct Upstream {
  const float* call;
  const float* d_loss;
  int reduction, apart;
  float inv_t;
  __device__ __forceinline__ float shared() const { return d_loss[0] * call[0] * inv_t; }
  __device__ __forceinline__ float row(int64_t r) const {
    if (reduction == VL_EACH) return d_loss[r] * inv_t;
    const float s = shared();
    return apart && s - s == 0.f ? (s != 0.f ? 1.f : 0.f) : s;
  }
  __device__ __forceinline__ float all() const {
    if (!apart || reduction == VL_EACH) return 1.f;
    const float s = shared();
    return s - s == 0.f ? s : 1.f;
  }
};

// What a row's share of the others is times: nothing where the row takes no part, which may
// hold NaN, or where it has no gradient, whose upstream gradient may be NaN or infinite.
__device__ __forceinline__ float row_factor(float up, float factor) {
  return up == 0.f || factor == 0.f ? 0.f : up * factor;
}

// Launches (vocab_loss.hip).
//
// The rows' known tokens into k, in ascending order.
void known_prepare_launch(const KnownRows& k, const GivenRows& given, int64_t rows, hipStream_t st);
// The row sums of logits [rows, width], columns first .. of the vocabulary, in `chunks`
// parts a row at part[chunk * rows + row].  `prepared`: k has the known tokens, and their
// logits go there; else `given` names them.
int64_t row_stats_chunks(int64_t rows, int64_t width);
template <typename T>
void row_stats_launch(const T* logits, int64_t ld, int64_t rows, int64_t width, int64_t first,
                      const KnownRows& k, const GivenRows& given, bool prepared, float c, int64_t chunks,
                      Part* part, hipStream_t st);
// Losses and the gradient's factors from `parts` parts a row, and the reduced loss.  With
// whole logits [rows, vocab] in memory (else NULL) the known tokens need no preparation.
// `scaled`: the parts' reference is a whole number K, and RI_M is then one too.
template <typename T>
void known_finish_launch(const KnownRows& k, const GivenRows& given, const T* logits, int64_t ld,
                         const Part* part, int64_t parts, int64_t rows, float c, bool scaled,
                         int reduction, float* loss, hipStream_t st);
// dlogits (TO, row stride ldo; columns [width, padded) and rows [rows, padded_rows) zero) of
// logits [rows, width], columns first .. of the vocabulary; may be in place.  `parts` (bf16 of
// float logits): in two parts, rows r and rows + r, which the padded rows take in.
template <typename TI, typename TO>
void row_grads_launch(const TI* logits, int64_t ld, int64_t rows, int64_t width, int64_t first,
                      const KnownRows& k, float c, const Upstream& up, TO* out, int64_t ldo,
                      int64_t padded_rows, int64_t padded, hipStream_t st, bool parts);

// The same of few rows in float32, tokens first: out [width][pad], zeros behind the rows.
void few_grads_launch(const float* logits, int64_t ld, int64_t rows, int64_t width, int64_t first,
                      const KnownRows& k, float c, const Upstream& up, float* out, int64_t pad,
                      hipStream_t st);

static inline int check_vocab_loss(const char* what, int64_t rows, int64_t vocab, int64_t known,
                                   float inv_t, int reduction) {
  ALODLM_CHECK_ARG(rows >= 0 && rows < (1ll << 24), "%s: rows out of range", what);
  ALODLM_CHECK_ARG(vocab >= 1 && vocab < (1ll << 30), "%s: vocabulary out of range", what);
  ALODLM_CHECK_ARG(known >= 1 && known <= VL_MAX_KNOWN, "%s: 1 to 256 known tokens a row", what);
  ALODLM_CHECK_ARG(inv_t > 0.f && inv_t * VL_LOG2E < INFINITY,
                   "%s: the temperature must be positive, its inverse times log2 e finite", what);
  ALODLM_CHECK_ARG(reduction >= 0 && reduction <= 2, "%s: bad reduction", what);
  return ALODLM_OK;
}
