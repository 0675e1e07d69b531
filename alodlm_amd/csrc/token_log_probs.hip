// Log probabilities of given tokens, entropy and top alternatives of logits over the
// vocabulary, and the gradient in the logits.
//
// Mathematics: with x = logits / T and m = max x, one pass keeps s = sum exp(x - m)
// and t = sum exp(x - m) (x - m) in float32 (rescaled when m moves), from which
// lse = m + log s and the entropy is log s - t / s: t is summed relative to the
// maximum, so nothing large cancels.
#include "common.h"

#define LP_THREADS 256

// Running (m, s, t) of the logits seen so far.
struct Softmax {
  float m, s, t;
  static __device__ __forceinline__ Softmax none() { return {-INFINITY, 0.f, 0.f}; }
  // x with a finite or -inf maximum so far; NaN and +inf end up in s.
  __device__ __forceinline__ void add(float x) {
    if (x > m) {
      rescale(x);
    }
    const float d = x - (m == -INFINITY ? 0.f : m);
    const float e = expf(d);
    s += e;
    t = fmaf(e, fmaxf(d, -1e30f), t);  // 0 * -inf does not count
  }
  __device__ __forceinline__ void rescale(float to) {
    if (m > -INFINITY) {
      const float d = fmaxf(m - to, -1e30f), f = expf(d);  // 0 * overflow does not count
      t = f * fmaf(s, d, t);
      s *= f;
    }
    m = to;
  }
  __device__ __forceinline__ void join(const Softmax& o) {
    const float to = fmaxf(m, o.m);
    Softmax b = o;
    if (to > m) rescale(to);
    if (to > b.m) b.rescale(to);
    s += b.s;
    t += b.t;
  }
};

__device__ __forceinline__ Softmax shfl_xor(const Softmax& x, int off) {
  Softmax o;
  o.m = __shfl_xor(x.m, off, 64);
  o.s = __shfl_xor(x.s, off, 64);
  o.t = __shfl_xor(x.t, off, 64);
  return o;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
token_log_probs_kernel(const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ targets,
                       int64_t V, int top, float inv_t, int64_t ignore, float* __restrict__ log_prob,
                       float* __restrict__ entropy, float* __restrict__ lse_out,
                       float* __restrict__ top_log_prob, int64_t* __restrict__ top_ids) {
  __shared__ Softmax part[LP_THREADS / 64];
  __shared__ float best_v[LP_THREADS / 64];
  __shared__ int64_t best_i[LP_THREADS / 64];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Softmax a = Softmax::none();
  for (int64_t c = threadIdx.x; c < V; c += LP_THREADS) a.add(Elem<T>::load(x, c) * inv_t);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) a.join(shfl_xor(a, off));
  if (lane == 0) part[wave] = a;
  __syncthreads();
  a = part[0];
  for (int w = 1; w < LP_THREADS / 64; ++w) a.join(part[w]);
  const bool empty = a.m == -INFINITY && a.s == 0.f;
  const float lse = empty ? -INFINITY : a.m + logf(a.s);
  if (threadIdx.x == 0) {
    const int64_t tg = targets[row];
    float lp = 0.f;
    if (tg != ignore) {
      lp = tg >= 0 && tg < V ? Elem<T>::load(x, tg) * inv_t : NAN;
      lp = empty && tg >= 0 && tg < V ? -INFINITY : lp - lse;
    }
    log_prob[row] = lp;
    entropy[row] = empty ? 0.f : logf(a.s) - a.t / a.s;
    lse_out[row] = lse;
  }
  // alternatives: the largest behind the one found last, in (value, index) order
  float last_v = INFINITY;
  int64_t last_i = -1;
  for (int k = 0; k < top; ++k) {
    float bv = -INFINITY;
    int64_t bi = V;
    for (int64_t c = threadIdx.x; c < V; c += LP_THREADS) {
      float v = Elem<T>::load(x, c);
      if (!(v == v)) v = -INFINITY;  // NaN ranks lowest
      if (v > last_v || (v == last_v && c <= last_i)) continue;
      if (v > bv || (v == bv && c < bi)) { bv = v; bi = c; }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float ov = __shfl_xor(bv, off, 64);
      const int64_t oi = __shfl_xor((long long)bi, off, 64);
      if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
    }
    __syncthreads();
    if (lane == 0) { best_v[wave] = bv; best_i[wave] = bi; }
    __syncthreads();
    for (int w = 0; w < LP_THREADS / 64; ++w)
      if (w == 0 || best_v[w] > bv || (best_v[w] == bv && best_i[w] < bi)) { bv = best_v[w]; bi = best_i[w]; }
    last_v = bv;
    last_i = bi;
    if (threadIdx.x == 0) {
      top_ids[row * top + k] = bi;
      top_log_prob[row * top + k] = empty ? -INFINITY : Elem<T>::load(x, bi) * inv_t - lse;
    }
  }
}

// dlogits = (g_target [c = target] + sum_k g_k [c = top_k] - p (g_target + sum_k g_k)
//            - g_entropy p (log p + entropy)) / T
template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
token_log_probs_bwd_kernel(const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ targets,
                           const int64_t* __restrict__ top_ids, const float* __restrict__ lse_in,
                           const float* __restrict__ entropy, const float* __restrict__ d_log_prob,
                           const float* __restrict__ d_entropy, const float* __restrict__ d_top,
                           int64_t V, int top, float inv_t, int64_t ignore, T* __restrict__ dlogits) {
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  const float lse = lse_in[row];
  const int64_t tg = targets[row];
  const float gt = d_log_prob && tg != ignore ? d_log_prob[row] : 0.f;
  const float gh = d_entropy ? d_entropy[row] : 0.f, H = entropy[row];
  float all = gt;
  if (d_top)
    for (int k = 0; k < top; ++k) all += d_top[row * top + k];
  for (int64_t c = threadIdx.x; c < V; c += LP_THREADS) {
    const float lp = Elem<T>::load(x, c) * inv_t - lse;
    float g = 0.f;
    if (lse != -INFINITY) {
      const float p = expf(lp);
      g = -p * fmaf(gh, fmaxf(lp, -1e30f) + H, all);
      if (c == tg) g += gt;
      if (d_top)
        for (int k = 0; k < top; ++k)
          if (top_ids[row * top + k] == c) g += d_top[row * top + k];
    }
    Elem<T>::store(dlogits + row * V, c, g * inv_t);
  }
}

static int check_shape(int64_t rows, int64_t vocab, int64_t top, int64_t ld, float inv_t) {
  ALODLM_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "token_log_probs: rows out of range");
  ALODLM_CHECK_ARG(vocab >= 1 && vocab < (1ll << 31) && ld >= vocab,
                   "token_log_probs: vocabulary or row stride out of range");
  ALODLM_CHECK_ARG(top >= 0 && top <= 64 && top <= vocab,
                   "token_log_probs: top must be 0 to 64 and at most the vocabulary");
  ALODLM_CHECK_ARG(inv_t > 0.f && inv_t < INFINITY, "token_log_probs: the temperature must be positive");
  return ALODLM_OK;
}

extern "C" int64_t alodlm_token_log_probs_workspace(int64_t, int64_t, int64_t) { return 0; }

extern "C" int alodlm_token_log_probs(const void* logits, int64_t ld, const int64_t* targets,
                                      int64_t rows, int64_t vocab, int64_t top,
                                      float inv_temperature, int64_t ignore, float* log_prob,
                                      float* entropy, float* lse, float* top_log_prob,
                                      int64_t* top_ids, float* workspace, int dtype, void* stream) {
  const int rc = check_shape(rows, vocab, top, ld, inv_temperature);
  if (rc) return rc;
  if (rows == 0) return ALODLM_OK;
  ALODLM_CHECK_ARG(top == 0 || (top_log_prob && top_ids), "token_log_probs: no room for the alternatives");
  ALODLM_DISPATCH(dtype, T, {
    token_log_probs_kernel<T><<<(unsigned)rows, LP_THREADS, 0, as_stream(stream)>>>(
        (const T*)logits, ld, targets, vocab, (int)top, inv_temperature, ignore, log_prob, entropy,
        lse, top_log_prob, top_ids);
  });
  ALODLM_CHECK_LAUNCH("token_log_probs");
  return ALODLM_OK;
}

extern "C" int alodlm_token_log_probs_bwd(const void* logits, int64_t ld, const int64_t* targets,
                                          const int64_t* top_ids, const float* lse,
                                          const float* entropy, const float* d_log_prob,
                                          const float* d_entropy, const float* d_top, int64_t rows,
                                          int64_t vocab, int64_t top, float inv_temperature,
                                          int64_t ignore, void* dlogits, int dtype, void* stream) {
  const int rc = check_shape(rows, vocab, top, ld, inv_temperature);
  if (rc) return rc;
  if (rows == 0) return ALODLM_OK;
  ALODLM_CHECK_ARG(!d_top || top == 0 || top_ids, "token_log_probs_bwd: no alternatives");
  ALODLM_DISPATCH(dtype, T, {
    token_log_probs_bwd_kernel<T><<<(unsigned)rows, LP_THREADS, 0, as_stream(stream)>>>(
        (const T*)logits, ld, targets, top_ids, lse, entropy, d_log_prob, d_entropy, d_top, vocab,
        (int)top, inv_temperature, ignore, (T*)dlogits);
  });
  ALODLM_CHECK_LAUNCH("token_log_probs_bwd");
  return ALODLM_OK;
}
