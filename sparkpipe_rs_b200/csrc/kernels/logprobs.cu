// Log probabilities of given tokens, the entropy of their distribution and its most
// probable tokens, from logits [T, V], sm_100a.
//
// For a row x: m = max x, S = sum exp(x_i - m), E = sum exp(x_i - m) (x_i - m);
//   log p_i = (x_i - m) - ln S,   entropy = ln S - E / S.
// m, S and E come from one pass: a running maximum, and sums that are rescaled when it
// grows. (x_i - m) is formed before ln S is taken off, so rows of the type's lowest value
// keep their probabilities. Sums are fp32 per thread and joined in fp64.
//
// Rows without a distribution: all -inf (a mask that leaves nothing) has log p = -inf,
// entropy 0 and no alternatives; a row with NaN or +inf gives NaN and no alternatives.
// Alternatives are ordered by logit, then by lower id; -inf logits are none (id -1, -inf).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <stdexcept>

#include "common.cuh"
#include "launch.h"
#include "pdl.h"

namespace sp {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256;

SP_DEVI float to_f32(float v) { return v; }
SP_DEVI float to_f32(__half v) { return __half2float(v); }
SP_DEVI float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

struct Stat {
  float m;   // running maximum
  float s;   // sum 2^((x - m) log2 e)
  float e;   // sum of the same terms times (x - m) log2 e
};

// Joins two partial sums; a part without terms has m = -inf and s = e = 0.
SP_DEVI void join(float& m, double& s, double& e, float m2, double s2, double e2) {
  const float top = fmaxf(m, m2);
  if (top == -INFINITY) {  // neither part has a term (NaN sums pass through)
    s += s2;
    e += e2;
    return;
  }
  const float d1 = m == -INFINITY ? 0.f : (m - top) * kLog2e, d2 = m2 == -INFINITY ? 0.f : (m2 - top) * kLog2e;
  const double w1 = exp2f(fmaxf(d1, -300.f)), w2 = exp2f(fmaxf(d2, -300.f));
  // terms of a part at distance d from the new maximum: t' = t + d
  const double t1 = fmaxf(d1, -300.f), t2 = fmaxf(d2, -300.f);
  e = w1 * (e + s * t1) + w2 * (e2 + s2 * t2);
  s = w1 * s + w2 * s2;
  m = top;
}

// (v, i) ranks before (w, j): larger logit, then lower id
SP_DEVI bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

}  // namespace

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const T* __restrict__ logits, long long ld, int V,
                                                                  const int* __restrict__ ids, int given, int k,
                                                                  float* __restrict__ lp, float* __restrict__ entropy,
                                                                  float* __restrict__ top_lp, int* __restrict__ top_id) {
  griddep_wait();
  griddep_launch();
  const long long row = blockIdx.x;
  const T* x = logits + row * ld;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  Stat a = {-INFINITY, 0.f, 0.f};
  for (int c = threadIdx.x; c < V; c += kThreads) {
    const float v = to_f32(x[c]);
    const float top = fmaxf(a.m, v);
    if (top > a.m) {
      const float d = a.m == -INFINITY ? 0.f : fmaxf((a.m - top) * kLog2e, -300.f);
      a.e = exp2f(d) * (a.e + a.s * d);
      a.s *= exp2f(d);
      a.m = top;
    }
    if (v == -INFINITY) continue;
    const float t = v - a.m;  // NaN for NaN and +inf logits: the sums carry it
    const float u = t < -200.f ? -200.f : t * kLog2e;
    const float p = exp2f(u);
    a.s += p;
    a.e += p * u;
  }
  float m = a.m;
  double s = a.s, e = a.e;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    join(m, s, e, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o),
         __shfl_xor_sync(0xffffffffu, e, o));
  __shared__ float sm[kThreads / 32];
  __shared__ double ss[kThreads / 32], se[kThreads / 32];
  __shared__ float bv[kThreads / 32];
  __shared__ int bi[kThreads / 32];
  if (lane == 0) {
    sm[w] = m;
    ss[w] = s;
    se[w] = e;
  }
  __syncthreads();
  m = sm[0];
  s = ss[0];
  e = se[0];
  for (int i = 1; i < kThreads / 32; ++i) join(m, s, e, sm[i], ss[i], se[i]);
  const bool bad = s != s, empty = !bad && s == 0.0;
  const float log_s = empty ? 0.f : (s < 2.0 ? log1pf(float(s - 1.0)) : logf(float(s)));
  const float base = empty ? 0.f : m;
  if (threadIdx.x == 0)
    entropy[row] = bad ? NAN : empty ? 0.f : float(log_s - e / s * 0.6931471805599453);
  for (int j = threadIdx.x; j < given; j += kThreads) {
    const int id = ids[row * given + j];
    lp[row * given + j] = id == -1 ? 0.f : (id < 0 || id >= V || bad) ? NAN : (to_f32(x[id]) - base) - log_s;
  }
  // k rounds: the best (logit, id) that ranks after the previous round's
  float pv = INFINITY;
  int pi = -1;
  for (int r = 0; r < k; ++r) {
    float best = -INFINITY;
    int at = 0x7fffffff;
    if (!bad && pi != 0x7fffffff)
      for (int c = threadIdx.x; c < V; c += kThreads) {
        const float v = to_f32(x[c]);
        if (v != -INFINITY && before(pv, pi, v, c) && before(v, c, best, at)) { best = v; at = c; }
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, best, o);
      const int oi = __shfl_xor_sync(0xffffffffu, at, o);
      if (before(ov, oi, best, at)) { best = ov; at = oi; }
    }
    __syncthreads();
    if (lane == 0) {
      bv[w] = best;
      bi[w] = at;
    }
    __syncthreads();
    best = bv[0];
    at = bi[0];
    for (int i = 1; i < kThreads / 32; ++i)
      if (before(bv[i], bi[i], best, at)) { best = bv[i]; at = bi[i]; }
    pv = best;
    pi = at;
    if (threadIdx.x == 0) {
      const bool none = at == 0x7fffffff;
      top_id[row * k + r] = none ? -1 : at;
      top_lp[row * k + r] = bad ? NAN : none ? -INFINITY : (best - base) - log_s;
    }
  }
}

void token_logprobs(const void* logits, int dtype, long long ld, int rows, int V, const int* ids, int given, int k,
                    float* lp, float* entropy, float* top_lp, int* top_id, cudaStream_t s) {
  if (rows <= 0) return;
  auto run = [&](auto* x, auto kern) {
    launch_k(kern, dim3((unsigned)rows), dim3(kThreads), 0, s, x, ld, V, ids, given, k, lp, entropy, top_lp, top_id);
  };
  if (dtype == 0) run(static_cast<const __nv_bfloat16*>(logits), token_logprobs_kernel<__nv_bfloat16>);
  else if (dtype == 1) run(static_cast<const __half*>(logits), token_logprobs_kernel<__half>);
  else run(static_cast<const float*>(logits), token_logprobs_kernel<float>);
}

}  // namespace sp
