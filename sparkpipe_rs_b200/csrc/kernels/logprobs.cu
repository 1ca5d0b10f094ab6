// Log probabilities of given tokens, the entropy of their distribution and its most
// probable tokens, from logits [T, V], sm_100a.
//
// For a row x: m = max x, S = sum exp(x_i - m), E = sum exp(x_i - m) (x_i - m);
//   log p_i = (x_i - m) - ln S,   entropy = ln S - E / S.
// m, S and E come from one pass: a running maximum, and sums that are rescaled when it
// grows. (x_i - m) is formed before ln S is taken off, so rows of the type's lowest value
// keep their probabilities. Terms are added up per batch of a thread, S's batches with
// their rounding errors kept (two fp32 words), the threads in fp64: a row with one sure
// token keeps what the others weigh, and ln S is log1p of it. E's batches, some twenty of a
// thread in a long row, are added in plain fp32 (entropy within 4e-8 of 64 bits, 2-norm).
//
// Rows without a distribution: all -inf (a mask that leaves nothing) has log p = -inf,
// entropy 0 and no alternatives; a row with NaN or +inf gives NaN and no alternatives.
// Alternatives are ordered by logit, then by lower id; -inf logits are none (id -1, -inf).
//
// What bounds it: one read of the logits. At 8,192 rows x 102,400 bf16 an SM takes in 11
// logits per clock, which leaves room for about eleven instructions and one exponential
// (16 per clock) for each, so the loop works on packed pairs: 7.6 instructions per logit, the
// exponentials' pipe two thirds busy, 300 us (5.6 TB/s). The alternatives cost one comparison
// per batch: while it streams, a thread notes the maximum of each batch of 16 or 32 logits in
// shared memory. Of the 64 maxima of four threads each (fewer in short rows), the k-th largest
// is a floor under the row's k-th largest logit; afterwards only batches whose maximum reaches
// it are read again (about k of them), and the logits at or above the floor are ranked by
// counting: 325 us with 20 alternatives. Should ties leave more of them than the list holds, k
// rounds of the CTA's maximum pick them one by one (1.2 ms for 8,192 rows of 102,400 equal logits).
//
// Few rows are split over the CTAs of a thread-block cluster, which join their sums and
// lists through distributed shared memory: one launch, no workspace, nothing that two
// streams or graphs could share.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>

#include "common.cuh"
#include "launch.h"
#include "logprobs.cuh"
#include "pdl.h"

namespace sp {

namespace {

constexpr int kLong = 256, kShort = 64;  // threads of a row's CTA
// 64 registers, which hold a batch and the next one's loads (8,192 rows x 102,400 with 20
// alternatives: 323 us, 346 us without the loads ahead; with 80 registers 342 us, with 48 and
// half as large batches 336 us)
constexpr int kCtasPerSm = 4;     // of 256 threads
constexpr int kBatch = 4;         // 16-byte vectors of a batch, in flight together
constexpr int kSlots = 16;        // recorded batch maxima of a thread (several batches each in longer rows)
constexpr int kGroups = 64;
// Logits at or above the floor that are ranked by counting, n comparisons each; of more, k rounds
// pick them (8,192 rows of 1,000 equal logits, 20 alternatives: 217 us, by counting 2,600; 64 rows
// of four values, 250 of each: 32 against 18).
constexpr int kList = 256;
constexpr int kHot = 512;         // (thread, slot) entries whose batches reach it
constexpr int kMaxCluster = 8;
constexpr int kNone = 0x7fffffff;

// maxima that keep NaN
SP_DEVI unsigned max_nan_bf16x2(unsigned a, unsigned b) {
  unsigned r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
SP_DEVI unsigned max_nan_f16x2(unsigned a, unsigned b) {
  unsigned r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 16 bytes of logits: their values, and the maximum (NaN dropped) of two such vectors.
template <typename T>
struct Logits;
template <>
struct Logits<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr unsigned kNegInf = 0xff80ff80u;
  // logits below `kLow` (-1e30) weigh nothing beside a maximum within (kMin, kMax)
  static constexpr float kMin = -1e29f, kMax = 1e29f;
  static SP_DEVI unsigned max_nan2(unsigned a, unsigned b) { return max_nan_bf16x2(a, b); }
  static SP_DEVI unsigned raise(unsigned w) { return max_nan_bf16x2(w, 0xf149f149u); }
  static SP_DEVI float value(__nv_bfloat16 v) { return __bfloat162float(v); }
  static SP_DEVI void pair(unsigned w, float& a, float& b) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  }
  static SP_DEVI unsigned max2(unsigned a, unsigned b) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
  }
};
template <>
struct Logits<__half> {
  static constexpr int N = 8;
  static constexpr unsigned kNegInf = 0xfc00fc00u;
  static constexpr float kMin = -60000.f, kMax = 65504.f * 2;  // raised to the type's lowest value, -65504
  static SP_DEVI unsigned max_nan2(unsigned a, unsigned b) { return max_nan_f16x2(a, b); }
  static SP_DEVI unsigned raise(unsigned w) { return max_nan_f16x2(w, 0xfbfffbffu); }
  static SP_DEVI float value(__half v) { return __half2float(v); }
  static SP_DEVI void pair(unsigned w, float& a, float& b) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w));
    a = f.x;
    b = f.y;
  }
  static SP_DEVI unsigned max2(unsigned a, unsigned b) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
  }
};
template <>
struct Logits<float> {
  static constexpr int N = 4;
  static constexpr unsigned kNegInf = 0xff800000u;
  static constexpr float kMin = -1e29f, kMax = 1e29f;
  static SP_DEVI unsigned max_nan2(unsigned a, unsigned b) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  static SP_DEVI unsigned raise(unsigned w) { return __float_as_uint(max_nan(__uint_as_float(w), -1e30f)); }
  static SP_DEVI float value(float v) { return v; }
  static SP_DEVI void pair(unsigned, float&, float&) {}
  static SP_DEVI unsigned max2(unsigned a, unsigned b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
};

// Values 2 j and 2 j + 1 of a vector.
template <typename T>
SP_DEVI void values2(const uint4& v, int j, float& a, float& b) {
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
  if (sizeof(T) == 4) {
    a = __uint_as_float(w[2 * j]);
    b = __uint_as_float(w[2 * j + 1]);
  } else {
    Logits<T>::pair(w[j], a, b);
  }
}

template <typename T>
SP_DEVI float batch_max(const uint4 (&v)[kBatch]) {
  using L = Logits<T>;
  unsigned m = L::max2(L::max2(v[0].x, v[0].y), L::max2(v[0].z, v[0].w));
#pragma unroll
  for (int i = 1; i < kBatch; ++i) m = L::max2(m, L::max2(L::max2(v[i].x, v[i].y), L::max2(v[i].z, v[i].w)));
  if (sizeof(T) == 4) return __uint_as_float(m);
  float a, b;
  L::pair(m, a, b);
  return fmaxf(a, b);
}

// Whether a batch is all -inf (no NaN either).
template <typename T>
SP_DEVI bool all_masked(const uint4 (&v)[kBatch]) {
  using L = Logits<T>;
  unsigned m = L::kNegInf;
#pragma unroll
  for (int i = 0; i < kBatch; ++i)
    m = L::max_nan2(m, L::max_nan2(L::max_nan2(v[i].x, v[i].y), L::max_nan2(v[i].z, v[i].w)));
  return m == L::kNegInf;
}

// The sums of a batch's terms. Beside a maximum of ordinary size (CLAMP false) very small
// logits are raised, two in one instruction, so that -inf needs no care further on.
template <typename T, bool CLAMP>
SP_DEVI void batch_terms(const uint4 (&v)[kBatch], float shift, float& s, float& e) {
  using L = Logits<T>;
  const u64t sh = pack2(shift, shift);
  u64t s0 = 0, s1 = 0, e0 = 0, e1 = 0;
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    uint4 r = v[i];
    if (!CLAMP) r = make_uint4(L::raise(r.x), L::raise(r.y), L::raise(r.z), L::raise(r.w));
#pragma unroll
    for (int j = 0; j < L::N / 2; j += 2) {
      float f0, f1, f2, f3;
      values2<T>(r, j, f0, f1);
      values2<T>(r, j + 1, f2, f3);
      logprob_terms<CLAMP>(f0, f1, sh, s0, e0);
      logprob_terms<CLAMP>(f2, f3, sh, s1, e1);
    }
  }
  float p, q;
  unpack2(add2(s0, s1), p, q);
  s = p + q;
  unpack2(add2(e0, e1), p, q);
  e = p + q;
}

struct Batch {
  uint4 v[kBatch];
};
// Out of line: rows of nothing but masked logits so far, huge logits, NaN.
template <typename T>
__device__ __noinline__ float2 rare_terms(Batch b, float shift) {
  float2 r;
  batch_terms<T, true>(b.v, shift, r.x, r.y);
  return r;
}

// (v, i) ranks before (w, j): larger logit, then lower id
SP_DEVI bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// This CTA's part of a row: single logits before the first 128-byte line and behind the last
// whole vector (at most one each per thread), vectors in between. Vectors that start with a
// line let a warp's load touch four lines, not five: 515 rows x 129,281 fp32 went from 64 to
// 57 us (129,280, whose rows all start with a line: 52 us).
template <typename T, int THREADS>
struct Part {
  const T* row;
  const uint4* body;
  int first;      // id of the body's first logit
  int v0, v1;     // this CTA's vectors
  int head, tail; // id of this thread's single logits, -1 for none

  SP_DEVI Part(const T* r, int V, int rank, int parts) : row(r) {
    constexpr int N = Logits<T>::N;
    const int skip = int((128 - (reinterpret_cast<uintptr_t>(r) & 127)) & 127) / (int)sizeof(T);
    first = min(skip, V);
    body = reinterpret_cast<const uint4*>(r + first);
    const int nv = (V - first) / N;
    v0 = int((long long)nv * rank / parts) & ~7;
    v1 = rank == parts - 1 ? nv : int((long long)nv * (rank + 1) / parts) & ~7;
    const int t = threadIdx.x;
    head = rank == 0 && t < first ? t : -1;
    const int behind = first + nv * N;
    tail = rank == parts - 1 && t < V - behind ? behind + t : -1;
  }
  SP_DEVI uint4 vector(int v) const {
    if (v < v1) return __ldg(body + v);
    constexpr unsigned n = Logits<T>::kNegInf;
    return make_uint4(n, n, n, n);
  }
  SP_DEVI float single(int id) const { return id >= 0 ? Logits<T>::value(row[id]) : -INFINITY; }
  // calls f(logit, id) for this thread's logits in batches [b0, b1) (vectors) or its single ones
  template <typename F>
  SP_DEVI void batches(int b0, int b1, F f) const {
    for (int b = b0; b < b1; ++b) {
      uint4 v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) v[i] = vector(v0 + (b * kBatch + i) * THREADS + threadIdx.x);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int at = first + (v0 + (b * kBatch + i) * THREADS + (int)threadIdx.x) * Logits<T>::N;
#pragma unroll
        for (int j = 0; j < Logits<T>::N / 2; ++j) {
          float x, y;
          values2<T>(v[i], j, x, y);
          f(x, at + 2 * j);
          f(y, at + 2 * j + 1);
        }
      }
    }
  }
  template <typename F>
  SP_DEVI void singles(F f) const {
    f(single(head), head);
    f(single(tail), tail);
  }
};

struct Stat {
  float m;
  double s, e;
};

template <int THREADS>
struct Shared {
  float slot[kSlots][THREADS];
  float group[kGroups];            // maxima of four threads' logits each (of the whole cluster)
  Stat stat[kMaxCluster * (THREADS / 32)]; // the cluster's warps (first CTA)
  float floor;
  float base, log_s;               // the row's maximum (0 for an empty row) and ln S
  int bad;
  int hot_n, n;
  int hot[kHot];                   // (thread, slot) whose batches reach the floor
  float v[kList];                  // logits at or above the floor (first CTA)
  int id[kList];
};

// Shared memory of the cluster's CTA q (q < 0: this CTA's own, without a cluster).
SP_DEVI void st_f32(float* p, float v, int q) {
  if (q < 0) *p = v;
  else asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_u32(p), q)), "f"(v) : "memory");
}
SP_DEVI void st_f64(double* p, double v, int q) {
  if (q < 0) *p = v;
  else asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(p), q)), "d"(v) : "memory");
}
SP_DEVI void st_s32(int* p, int v, int q) {
  if (q < 0) *p = v;
  else asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(mapa_shared(smem_u32(p), q)), "r"(v) : "memory");
}
SP_DEVI int add_s32(int* p, int v, int q) {
  if (q < 0) return atomicAdd(p, v);
  int r;
  asm volatile("atom.shared::cluster.add.s32 %0, [%1], %2;" : "=r"(r) : "r"(mapa_shared(smem_u32(p), q)), "r"(v) : "memory");
  return r;
}

// Joins the warps' sums; every lane of the calling warp gets the row's (m, S, E).
template <int THREADS>
SP_DEVI void join_stats(const Shared<THREADS>& sh, int n, float& m, double& s, double& e) {
  const int lane = threadIdx.x & 31;
  m = -INFINITY;
  for (int i = lane; i < n; i += 32) m = fmaxf(m, sh.stat[i].m);
  m = warp_max(m);
  s = e = 0.0;
  for (int i = lane; i < n; i += 32) {
    const Stat t = sh.stat[i];
    const float d = t.m == -INFINITY ? 0.f : fmaxf((t.m - m) * kLog2e, -300.f);
    const double f = fast_exp2(d);
    s += f * t.s;
    e += f * (t.e + t.s * d);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    e += __shfl_xor_sync(0xffffffffu, e, o);
  }
}

// More logits reach the floor than the list holds: each thread offers its best one not
// yet taken, the CTA takes the best of these, k times. The next offer of the thread whose
// one was taken is found by its whole warp.
template <typename T, int THREADS>
__device__ __noinline__ void pick_rounds(const Part<T, THREADS>& part, int nb, int k, Shared<THREADS>& sh) {
  constexpr int WARPS = THREADS / 32;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  float best = -INFINITY;
  int at = kNone;
  auto first_of_warp = [](float& v, int& i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, v, o);
      const int oi = __shfl_xor_sync(0xffffffffu, i, o);
      if (before(ov, oi, v, i)) { v = ov; i = oi; }
    }
  };
  auto offer = [&](float v, int i) {
    if (v != -INFINITY && i >= 0 && before(v, i, best, at)) { best = v; at = i; }
  };
  part.batches(0, nb, offer);
  part.singles(offer);
  for (int r = 0; r < k; ++r) {
    float pv = best;
    int pi = at;
    first_of_warp(pv, pi);
    __syncthreads();
    if (lane == 0) {
      sh.v[w] = pv;
      sh.id[w] = pi;
    }
    __syncthreads();
    for (int i = 0; i < WARPS; ++i)
      if (before(sh.v[i], sh.id[i], pv, pi)) { pv = sh.v[i]; pi = sh.id[i]; }
    if (pi == kNone) break;  // the same for every thread
    if (threadIdx.x == 0) {
      sh.v[WARPS + r] = pv;
      sh.id[WARPS + r] = pi;
      sh.n = r + 1;
    }
    const unsigned taken = __ballot_sync(0xffffffffu, at == pi);
    if (taken) {  // this warp's thread `from`: its best logit that ranks after the one taken
      const int from = __ffs(taken) - 1;
      float nv = -INFINITY;
      int ni = kNone;
      auto next = [&](float v, int i) {
        if (v != -INFINITY && i >= 0 && before(pv, pi, v, i) && before(v, i, nv, ni)) { nv = v; ni = i; }
      };
      for (int v = part.v0 + w * 32 + from + lane * THREADS; v < part.v1; v += 32 * THREADS) {
        const uint4 q = __ldg(part.body + v);
#pragma unroll
        for (int j = 0; j < Logits<T>::N / 2; ++j) {
          float x, y;
          values2<T>(q, j, x, y);
          next(x, part.first + v * Logits<T>::N + 2 * j);
          next(y, part.first + v * Logits<T>::N + 2 * j + 1);
        }
      }
      if (lane == from) part.singles(next);
      first_of_warp(nv, ni);
      if (lane == from) {
        best = nv;
        at = ni;
      }
    }
  }
  __syncthreads();
}

}  // namespace

// One row per cluster of `parts` CTAs (1: no cluster).
template <typename T, bool TOP, bool CLUSTER, int THREADS>
__global__ void __launch_bounds__(THREADS, kCtasPerSm * kLong / THREADS)
    token_logprobs_kernel(const T* __restrict__ logits, long long ld, int V, const int* __restrict__ ids, int given,
                          int k, int parts, float* __restrict__ lp, float* __restrict__ entropy,
                          float* __restrict__ top_lp, int* __restrict__ top_id) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int WARPS = THREADS / 32, GROUP = THREADS / kGroups;
  Shared<THREADS>& sh = *reinterpret_cast<Shared<THREADS>*>(smem);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int rank = CLUSTER ? (int)cluster_ctarank() : 0;
  const long long row = CLUSTER ? blockIdx.x / parts : blockIdx.x;
  if (CLUSTER) cluster_sync();  // all its CTAs have started: they will write one another's shared memory
  griddep_wait();
  griddep_launch();
  const T* x = logits + row * ld;
  const Part<T, THREADS> part(x, V, rank, CLUSTER ? parts : 1);
  // the first given tokens' logits, on their way while the row streams
  int id = -1;
  float xid = 0.f;
  if (rank == 0 && (int)threadIdx.x < given) {
    id = ids[row * given + threadIdx.x];
    if (id >= 0 && id < V) xid = Logits<T>::value(x[id]);
  }
  const int nb = (part.v1 - part.v0 + kBatch * THREADS - 1) / (kBatch * THREADS);
  const int per_slot = (nb + kSlots - 1) / kSlots;

  LogprobSums a;
  float slot_max = -INFINITY;
  int slot = 0, left = per_slot;
  auto take = [&](uint4 (&v)[kBatch]) {
    const float top = batch_max<T>(v);
    a.raise(top);
    float bs, be;
    if (a.m > Logits<T>::kMin && a.m < Logits<T>::kMax) {
      batch_terms<T, false>(v, -a.m, bs, be);
    } else if (a.m == -INFINITY && all_masked<T>(v)) {
      bs = be = 0.f;  // a mask so far, which costs one maximum
    } else {
      Batch copy;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) copy.v[i] = v[i];
      const float2 r = rare_terms<T>(copy, a.shift());
      bs = r.x;
      be = r.y;
    }
    a.add(bs, be);
    if (TOP && per_slot == 1) {
      sh.slot[slot++][threadIdx.x] = top;
    } else if (TOP) {
      slot_max = fmaxf(slot_max, top);
      if (--left == 0) {
        sh.slot[slot++][threadIdx.x] = slot_max;
        slot_max = -INFINITY;
        left = per_slot;
      }
    }
  };
  const int whole = (part.v1 - part.v0) / (kBatch * THREADS);
  const uint4* src = part.body + part.v0 + threadIdx.x;
  // the next batch's loads go out before this one's arithmetic
  uint4 nx[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) nx[i] = part.vector(part.v0 + i * THREADS + threadIdx.x);
#pragma unroll 1
  for (int b = 0; b < whole; ++b) {
    uint4 v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) v[i] = nx[i];
    src += kBatch * THREADS;
    if (b + 1 < whole) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) nx[i] = __ldg(src + i * THREADS);
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) nx[i] = part.vector(part.v0 + (whole * kBatch + i) * THREADS + threadIdx.x);
    }
    take(v);
  }
  if (whole < nb) take(nx);
  if (TOP && per_slot > 1 && left != per_slot) sh.slot[slot++][threadIdx.x] = slot_max;
  const float one = part.single(part.head), two = part.single(part.tail);
  if (part.head >= 0 || part.tail >= 0) {
    const float top = fmaxf(one, two);
    a.raise(top);
    const float shift = a.shift();
    u64t s0 = 0, e0 = 0;
    logprob_terms<true>(one, two, pack2(shift, shift), s0, e0);
    float p, q, f, g;
    unpack2(s0, p, q);
    unpack2(e0, f, g);
    a.add(p + q, f + g);
  }

  // the warps' sums, to the cluster's first CTA; 64 group maxima, to all its CTAs
  const int first = CLUSTER ? 0 : -1;
  float m = a.m;
  if (TOP && !CLUSTER) {
    // Short rows have a vector for few threads: groups of one or two, that k of them have a
    // logit (2,001 rows x 556 with 20 alternatives: 21 us, in fours 229).
    const int vectors = part.v1 - part.v0;
    const int wide = min(GROUP, vectors <= kGroups ? 1 : vectors <= 2 * kGroups ? 2 : GROUP);
    for (int o = 1; o < wide; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane % wide == 0 && threadIdx.x / wide < kGroups) sh.group[threadIdx.x / wide] = m;
  }
  if (TOP && CLUSTER) {
    const int wide = GROUP * parts;  // threads of a group, at most a warp
    for (int o = 1; o < wide; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane % wide == 0)
      for (int q = 0; q < parts; ++q) st_f32(&sh.group[(rank * THREADS + threadIdx.x) / wide], m, q);
  }
  m = warp_max(m);
  {
    const float d = a.m == -INFINITY ? 0.f : fmaxf((a.m - m) * kLog2e, -300.f);
    const float f = fast_exp2(d);
    double s = double(a.hi * f) + double(a.lo * f), e = double(f * fmaf(a.hi, d, a.e));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      e += __shfl_xor_sync(0xffffffffu, e, o);
    }
    if (lane == 0) {
      Stat* t = &sh.stat[rank * WARPS + w];
      st_f32(&t->m, m, first);
      st_f64(&t->s, s, first);
      st_f64(&t->e, e, first);
    }
  }
  if (TOP && threadIdx.x == 0) sh.n = sh.hot_n = 0;
  if (CLUSTER) cluster_sync();
  else __syncthreads();

  // the join by the last warp of the first CTA, the floor by the first warp of each
  if (rank == 0 && w == WARPS - 1) {
    double s, e;
    join_stats(sh, (CLUSTER ? parts : 1) * WARPS, m, s, e);
    if (lane == 0) {
      const bool bad = s != s, empty = !bad && s == 0.0;
      const float log_s = empty ? 0.f : s < 2.0 ? log1pf(float(s - 1.0)) : logf(float(s));
      sh.bad = bad;
      sh.base = empty ? 0.f : m;
      sh.log_s = log_s;
      entropy[row] = bad ? NAN : empty ? 0.f : float(log_s - e / s * kLn2);
    }
  }
  int n = 0;
  if (TOP) {
    if (w == 0) {
      // the largest group maximum that k of the 64 reach
      const float g0 = sh.group[lane], g1 = sh.group[lane + 32];
      int r0 = 0, r1 = 0;
#pragma unroll
      for (int i = 0; i < kGroups; i += 4) {
        const float4 g = *reinterpret_cast<const float4*>(&sh.group[i]);
        r0 += (g.x >= g0) + (g.y >= g0) + (g.z >= g0) + (g.w >= g0);
        r1 += (g.x >= g1) + (g.y >= g1) + (g.z >= g1) + (g.w >= g1);
      }
      const float f = warp_max(fmaxf(r0 >= k ? g0 : -INFINITY, r1 >= k ? g1 : -INFINITY));
      if (lane == 0) sh.floor = f;
    }
    __syncthreads();
    const float floor = sh.floor;
    auto see = [&](float v, int i) {
      if (v >= floor && v != -INFINITY && i >= 0) {
        const int at = add_s32(&sh.n, 1, first);
        if (at < kList) {
          st_f32(&sh.v[at], v, first);
          st_s32(&sh.id[at], i, first);
        }
      }
    };
    if (a.m >= floor && a.m != -INFINITY) {
#pragma unroll 4
      for (int q = 0; q < slot; ++q)
        if (sh.slot[q][threadIdx.x] >= floor) {
          const int at = atomicAdd(&sh.hot_n, 1);
          if (at < kHot) sh.hot[at] = q * THREADS + threadIdx.x;
        }
      if (fmaxf(one, two) >= floor) part.singles(see);
    }
    __syncthreads();
    // one warp per entry: its batches' logits side by side, a lane each
    const int entries = sh.hot_n;
    if (entries > kHot) {
      if (threadIdx.x == 0) add_s32(&sh.n, kList + 1, first);
    } else {
      constexpr int N = Logits<T>::N, kAhead = 4;
      const int pieces = (per_slot * kBatch * N + 31) / 32;  // of an entry, a logit per lane
      for (int i0 = w; i0 < entries * pieces; i0 += kAhead * WARPS) {
        float v[kAhead];
        int at[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {  // loads first: they come from L2 or memory
          const int i = i0 + u * WARPS;
          at[u] = -1;
          v[u] = -INFINITY;
          if (i < entries * pieces) {
            const int entry = pieces == 1 ? i : i / pieces;
            const int t = sh.hot[entry] % THREADS, q = sh.hot[entry] / THREADS;
            const int j = (i - entry * pieces) * 32 + lane;
            const int b = q * per_slot * kBatch + j / N;  // the thread's vector
            const int vec = part.v0 + b * THREADS + t;
            if (j < per_slot * kBatch * N && b < nb * kBatch && vec < part.v1) {
              at[u] = part.first + vec * N + j % N;
              v[u] = Logits<T>::value(x[at[u]]);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) see(v[u], at[u]);
      }
    }
    if (CLUSTER) cluster_sync();
    else __syncthreads();
    if (CLUSTER && rank != 0) return;
    n = sh.n;
  } else {
    if (CLUSTER && rank != 0) return;
    __syncthreads();
  }

  const bool bad = sh.bad;
  const float base = sh.base, log_s = sh.log_s;
  for (int j = threadIdx.x; j < given; j += THREADS) {
    if (j >= THREADS) {
      id = ids[row * given + j];
      if (id >= 0 && id < V) xid = Logits<T>::value(x[id]);
    }
    lp[row * given + j] = id == -1 ? 0.f : (id < 0 || id >= V || bad) ? NAN : (xid - base) - log_s;
  }
  if (TOP) {
    int base_at = 0;
    if (n > kList) {
      __syncthreads();  // every warp has read sh.n
      const Part<T, THREADS> whole(x, V, 0, 1);
      if (threadIdx.x == 0) sh.n = 0;
      pick_rounds(whole, (whole.v1 - whole.v0 + kBatch * THREADS - 1) / (kBatch * THREADS), k, sh);
      n = sh.n;
      base_at = WARPS;
    }
    // a logit's place is how many rank before it
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const float v = sh.v[base_at + i];
      const int at = sh.id[base_at + i];
      int r = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) r += before(sh.v[base_at + j], sh.id[base_at + j], v, at);
      if (r < k) {
        top_id[row * k + r] = bad ? -1 : at;
        top_lp[row * k + r] = bad ? NAN : (v - base) - log_s;
      }
    }
    for (int r = n + threadIdx.x; r < k; r += THREADS) {
      top_id[row * k + r] = -1;
      top_lp[row * k + r] = bad ? NAN : -INFINITY;
    }
  }
}

template <typename T, bool TOP, bool CLUSTER, int THREADS>
static void launch(const T* logits, long long ld, int rows, int V, const int* ids, int given, int k, int parts,
                   float* lp, float* entropy, float* top_lp, int* top_id, cudaStream_t s) {
  auto kern = token_logprobs_kernel<T, TOP, CLUSTER, THREADS>;
  prefer_max_smem_carveout(reinterpret_cast<const void*>(kern));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attrs[2];
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = sizeof(Shared<THREADS>);
  cfg.stream = s;
  cfg.attrs = attrs;
  if (CLUSTER) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attrs[cfg.numAttrs].val.clusterDim.x = parts;
    attrs[cfg.numAttrs].val.clusterDim.y = 1;
    attrs[cfg.numAttrs].val.clusterDim.z = 1;
    cfg.numAttrs += 1;
  }
  if (pdl_enabled()) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs += 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, logits, ld, V, ids, given, k, parts, lp, entropy, top_lp,
                                           top_id);
  if (e != cudaSuccess) throw std::runtime_error(std::string("token_logprobs launch failed: ") + cudaGetErrorString(e));
}

template <typename T>
static void dispatch(const T* logits, long long ld, int rows, int V, const int* ids, int given, int k, int num_sms,
                     float* lp, float* entropy, float* top_lp, int* top_id, cudaStream_t s) {
  // CTAs per row: eight or four as long as that is at most seven CTAs for four SMs (clusters do
  // not fill the last ones) and each CTA has half a batch. 102,400 bf16 with 20 alternatives:
  // one row takes 6.6 us in eight, 7.4 in four, 12 unsplit; 32 rows 8.9 in eight, 9.3 in four;
  // 64 rows 10.5 in four, 12.7 unsplit; 74 rows 13.0 in four, 12.7 unsplit. In two a row's join
  // eats what its stream gains: 110 rows 13.2 either way, of 32,000 logits 8.2 against 7.1.
  const int batch = kBatch * kLong * Logits<T>::N;
  int parts = kMaxCluster;
  while (parts >= 4 && ((long long)rows * parts * 4 > 7ll * num_sms || V / parts < batch / 2)) parts /= 2;
  if (parts < 4) parts = 1;
  // More short rows than the SMs hold at once take 64 threads each, which leave and are followed
  // sooner (bf16, 20 alternatives): 8,192 rows x 1,000 43 us, in 256 threads 74; 8,192 x 16,384 86
  // and 112; 2,001 x 16,384 26 and 29, but 1,200 x 16,384 23 and 20, 600 x 8,192 12.7 and 11.5,
  // 8,192 x 65,536 266 and 220.
  const int vectors = V / Logits<T>::N;
  const bool small = parts == 1 && ((rows > kCtasPerSm * num_sms && vectors <= 512) ||
                                    (rows > 3 * kCtasPerSm * num_sms && vectors <= 2048));
  auto run = [&](auto top, auto cluster, auto threads) {
    launch<T, decltype(top)::value, decltype(cluster)::value, decltype(threads)::value>(
        logits, ld, rows, V, ids, given, k, parts, lp, entropy, top_lp, top_id, s);
  };
  using Yes = std::true_type;
  using No = std::false_type;
  const std::integral_constant<int, kLong> wide;
  const std::integral_constant<int, kShort> narrow;
  if (k > 0) parts > 1 ? run(Yes{}, Yes{}, wide) : small ? run(Yes{}, No{}, narrow) : run(Yes{}, No{}, wide);
  else parts > 1 ? run(No{}, Yes{}, wide) : small ? run(No{}, No{}, narrow) : run(No{}, No{}, wide);
}

void token_logprobs(const void* logits, int dtype, long long ld, int rows, int V, const int* ids, int given, int k,
                    int num_sms, float* lp, float* entropy, float* top_lp, int* top_id, cudaStream_t s) {
  if (rows <= 0) return;
  auto run = [&](auto* x) { dispatch(x, ld, rows, V, ids, given, k, num_sms, lp, entropy, top_lp, top_id, s); };
  if (dtype == 0) run(static_cast<const __nv_bfloat16*>(logits));
  else if (dtype == 1) run(static_cast<const __half*>(logits));
  else run(static_cast<const float*>(logits));
}

}  // namespace sp
