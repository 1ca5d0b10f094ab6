// Running maximum, sum and entropy sum of logits, on packed fp32 pairs.
#pragma once
#include "common.cuh"

namespace sp {

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;

using u64t = unsigned long long;

// Packed fp32 pairs (one instruction for two).
SP_DEVI u64t pack2(float a, float b) {
  u64t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
SP_DEVI void unpack2(u64t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
SP_DEVI u64t add2(u64t a, u64t b) {
  u64t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SP_DEVI u64t mul2(u64t a, u64t b) {
  u64t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SP_DEVI u64t fma2(u64t a, u64t b, u64t c) {
  u64t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// max that keeps NaN
SP_DEVI float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Running sums of a thread: terms 2^u, u = (x - m) log2 e, in hi + lo, and terms 2^u u in e, with
// add_long in e + el.
struct LogprobSums {
  float m = -INFINITY, hi = 0.f, lo = 0.f, e = 0.f, el = 0.f;

  SP_DEVI void raise(float top) {  // a larger maximum
    if (top > m) {
      const float d = fmaxf((m - top) * kLog2e, -300.f);  // m = -inf: the sums are 0
      const float w = fast_exp2(d);
      e = w * fmaf(hi, d, e);
      el *= w;
      hi *= w;
      lo *= w;
      m = top;
    }
  }
  SP_DEVI float shift() const { return m == -INFINITY ? 0.f : -m; }  // only -inf so far: u = -inf
  // a + b in `a`, what its rounding leaves added to `low`
  static SP_DEVI void keep(float& a, float& low, float b) {
    const float t = a + b, z = t - a;
    low += (a - (t - z)) + (b - z);
    a = t;
  }
  SP_DEVI void add(float s, float f) {
    keep(hi, lo, s);
    e += f;
  }
  // for hundreds of additions, whose roundings would show in the entropy
  SP_DEVI void add_long(float s, float f) {
    keep(hi, lo, s);
    keep(e, el, f);
  }
};

// Adds the terms of two logits. CLAMP bounds u below, so that 0 * u stays 0 for -inf (and for
// differences past fp32's range).
template <bool CLAMP>
SP_DEVI void logprob_terms(float a, float b, u64t shift, u64t& s, u64t& e) {
  u64t u = mul2(add2(pack2(a, b), shift), pack2(kLog2e, kLog2e));
  float u0, u1;
  unpack2(u, u0, u1);
  if (CLAMP) {
    u0 = max_nan(u0, -200.f);
    u1 = max_nan(u1, -200.f);
    u = pack2(u0, u1);
  }
  const u64t p = pack2(fast_exp2(u0), fast_exp2(u1));
  s = add2(s, p);
  e = fma2(p, u, e);
}

}  // namespace sp
