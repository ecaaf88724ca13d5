// Running statistics of a row's logits, shared by the kernels that reduce a row to its log-sum-exp and entropy.
#pragma once
#include "common.cuh"

namespace kf_row {

typedef unsigned long long u64;
constexpr float LOG2E = 1.4426950408889634f;

// max(a, b), NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two 32-bit numbers in one instruction each (sm_100a)
__device__ __forceinline__ u64 pack2(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(u64 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Running maximum (of what is a number), sum of exponentials and sum of d exp(d), and how a second set joins the first.  A NaN
// among the logits is a NaN in s.  A maximum so far below the new one that its terms are 0 beside it leaves nothing: d s may be infinite then (the
// lowest number of all is a common mask), and times 0 it would be NaN.
struct Stats { float m, s, u; };
__device__ __forceinline__ void move_to(Stats& a, float m) {
  if (m != a.m) {
    const float d = a.m - m, f = exp2_fast(d * LOG2E);
    a.u = f == 0.f ? 0.f : f * (a.u + d * a.s);
    a.s *= f;
    a.m = m;
  }
}
__device__ __forceinline__ void join(Stats& a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  move_to(a, m);
  move_to(b, m);
  a.s += b.s;
  a.u += b.u;
}


// s and u of the numbers `get(0) .. get(N - 1)` join `a`, whose maximum already counts them.  exp(-200) is 0 in 32 bits, and
// 0 * -200 is 0: a masked column (-inf) adds nothing.
template <int N, typename F>
__device__ __forceinline__ void add_exponentials(Stats& a, F get) {
  const float ref = a.m == -INFINITY ? 0.f : a.m;
  const u64 minus = pack2(-ref, -ref), scale = pack2(LOG2E, LOG2E);
  u64 s2 = 0ull, u2 = 0ull;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float2 d = unpack2(add2(pack2(get(i), get(i + 1)), minus));
    const u64 low = pack2(max_nan(d.x, -200.f), max_nan(d.y, -200.f));
    d = unpack2(mul2(low, scale));
    const u64 w = pack2(exp2_fast(d.x), exp2_fast(d.y));
    s2 = add2(s2, w);
    u2 = fma2(low, w, u2);
  }
  const float2 s = unpack2(s2), u = unpack2(u2);
  a.s += s.x + s.y;
  a.u += u.x + u.y;
}

// The results for a token whose logit is `given` (NaN for one that is no column).  NaN and +inf among the logits give NaN.
__device__ __forceinline__ bool is_no_distribution(const Stats& a) { return a.s != a.s || a.m == INFINITY; }
__device__ __forceinline__ float row_logprob(const Stats& a, float given) {
  if (is_no_distribution(a)) return __int_as_float(0x7fffffff);
  if (a.m == -INFINITY) return given == given ? -INFINITY : given;
  return (given - a.m) - logf(a.s);
}
__device__ __forceinline__ float row_entropy(const Stats& a) {
  if (is_no_distribution(a)) return __int_as_float(0x7fffffff);
  return a.m == -INFINITY ? 0.f : logf(a.s) - a.u / a.s;
}

}  // namespace kf_row
