// What a row of logits says of its tokens, in parts that join: the maximum M of the values, S = sum
// exp(x - M), T = sum exp(x - M) (x - M), and the greatest values as keys. From the whole row
//   log p(t) = x_t - M - ln S,     entropy = ln S - T / S
// and the alternatives in the order of the keys. A NaN, or +infinity, makes S a NaN and with it
// every number of the row; a row of nothing but -infinity has no distribution (NaN too).
#pragma once
#include "common.cuh"

#define MB_SCORES_TOP 32     // alternatives at most

struct Mass {
  float m, s, t;
};

__device__ __forceinline__ f32_pair pair_add(f32_pair a, f32_pair b) {
  f32_pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^y; what is below the smallest normal value is 0
__device__ __forceinline__ float exp2_fast(float y) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
  return e;
}

__device__ __forceinline__ Mass mass_none() { return {-INFINITY, 0.f, 0.f}; }

// The two parts' mass over their common maximum. A part that weighs nothing beside the other (all of it
// -infinity, or the type's lowest value) adds nothing, but a NaN stays one.
__device__ __forceinline__ Mass mass_over(Mass a, float m) {
  const float d = a.m - m, e = a.m == -INFINITY ? 0.f : expf(d);
  return {m, e * a.s, e > 0.f ? e * fmaf(d, a.s, a.t) : e * a.s};
}
// Parts that are joined bring S - 1 instead of S: most rows have one value far above all others, and its 1 in
// a sum of 32 bits would round away what ln S = log1p(S - 1) is made of (a log probability of -0.0104 was off by
// 3.5e-7).
__device__ __forceinline__ Mass rest_none() { return {-INFINITY, -1.f, 0.f}; }
__device__ __forceinline__ Mass rest_join(Mass a, Mass b) {
  const bool first = a.m >= b.m;
  const Mass top = first ? a : b, low = first ? b : a;
  const Mass less = mass_over({low.m, low.s + 1.f, low.t}, top.m);
  return {top.m, top.s + less.s, top.t + less.t};
}

// N values onto the sums over a maximum `m` that is final (0 stands for -infinity): s += sum e^(x - m),
// t += sum e^(x - m) (x - m), two at a time. -infinity adds nothing, a NaN stays.
template <int N> __device__ __forceinline__ void mass_add(const float* x, float m, float& s, float& t) {
  const f32_pair less = pair_of(-m, -m);
  f32_pair ps[2] = {0, 0}, pt[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    f32_pair d = pair_add(pair_of(x[j], x[j + 1]), less), y = d;
    pair_mul(y, pair_of(1.4426950408889634f, 1.4426950408889634f));
    const f32_pair e = pair_of(exp2_fast(pair_half(y, 0)), exp2_fast(pair_half(y, 1)));
    d = pair_of(fmaxf(pair_half(d, 0), -1e30f), fmaxf(pair_half(d, 1), -1e30f));
    ps[(j >> 1) & 1] = pair_add(ps[(j >> 1) & 1], e);
    pair_fma(pt[(j >> 1) & 1], e, d);
  }
  const f32_pair a = pair_add(ps[0], ps[1]), b = pair_add(pt[0], pt[1]);
  s += pair_half(a, 0) + pair_half(a, 1);
  t += pair_half(b, 0) + pair_half(b, 1);
}

// A value and its id as one number: the greater value first, the lowest id among equals, -0 equal to
// +0, a NaN behind everything. 0: no value.
typedef unsigned long long TopKey;
__device__ __forceinline__ uint32_t key_place(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ TopKey key_of(float x, int id) {
  return (TopKey)key_place(x) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ int key_id(TopKey k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(TopKey k) {
  const uint32_t p = (uint32_t)(k >> 32);
  return p == 0u ? __uint_as_float(0x7fc00000u) : __uint_as_float(p & 0x80000000u ? p ^ 0x80000000u : ~p);
}

struct ScoreOut {
  float *logprobs, *entropy;
  int* top_ids;
  float* top_logprobs;
};

// What a warp makes of a row's joined mass (S - 1 in place of S), the given token's logit (a NaN where there
// is none) and the greatest values in order, lane j the j-th's key (0 where there are no more). What is left
// then are values of -infinity (or NaNs, in a row whose numbers are NaN anyway): the lowest ids that are not listed.
__device__ __forceinline__ void finish_row(Mass v, float given, TopKey key, int top, int row,
                                           const ScoreOut& out) {
  const int lane = threadIdx.x & 31;
  const float ln_s = log1pf(v.s);
  if (lane == 0) {
    out.logprobs[row] = given - v.m - ln_s;
    const float h = ln_s - v.t / (1.f + v.s);
    out.entropy[row] = h < 0.f ? 0.f : h;
  }
  if (top == 0) return;
  int id = key_id(key);
  float value = key_value(key);
  const unsigned found = __ballot_sync(0xffffffffu, key != 0 && lane < top);
  for (int j = __popc(found), next = 0; j < top; ++j, ++next) {
    while (__any_sync(0xffffffffu, lane < j && id == next)) ++next;
    if (lane == j) {
      id = next;
      value = -INFINITY;
    }
  }
  if (lane < top) {
    out.top_ids[(size_t)row * top + lane] = id;
    out.top_logprobs[(size_t)row * top + lane] = value - v.m - ln_s;
  }
}
