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

__device__ __forceinline__ Mass mass_none() { return {-INFINITY, 0.f, 0.f}; }

// The two parts' mass over their common maximum. A part that weighs nothing beside the other (all of it
// -infinity, or the type's lowest value) adds nothing, but a NaN stays one.
__device__ __forceinline__ Mass mass_over(Mass a, float m) {
  const float d = a.m - m, e = a.m == -INFINITY ? 0.f : expf(d);
  return {m, e * a.s, e > 0.f ? e * fmaf(d, a.s, a.t) : e * a.s};
}
__device__ __forceinline__ Mass mass_join(Mass a, Mass b) {
  const float m = fmaxf(a.m, b.m);
  a = mass_over(a, m);
  b = mass_over(b, m);
  return {m, a.s + b.s, a.t + b.t};
}

// One value onto a mass whose maximum `m` is final (0 stands for -infinity): -infinity adds nothing,
// a NaN stays.
__device__ __forceinline__ void mass_add(float x, float m, float& s, float& t) {
  const float d = x - m, e = __expf(d);
  s += e;
  t = fmaf(e, fmaxf(d, -1e30f), t);
}

__device__ __forceinline__ Mass mass_warp(Mass v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Mass w;
    w.m = __shfl_xor_sync(0xffffffffu, v.m, o);
    w.s = __shfl_xor_sync(0xffffffffu, v.s, o);
    w.t = __shfl_xor_sync(0xffffffffu, v.t, o);
    v = mass_join(v, w);
  }
  return v;
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
__device__ __forceinline__ TopKey key_max_warp(TopKey k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const TopKey c = __shfl_xor_sync(0xffffffffu, k, o);
    if (c > k) k = c;
  }
  return k;
}

__device__ TopKey block_key_max(TopKey k, TopKey* sh) {
  k = key_max_warp(k);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  __syncthreads();
  if (lane == 0) sh[warp] = k;
  __syncthreads();
  k = sh[0];
  for (int w = 1; w < warps; ++w)
    if (sh[w] > k) k = sh[w];
  return k;
}
__device__ Mass block_mass(Mass v, Mass* sh) {
  v = mass_warp(v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < warps; ++w) v = mass_join(v, sh[w]);
  return v;
}

struct ScoreOut {
  float *logprobs, *entropy;
  int* top_ids;
  float* top_logprobs;
};

// A block of 128 threads joins the parts of a row: their masses and, in any order, their keys.
// `given`: the given token's logit, a NaN where there is none.
__device__ void join_parts(const Mass* mass, const TopKey* keys, int parts, int top, float given, int row,
                           const ScoreOut& out) {
  __shared__ Mass sh_mass[4];
  __shared__ TopKey sh_key[4];
  Mass v = mass_none();
  for (int p = threadIdx.x; p < parts; p += 128) v = mass_join(v, mass[p]);
  v = block_mass(v, sh_mass);
  const float ln_s = logf(v.s);
  if (threadIdx.x == 0) {
    out.logprobs[row] = given - v.m - ln_s;
    const float h = ln_s - v.t / v.s;
    out.entropy[row] = h < 0.f ? 0.f : h;
  }
  TopKey last = ~(TopKey)0;
  for (int j = 0; j < top; ++j) {
    TopKey best = 0;
    for (int i = threadIdx.x; i < parts * top; i += 128) {
      const TopKey k = keys[i];
      if (k < last && k > best) best = k;
    }
    last = block_key_max(best, sh_key);
    if (threadIdx.x == 0) {
      out.top_ids[(size_t)row * top + j] = key_id(last);
      out.top_logprobs[(size_t)row * top + j] = key_value(last) - v.m - ln_s;
    }
  }
}
