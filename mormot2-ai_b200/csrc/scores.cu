// Log probabilities of given tokens, with the entropy and the greatest alternatives, from float32
// logits (the formulas stand in scores.cuh). Every logit is read once, into registers: a cluster of up
// to eight CTAs shares a row, a thread holds 40 values of it at a time. Over the block's maximum they are
// added up; the alternatives are picked out by a bar that at least `top` of them pass. The cluster's
// first CTA then joins the parts through distributed shared memory, so that one launch does it all.
#include "scores.cuh"

MB_DEFINE_LAST_ERROR

#define SC_THREADS 256
#define SC_WARPS (SC_THREADS / 32)
#define SC_EACH 40                      // values of a thread in a round
#define SC_ROUND (SC_THREADS * SC_EACH)
#define SC_ROOM 512                     // values that may pass the bar; more are picked one by one
#define SC_CLUSTER 8

__device__ __forceinline__ uint32_t sc_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t sc_at_leader(const void* p) {     // this shared address in CTA 0
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(0));
  return r;
}
__device__ __forceinline__ void sc_put(uint32_t at, TopKey v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
__device__ __forceinline__ void sc_put(uint32_t at, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}
__device__ __forceinline__ void sc_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void sc_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The `top`-th greatest of the warp's values, each lane one
__device__ __forceinline__ float warp_nth(float v, int top) {
  const int lane = threadIdx.x & 31;
  int above = 0;
#pragma unroll
  for (int i = 1; i < 32; ++i) above += __shfl_sync(0xffffffffu, v, (lane + i) & 31) > v;
  float least = above < top ? v : INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  return least;
}

#define SC_FEW 8       // alternatives up to which the warps' bars are near enough

struct ScShared {
  float best[2][SC_WARPS], bar[2][SC_WARPS], s[SC_WARPS], t[SC_WARPS];
  alignas(16) uint32_t place[SC_ROOM];      // of the keys that passed the bar, and their ids
  uint32_t id[SC_ROOM];
  alignas(16) uint32_t heads[SC_THREADS];   // the threads' greatest values that passed the warps' bars
  TopKey sorted[MB_SCORES_TOP], pick[SC_WARPS];
  int taken[MB_SCORES_TOP], count, n_heads, equal[2];
  uint32_t least;
  // of the cluster's first CTA: every CTA's part
  Mass mass[SC_CLUSTER];
  TopKey keys[SC_CLUSTER][MB_SCORES_TOP];
};

// Values `base` .. of the row's part x[0 .. n): value 4 i + j of a thread is at `place`
template <bool WIDE>
__device__ __forceinline__ int sc_place(int base, int k) {
  return WIDE ? base + 4 * ((k >> 2) * SC_THREADS + threadIdx.x) + (k & 3) : base + k * SC_THREADS + threadIdx.x;
}
template <bool WIDE>
__device__ __forceinline__ void sc_load(const float* __restrict__ x, int base, int n, float* v) {
  if (WIDE) {
#pragma unroll
    for (int i = 0; i < SC_EACH; i += 4) {
      const int at = sc_place<true>(base, i);
      if (at + 4 <= n) {
        const float4 f = *(const float4*)(x + at);
        v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i + j] = at + j < n ? x[at + j] : -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < SC_EACH; ++i) {
      const int at = sc_place<false>(base, i);
      v[i] = at < n ? x[at] : -INFINITY;
    }
  }
}

// How many of list[0 .. n) are above p
__device__ __forceinline__ int sc_above(const uint32_t* list, int n, uint32_t p) {
  int above = 0, j = 0;
  for (; j + 4 <= n; j += 4) {
    const uint4 q = *(const uint4*)(list + j);
    above += (q.x > p) + (q.y > p) + (q.z > p) + (q.w > p);
  }
  for (; j < n; ++j) above += list[j] > p;
  return above;
}

// The `top` greatest of the `n` keys in sh.place and sh.id, in order into sh.sorted: a key's place is the
// number of keys above it, for which its value alone is looked at unless two are equal.
__device__ __forceinline__ void sc_sort(int n, int top, int parity, ScShared& sh) {
  for (int i = threadIdx.x; i < n; i += SC_THREADS) {
    const uint32_t p = sh.place[i];
    const int above = sc_above(sh.place, n, p);
    if (above < top) {
      sh.sorted[above] = (TopKey)p << 32 | sh.id[i];
      if (atomicAdd(&sh.taken[above], 1) > 0) sh.equal[parity] = 1;
    }
  }
  __syncthreads();
  if (!sh.equal[parity]) return;
  for (int i = threadIdx.x; i < n; i += SC_THREADS) {
    const TopKey k = (TopKey)sh.place[i] << 32 | sh.id[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += ((TopKey)sh.place[j] << 32 | sh.id[j]) > k;
    if (above < top) sh.sorted[above] = k;
  }
  __syncthreads();
}

// The same of the round's values themselves, where so many passed that they were not noted (many equal
// ones, or large ones side by side): the greatest below the last one, `top` times. They are read again.
__device__ __noinline__ void sc_pick(const float* __restrict__ x, int base, int n, int id0, int held, int top,
                                     ScShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const TopKey old = threadIdx.x < held ? sh.sorted[threadIdx.x] : 0;
  const int end = min(n, base + SC_ROUND);
  TopKey last = ~(TopKey)0;
  for (int r = 0; r < top; ++r) {
    TopKey k = old < last ? old : 0;
    for (int i = base + threadIdx.x; i < end; i += SC_THREADS) {
      const float v = x[i];
      const TopKey c = v > -INFINITY ? key_of(v, id0 + i) : 0;
      if (c < last && c > k) k = c;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const TopKey c = __shfl_xor_sync(0xffffffffu, k, o);
      if (c > k) k = c;
    }
    __syncthreads();
    if (lane == 0) sh.pick[warp] = k;
    __syncthreads();
    last = 0;
    for (int w = 0; w < SC_WARPS; ++w)
      if (sh.pick[w] > last) last = sh.pick[w];
    if (threadIdx.x == 0) sh.sorted[r] = last;
  }
  __syncthreads();
}

template <bool WIDE, bool TOP>
__device__ __forceinline__ Mass sc_part(const float* __restrict__ x, int n, int id0, int top, ScShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = -INFINITY, s = 0.f, t = 0.f;
  float bar = -3.402823466e38f;        // the lowest finite value: -infinity and NaN never pass
  int held = 0;                        // keys in sh.sorted
  for (int base = 0, parity = 0; base < n; base += SC_ROUND, parity ^= 1) {
    float v[SC_EACH];
    sc_load<WIDE>(x, base, n, v);
    float best = v[0];
#pragma unroll
    for (int i = 1; i < SC_EACH; ++i) best = fmaxf(best, v[i]);
    const float most_warp = warp_max(best);
    const float nth = TOP ? top == 1 ? most_warp : warp_nth(best, top) : 0.f;
    if (lane == 0) {
      sh.best[parity][warp] = most_warp;
      if (TOP) sh.bar[parity][warp] = nth;
    }
    if (TOP) {
      if (threadIdx.x < MB_SCORES_TOP) sh.taken[threadIdx.x] = 0;
      if (threadIdx.x == 0) sh.count = held, sh.n_heads = 0, sh.equal[parity] = 0, sh.least = ~0u;
      if (threadIdx.x < held) {
        sh.place[threadIdx.x] = (uint32_t)(sh.sorted[threadIdx.x] >> 32);
        sh.id[threadIdx.x] = (uint32_t)sh.sorted[threadIdx.x];
      }
    }
    __syncthreads();
    float most = m;
#pragma unroll
    for (int w = 0; w < SC_WARPS; ++w) {
      most = fmaxf(most, sh.best[parity][w]);
      if (TOP) bar = fmaxf(bar, sh.bar[parity][w]);
    }
    if (TOP && top > SC_FEW) {
      // The `top`-th of the threads' greatest values is a bar too, and one that few others pass; only those
      // that pass the warps' bars (at least `top` do, if so many are finite) can be above it.
      const uint32_t p = key_place(best);
      if (best >= bar) sh.heads[atomicAdd(&sh.n_heads, 1)] = p;
      __syncthreads();
      const int heads = sh.n_heads;
      if (best >= bar && sc_above(sh.heads, heads, p) < top) atomicMin(&sh.least, p);
      __syncthreads();
      if (heads >= top) bar = fmaxf(bar, key_value((TopKey)sh.least << 32));
    }
    if (TOP && best >= bar) {
      int mine = 0;
#pragma unroll
      for (int i = 0; i < SC_EACH; ++i) mine += v[i] >= bar;
      int to = atomicAdd(&sh.count, mine);
      if (to + mine <= SC_ROOM) {
#pragma unroll
        for (int i = 0; i < SC_EACH; ++i)
          if (v[i] >= bar) {
            sh.place[to] = key_place(v[i]);
            sh.id[to++] = ~(uint32_t)(id0 + sc_place<WIDE>(base, i));
          }
      }
    }
    const Mass before = mass_over({m, s, t}, most);
    m = most, s = before.s, t = before.t;
    mass_add<SC_EACH>(v, m == -INFINITY ? 0.f : m, s, t);
    if (!TOP) continue;
    __syncthreads();
    const int passed = sh.count;       // the keys held among them
    if (passed <= SC_ROOM) {
      sc_sort(passed, top, parity, sh);
      held = min(top, passed);
    } else {
      sc_pick(x, base, n, id0, held, top, sh);
      held = top;
    }
    if (held == top) bar = fmaxf(bar, key_value(sh.sorted[top - 1]));
  }
  // keys that are not there are 0
  if (TOP && threadIdx.x < top && threadIdx.x >= held) sh.sorted[threadIdx.x] = 0;
  s = warp_sum(s);
  t = warp_sum(t);
  if (lane == 0) sh.s[warp] = s, sh.t[warp] = t;
  __syncthreads();
  s = warp_sum(lane < SC_WARPS ? sh.s[lane] : 0.f);
  t = warp_sum(lane < SC_WARPS ? sh.t[lane] : 0.f);
  return {m, s, t};
}

template <bool TOP>
__global__ void __launch_bounds__(SC_THREADS, 4)
token_scores_kernel(const float* __restrict__ logits, size_t stride, int V, int parts, int per,
                    const int* __restrict__ tokens, int top, ScoreOut out) {
  mb_grid_wait();
  mb_grid_launch_next();
  __shared__ ScShared sh;
  if (parts > 1) sc_arrive();                  // every CTA of the cluster has begun: see the wait
  const int row = blockIdx.x / parts, part = parts > 1 ? (int)sc_rank() : 0;
  const float* x = logits + (size_t)row * stride;
  float given = __uint_as_float(0x7fc00000u);
  if (part == 0 && threadIdx.x == 0) {         // asked for ahead of everything
    const int token = tokens[row];
    if (token >= 0 && token < V) given = x[token];
  }
  const int i0 = part * per, n = max(0, min(per, V - i0));
  const bool wide = ((uintptr_t)x & 15) == 0;
  const Mass v = wide ? sc_part<true, TOP>(x + i0, n, i0, top, sh) : sc_part<false, TOP>(x + i0, n, i0, top, sh);
  if (parts > 1) {
    sc_wait();
    if (threadIdx.x == 0) {
      sc_put(sc_at_leader(&sh.mass[part].m), v.m);
      sc_put(sc_at_leader(&sh.mass[part].s), v.s);
      sc_put(sc_at_leader(&sh.mass[part].t), v.t);
    }
    if (TOP && threadIdx.x < top) sc_put(sc_at_leader(&sh.keys[part][threadIdx.x]), sh.sorted[threadIdx.x]);
    sc_arrive();
    sc_wait();
    if (part > 0) return;
  } else {
    if (threadIdx.x == 0) sh.mass[0] = v;
    if (TOP && threadIdx.x < top) sh.keys[0][threadIdx.x] = sh.sorted[threadIdx.x];
    __syncthreads();
  }
  if (threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  Mass all = lane < parts ? sh.mass[lane] : mass_none();
#pragma unroll
  for (int o = SC_CLUSTER / 2; o > 0; o >>= 1)
    all = mass_join(all, {__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o),
                          __shfl_xor_sync(0xffffffffu, all.t, o)});
  TopKey mine = 0;
  if (TOP) {      // every part's keys are in order: the greatest of their heads, `top` times
    int head = 0;
    for (int j = 0; j < top; ++j) {
      const TopKey k = lane < parts && head < top ? sh.keys[lane][head] : 0;
      TopKey best = k;
#pragma unroll
      for (int o = SC_CLUSTER / 2; o > 0; o >>= 1) {
        const TopKey c = __shfl_xor_sync(0xffffffffu, best, o);
        if (c > best) best = c;
      }
      best = __shfl_sync(0xffffffffu, best, 0);
      if (k == best) ++head;
      if (lane == j) mine = best;
    }
  }
  all = {__shfl_sync(0xffffffffu, all.m, 0), __shfl_sync(0xffffffffu, all.s, 0), __shfl_sync(0xffffffffu, all.t, 0)};
  finish_row(all, __shfl_sync(0xffffffffu, given, 0), mine, top, row, out);
}

// For every row r of logits [rows, V] (`stride` values from row to row): logprobs[r] of tokens[r] (NaN
// where that is no token below V), entropy[r], and the `top` greatest values' ids and log
// probabilities. `sms`: the device's multiprocessors.
MB_EXPORT int mb_token_scores(const float* logits, long long stride, int rows, int V,
                              const int* tokens, int top, float* logprobs, float* entropy,
                              int* top_ids, float* top_logprobs, int sms, void* stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || top < 0 || top > MB_SCORES_TOP || top > V)
    MB_FAIL("mb_token_scores: %d alternatives of a vocabulary of %d", top, V);
  // few rows: parts of at least 2,048 values, for the latency; many: whole rounds
  const int least = (long long)rows * 2 < sms ? 2048 : SC_ROUND;
  int parts = 1;
  while (parts < SC_CLUSTER && (long long)parts * least < V) parts *= 2;
  if ((long long)rows * parts > 0x7fffffffll) MB_FAIL("mb_token_scores: %d rows in one call", rows);
  const int per = (((V + parts - 1) / parts) + 3) & ~3;
  const ScoreOut out = {logprobs, entropy, top_ids, top_logprobs};
  cudaError_t e = mb_launch_clusters(top > 0 ? token_scores_kernel<true> : token_scores_kernel<false>,
                                     dim3(rows * parts), dim3(SC_THREADS), 0, (cudaStream_t)stream, parts,
                                     logits, (size_t)stride, V, parts, per, tokens, top, out);
  if (e != cudaSuccess) MB_FAIL("mb_token_scores: %s", cudaGetErrorString(e));
  return 0;
}
