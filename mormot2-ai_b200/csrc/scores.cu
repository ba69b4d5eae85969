// Log probabilities of given tokens, with the entropy and the greatest alternatives, from float32
// logits (the formulas stand in scores.cuh). Every logit is read once, into registers: a cluster of up
// to eight CTAs shares a row, a thread holds 24 or 40 values of it at a time. They are added up over the
// thread's maximum; the alternatives are picked out by a bar that at least `top` of them pass. The cluster's
// first CTA then joins the parts through distributed shared memory, so that one launch does it all.
//
// Bound: many rows by the logits' bytes (2,048 rows of 151,936: 175 us without alternatives, 7.1 TB/s, 198 with
// 5, 226 with 20); few rows by the chain of barriers from the first value to the last sum (one row: 4.1 us
// without, 8.3 with 5). Taken back: CTAs that stay for several rows and ask for the next row ahead (the
// values asked for take the registers of a CTA: 303 us where CTAs that go take 223), the rest of a row
// brought into L2 while the first values are looked at (237), a place in the list for a whole warp at a time
// (204), keys put in order only at a part's end (273 where every round's take 265).
#include "scores.cuh"

MB_DEFINE_LAST_ERROR

#define SC_THREADS 256
#define SC_WARPS (SC_THREADS / 32)
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
__device__ __forceinline__ void sc_put(uint32_t at, uint32_t v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
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
  int above = 0;
#pragma unroll
  for (int i = 1; i < 32; ++i) above += __shfl_xor_sync(0xffffffffu, v, i) > v;
  float least = above < top ? v : INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  return least;
}

// The `nth` greatest of the warp's values, each lane one, for a small `nth`
__device__ __forceinline__ float warp_few(float v, int nth) {
  const int lane = threadIdx.x & 31;
  float m = warp_max(v);
  for (int i = 1; i < nth; ++i) {
    if (lane == __ffs(__ballot_sync(0xffffffffu, v == m)) - 1) v = -INFINITY;
    m = warp_max(v);
  }
  return m;
}

struct ScShared {
  float best[SC_WARPS], bar[SC_WARPS];
  alignas(16) uint32_t place[SC_ROOM];      // of the keys held, in order, and of those that passed the bar
  uint32_t id[SC_ROOM];                     // and their ids
  TopKey sorted[MB_SCORES_TOP], pick[SC_WARPS];
  int taken[MB_SCORES_TOP], passed[3], equal[2], tops[SC_WARPS];
  float most[SC_WARPS], s[SC_WARPS], t[SC_WARPS];
  // of the cluster's first CTA: every CTA's part
  Mass mass[SC_CLUSTER];
  alignas(16) uint32_t all_place[SC_CLUSTER * MB_SCORES_TOP];
  uint32_t all_id[SC_CLUSTER * MB_SCORES_TOP];
};

// Values `base` .. of the row's part x[0 .. n): value 4 i + j of a thread is at `place`
template <bool WIDE>
__device__ __forceinline__ int sc_place(int base, int k) {
  return WIDE ? base + 4 * ((k >> 2) * SC_THREADS + threadIdx.x) + (k & 3) : base + k * SC_THREADS + threadIdx.x;
}
template <int EACH, bool WIDE>
__device__ __forceinline__ void sc_load(const float* __restrict__ x, int base, int n, float* v) {
  if (WIDE) {
#pragma unroll
    for (int i = 0; i < EACH; i += 4) {
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
    for (int i = 0; i < EACH; ++i) {
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

// The `top` greatest of `n` keys, in order into sh.sorted: a key's place is the number of keys above it,
// for which its value alone is looked at unless two are equal. `turn` counts these calls (sh.taken and
// sh.equal[turn & 1] are 0 before each).
__device__ __forceinline__ void sc_sort(const uint32_t* place, const uint32_t* id, int n, int top, int turn,
                                        ScShared& sh) {
  for (int i = threadIdx.x; i < n; i += SC_THREADS) {
    const uint32_t p = place[i];
    const int above = sc_above(place, n, p);
    if (above < top) {
      sh.sorted[above] = (TopKey)p << 32 | id[i];
      if (atomicAdd(&sh.taken[above], 1) > 0) sh.equal[turn & 1] = 1;
    }
  }
  __syncthreads();
  const int equal = sh.equal[turn & 1];
  if (threadIdx.x < MB_SCORES_TOP) sh.taken[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.equal[(turn + 1) & 1] = 0;
  if (!equal) return;
  for (int i = threadIdx.x; i < n; i += SC_THREADS) {
    const TopKey k = (TopKey)place[i] << 32 | id[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += ((TopKey)place[j] << 32 | id[j]) > k;
    if (above < top) sh.sorted[above] = k;
  }
  __syncthreads();
}

// The same of the round's values themselves, where so many passed that they were not noted (many equal
// ones, or large ones side by side): the greatest below the last one, `top` times. They are read again.
__device__ __noinline__ void sc_pick(const float* __restrict__ x, int base, int end, int id0, int held, int top,
                                     ScShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const TopKey old = threadIdx.x < held ? sh.sorted[threadIdx.x] : 0;
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

// What a CTA finds in its part of a row, x[0 .. n) with ids from id0 on: the mass (every thread has it, S - 1
// in place of S), and in sh.sorted the greatest `top` keys in order, 0 where there are no more finite values.
//
// The first round sets a bar that few values pass and the `top` greatest do: with every warp's ceil(top / 8)
// greatest threads there are `top`, so the least of these threads' greatest values is one (of 10,240 values
// some 45 pass it for 20 alternatives, where the `top`-th thread of the best warp lets 200 pass). From then
// on the bar is the `top`-th greatest value so far, which hardly any value passes, and a round costs what the
// sums cost, and one barrier. Each thread's sums are over the greatest value that it has seen itself.
template <int EACH, bool WIDE, bool TOP>
__device__ __forceinline__ Mass sc_part(const float* __restrict__ x, int n, int id0, int top, int& turn, ScShared& sh) {
  constexpr int ROUND = SC_THREADS * EACH;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Mass mine = mass_none();
  float bar = -3.402823466e38f;        // the lowest finite value: -infinity and NaN never pass
  int held = 0, third = 0;             // keys in sh.sorted; the round's counter of three
  if (TOP) {
    if (threadIdx.x < MB_SCORES_TOP) sh.taken[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.passed[0] = sh.equal[0] = 0;
  }
  for (int base = 0; base < n; base += ROUND) {
    float v[EACH];
    sc_load<EACH, WIDE>(x, base, n, v);
    float best = v[0];
#pragma unroll
    for (int i = 1; i < EACH; ++i) best = fmaxf(best, v[i]);
    if (TOP && base == 0) {
      // Every warp's so many greatest threads together are `top` threads or more (for one, the best will do).
      const float few = warp_few(best, (top + SC_WARPS - 1) / SC_WARPS);
      if (lane == 0) sh.best[warp] = few > -INFINITY ? few : -INFINITY;       // (a NaN is none)
      __syncthreads();
      float least = sh.best[0];
#pragma unroll
      for (int w = 1; w < SC_WARPS; ++w) least = top == 1 ? fmaxf(least, sh.best[w]) : fminf(least, sh.best[w]);
      if (least > -INFINITY) {
        bar = fmaxf(bar, least);
      } else {
        // a warp without so many finite values: the `top`-th of the best warp's threads
        const float nth = warp_nth(best, top);
        if (lane == 0) sh.bar[warp] = nth;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SC_WARPS; ++w) bar = fmaxf(bar, sh.bar[w]);
      }
    }
    if (TOP && best >= bar) {
      // four at a time: hardly any pass
#pragma unroll
      for (int i = 0; i < EACH; i += 4) {
        if (!(fmaxf(fmaxf(v[i], v[i + 1]), fmaxf(v[i + 2], v[i + 3])) >= bar)) continue;
#pragma unroll
        for (int j = i; j < i + 4; ++j)
          if (v[j] >= bar) {
            const int to = held + atomicAdd(&sh.passed[third], 1);
            if (to < SC_ROOM) {
              sh.place[to] = key_place(v[j]);
              sh.id[to] = ~(uint32_t)(id0 + sc_place<WIDE>(base, j));
            }
          }
      }
    }
    if (best > mine.m) mine = mass_over(mine, best);
    mass_add<EACH>(v, mine.m == -INFINITY ? 0.f : mine.m, mine.s, mine.t);
    if (!TOP) continue;
    const int next = third == 2 ? 0 : third + 1;
    if (threadIdx.x == 0) sh.passed[next] = 0;      // read two rounds ago, a barrier ago by all
    __syncthreads();
    const int passed = sh.passed[third];
    third = next;
    if (passed == 0) continue;
    if (held + passed <= SC_ROOM) {
      sc_sort(sh.place, sh.id, held + passed, top, turn++, sh);
      held = min(top, held + passed);
    } else {
      sc_pick(x, base, min(n, base + ROUND), id0, held, top, sh);
      held = top;
    }
    if (threadIdx.x < held) {
      sh.place[threadIdx.x] = (uint32_t)(sh.sorted[threadIdx.x] >> 32);
      sh.id[threadIdx.x] = (uint32_t)sh.sorted[threadIdx.x];
    }
    // what is to come has to be above the last of them (the next value up: equal ones come later)
    if (held == top) bar = key_value(((sh.sorted[top - 1] >> 32) + 1) << 32);
  }
  if (TOP && threadIdx.x < top && threadIdx.x >= held) sh.sorted[threadIdx.x] = 0;
  const float most_warp = warp_max(mine.m);
  if (lane == 0) sh.most[warp] = most_warp;
  __syncthreads();
  float most = sh.most[0];
#pragma unroll
  for (int w = 1; w < SC_WARPS; ++w) most = fmaxf(most, sh.most[w]);
  // (a thread's sums have its own greatest value's 1 in them: see rest_join)
  const unsigned tops = __ballot_sync(0xffffffffu, mine.m == most);
  if (lane == 0) sh.tops[warp] = __popc(tops);
  mine = mine.m == most ? Mass{most, mine.s - 1.f, mine.t} : mass_over(mine, most);
  mine.s = warp_sum(mine.s);
  mine.t = warp_sum(mine.t);
  if (lane == 0) sh.s[warp] = mine.s, sh.t[warp] = mine.t;
  __syncthreads();
  mine = {most, 0.f, 0.f};
  int all = -1;
#pragma unroll
  for (int w = 0; w < SC_WARPS; ++w) mine.s += sh.s[w], mine.t += sh.t[w], all += sh.tops[w];
  mine.s += (float)all;
  return mine;
}

template <int EACH, int CTAS, bool TOP>
__global__ void __launch_bounds__(SC_THREADS, CTAS)
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
  int turn = 0;
  const Mass v = wide ? sc_part<EACH, true, TOP>(x + i0, n, i0, top, turn, sh)
                      : sc_part<EACH, false, TOP>(x + i0, n, i0, top, turn, sh);
  if (parts > 1) {
    sc_wait();
    if (threadIdx.x == 0) {
      sc_put(sc_at_leader(&sh.mass[part].m), v.m);
      sc_put(sc_at_leader(&sh.mass[part].s), v.s);
      sc_put(sc_at_leader(&sh.mass[part].t), v.t);
    }
    if (TOP && threadIdx.x < top) {
      const TopKey k = sh.sorted[threadIdx.x];
      sc_put(sc_at_leader(&sh.all_place[part * top + threadIdx.x]), (uint32_t)(k >> 32));
      sc_put(sc_at_leader(&sh.all_id[part * top + threadIdx.x]), (uint32_t)k);
    }
    sc_arrive();
    sc_wait();
    if (part > 0) return;
    if (TOP) {
      if (threadIdx.x < top) sh.sorted[threadIdx.x] = 0;      // there may be fewer keys
      __syncthreads();
      sc_sort(sh.all_place, sh.all_id, parts * top, top, turn, sh);
    }
  } else {
    if (threadIdx.x == 0) sh.mass[0] = v;
    __syncthreads();
  }
  if (threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  Mass all = lane < parts ? sh.mass[lane] : rest_none();
#pragma unroll
  for (int o = SC_CLUSTER / 2; o > 0; o >>= 1)
    all = rest_join(all, {__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o),
                          __shfl_xor_sync(0xffffffffu, all.t, o)});
  const TopKey mine = TOP && lane < top ? sh.sorted[lane] : 0;
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
  // 24 values a thread leave room for five CTAs on a multiprocessor, whose loads cover each other's barriers;
  // where a few rows in eight parts each fit the device at once all the same, and a part would take three
  // rounds of 24, it takes fewer of 40. 5 alternatives, us with 40 | 24: of 151,936 values 1 row 8.1 | 10.2,
  // 64 rows 15.6 | 17.3, 300 rows 54 | 42, 2,048 rows 220 | 197; 37 rows of 50,257 8.9 | 8.7, 64 of 32,768
  // 9.1 | 7.9.
  const bool few = (long long)rows * SC_CLUSTER <= 4 * sms && V > 65536;
  // As many parts a row as make the rounds of CTAs the shortest, a part's start and end counting as 4,096
  // values, and none of less than 2,048.
  const int slots = (few ? 4 : 5) * sms;
  int parts = 1;
  long long cost = 0;
  for (int p = 1; p <= SC_CLUSTER && (p == 1 || (long long)V >= 2048ll * p); p *= 2) {
    const long long c = ((long long)rows * p + slots - 1) / slots * ((V + p - 1) / p + 4096);
    if (p == 1 || c < cost) cost = c, parts = p;
  }
  const int per = (((V + parts - 1) / parts) + 3) & ~3;
  const ScoreOut out = {logprobs, entropy, top_ids, top_logprobs};
  const auto kernel = few ? top > 0 ? token_scores_kernel<40, 4, true> : token_scores_kernel<40, 4, false>
                          : top > 0 ? token_scores_kernel<24, 5, true> : token_scores_kernel<24, 5, false>;
  cudaError_t e = mb_launch_clusters(kernel,
                                     dim3(rows * parts), dim3(SC_THREADS), 0, (cudaStream_t)stream, parts,
                                     logits, (size_t)stride, V, parts, per, tokens, top, out);
  if (e != cudaSuccess) MB_FAIL("mb_token_scores: %s", cudaGetErrorString(e));
  return 0;
}
