// Where the tokens of a packed step lie, from the lengths of its sequences: per token the index of
// its sequence, its position and its slot; per sequence its first row; and the rows of a page table that
// the sequences grow into. The lengths are added up once a block, by a scan over 1,024 sequences at a time; a
// block then finds the sequence of each of its 1,024 tokens (or pages) by bisection of these sums.
//
// Bound by the launch and by the chain through a block (load, scan, bisection, store); the bytes would take
// less than half a microsecond. In a graph: 4 sequences of 459 tokens 2.1 us, 64 of 16,321 3.2, 700 of 130,552
// 4.1; their pages 2.3, 3.0 and 4.5. Among a program's own launches the host is the limit, at 7 us a call.
#include "common.cuh"

MB_DEFINE_LAST_ERROR

#define INDEX_THREADS 256
#define INDEX_ROUND 1024      // sequences whose sums stand in shared memory at a time
#define INDEX_SPAN 1024       // tokens or pages of a block

// Whole pages for `length` positions, a ring's at most
__device__ __forceinline__ int pages_of(long long length, int ring) {
  const long long n = length <= 0 ? 0 : (length + MB_PAGE - 1) / MB_PAGE;
  return (int)(ring > 0 && n > ring ? ring : n);
}

struct Lengths {        // what a sequence brings: new tokens, or new pages
  const int *past, *fresh, *held;      // held null: tokens
  int ring;
  __device__ __forceinline__ int operator()(int b) const {
    const int n = max(fresh[b], 0);
    if (held == nullptr) return n;
    return max(0, pages_of((long long)past[b] + n, ring) - max(held[b], 0));
  }
};

// The sums of up to INDEX_ROUND sequences from b0 on, each the total before it (sums[n] the total behind
// the last). Every thread takes four neighbouring sequences.
__device__ long long scan_round(const Lengths& len, int b0, int n, long long base, long long* sums,
                                long long* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long v[4], mine = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = 4 * threadIdx.x + j;
    v[j] = i < n ? len(b0 + i) : 0;
    mine += v[j];
  }
  long long up = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long w = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += w;
  }
  __syncthreads();                       // the round before has been read
  if (lane == 31) red[warp] = up;
  __syncthreads();
  long long at = base + up - mine;
  for (int w = 0; w < warp; ++w) at += red[w];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = 4 * threadIdx.x + j;
    if (i < n) sums[i] = at;
    at += v[j];
    if (i == n - 1) sums[n] = at;
  }
  __syncthreads();
  return sums[n];
}

// The last of sums[0 .. n - 1] that is not above i
__device__ __forceinline__ int owner_of(const long long* sums, int n, long long i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(INDEX_THREADS)
step_index_kernel(const int* __restrict__ slots, const int* __restrict__ past,
                  const int* __restrict__ fresh, int B, long long T, int* __restrict__ seq_start,
                  int* __restrict__ tok_seq, int* __restrict__ tok_pos, int* __restrict__ tok_slot) {
  mb_grid_wait();
  mb_grid_launch_next();
  __shared__ long long sums[INDEX_ROUND + 1], red[INDEX_THREADS / 32];
  const long long t0 = (long long)blockIdx.x * INDEX_SPAN, t1 = min(T, t0 + INDEX_SPAN);
  const Lengths len{past, fresh, nullptr, 0};
  long long base = 0;
  if (B == 0 && threadIdx.x == 0) seq_start[0] = 0;
  for (int b0 = 0; b0 < B; b0 += INDEX_ROUND) {
    const int n = min(INDEX_ROUND, B - b0);
    const long long end = scan_round(len, b0, n, base, sums, red);
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i <= n; i += INDEX_THREADS)
        if (i < n || b0 + n == B) seq_start[b0 + i] = (int)sums[i];
    for (long long t = max(t0, base) + threadIdx.x; t < min(t1, end); t += INDEX_THREADS) {
      const int i = owner_of(sums, n, t), b = b0 + i;
      tok_seq[t] = b;
      tok_pos[t] = past[b] + (int)(t - sums[i]);
      tok_slot[t] = slots[b];
    }
    base = end;
    if (blockIdx.x > 0 && base >= t1) break;
  }
}

__global__ void __launch_bounds__(INDEX_THREADS)
map_pages_kernel(int* __restrict__ table, int n_slots, int max_pages, const int* __restrict__ slots,
                 const int* __restrict__ past, const int* __restrict__ fresh,
                 const int* __restrict__ held, int B, const int* __restrict__ pages, int N, int ring) {
  mb_grid_wait();
  mb_grid_launch_next();
  __shared__ long long sums[INDEX_ROUND + 1], red[INDEX_THREADS / 32];
  const long long t0 = (long long)blockIdx.x * INDEX_SPAN, t1 = min((long long)N, t0 + INDEX_SPAN);
  const Lengths len{past, fresh, held, ring};
  long long base = 0;
  for (int b0 = 0; b0 < B; b0 += INDEX_ROUND) {
    const int n = min(INDEX_ROUND, B - b0);
    const long long end = scan_round(len, b0, n, base, sums, red);
    for (long long t = max(t0, base) + threadIdx.x; t < min(t1, end); t += INDEX_THREADS) {
      const int i = owner_of(sums, n, t), b = b0 + i;
      const int slot = slots[b];
      const long long entry = max(held[b], 0) + (t - sums[i]);
      if (slot >= 0 && slot < n_slots && entry < max_pages)
        table[(size_t)slot * max_pages + entry] = pages[t];
    }
    base = end;
    if (base >= t1) break;
  }
}

// The arrays of a step that packs sequences 0 .. B - 1 one after another, `fresh[b]` new tokens each
// (none where that is 0 or less): seq_start [B + 1], and of the first T tokens tok_seq, tok_pos
// (past[b] and on) and tok_slot (slots[b]). Rows behind the last token are left as they are.
MB_EXPORT int mb_step_index(const int* slots, const int* past, const int* fresh, int B, long long T,
                            int* seq_start, int* tok_seq, int* tok_pos, int* tok_slot, void* stream) {
  if (B < 0 || T < 0 || T > 0x7fffffffll) MB_FAIL("mb_step_index: %d sequences, %lld tokens", B, T);
  const int blocks = (int)((T + INDEX_SPAN - 1) / INDEX_SPAN);
  mb_launch(step_index_kernel, dim3(blocks > 0 ? blocks : 1), dim3(INDEX_THREADS), 0,
            (cudaStream_t)stream, slots, past, fresh, B, T, seq_start, tok_seq, tok_pos, tok_slot);
  MB_CHECK_LAUNCH("mb_step_index");
}

// Entries held[b] .. of row slots[b] of table [n_slots, max_pages], up to the whole pages that past[b] +
// fresh[b] positions take (`ring` > 0: at most so many), receive the next of pages [N], sequence
// after sequence. Entries outside the table, and those that `pages` is too short for, are left.
MB_EXPORT int mb_map_pages(int* table, int n_slots, int max_pages, const int* slots, const int* past,
                           const int* fresh, const int* held, int B, const int* pages, int N, int ring,
                           void* stream) {
  if (B < 0 || N < 0 || ring < 0) MB_FAIL("mb_map_pages: %d sequences, %d pages, a ring of %d", B, N, ring);
  if (B == 0 || N == 0) return 0;
  mb_launch(map_pages_kernel, dim3((N + INDEX_SPAN - 1) / INDEX_SPAN), dim3(INDEX_THREADS), 0,
            (cudaStream_t)stream, table, n_slots, max_pages, slots, past, fresh, held, B, pages, N, ring);
  MB_CHECK_LAUNCH("mb_map_pages");
}
