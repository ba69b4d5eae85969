// Log probabilities of given tokens, with the entropy and the greatest alternatives, from float32
// logits (the formulas stand in scores.cuh). Two kernels: a row is cut into chunks, whose blocks leave
// a mass and their greatest keys; a block a row joins them.
#include "scores.cuh"

MB_DEFINE_LAST_ERROR

#define SCORE_THREADS 256
#define SCORE_CHUNK 8192

__global__ void __launch_bounds__(SCORE_THREADS)
score_chunks_kernel(const float* __restrict__ logits, size_t stride, int V, int chunk, int top,
                    Mass* __restrict__ mass, TopKey* __restrict__ keys) {
  mb_grid_wait();
  mb_grid_launch_next();
  __shared__ Mass sh_mass[SCORE_THREADS / 32];
  __shared__ TopKey sh_key[SCORE_THREADS / 32];
  const int i0 = blockIdx.y * chunk, n = min(chunk, V - i0);
  const float* x = logits + (size_t)blockIdx.x * stride + i0;
  const size_t part = (size_t)blockIdx.x * gridDim.y + blockIdx.y;
  Mass v = mass_none();
  for (int i = threadIdx.x; i < n; i += SCORE_THREADS) v.m = fmaxf(v.m, x[i]);
  const float m = v.m == -INFINITY ? 0.f : v.m;
  for (int i = threadIdx.x; i < n; i += SCORE_THREADS) mass_add(x[i], m, v.s, v.t);
  v = block_mass(v, sh_mass);
  if (threadIdx.x == 0) mass[part] = v;
  TopKey last = ~(TopKey)0;
  for (int j = 0; j < top; ++j) {
    TopKey best = 0;
    for (int i = threadIdx.x; i < n; i += SCORE_THREADS) {
      const TopKey k = key_of(x[i], i0 + i);
      if (k < last && k > best) best = k;
    }
    last = block_key_max(best, sh_key);
    if (threadIdx.x == 0) keys[part * top + j] = last;
  }
}

__global__ void __launch_bounds__(128)
score_join_kernel(const Mass* __restrict__ mass, const TopKey* __restrict__ keys, int parts, int top,
                  const float* __restrict__ logits, size_t stride, int V,
                  const int* __restrict__ tokens, ScoreOut out) {
  mb_grid_wait();
  mb_grid_launch_next();
  const int row = blockIdx.x, t = tokens[row];
  const bool ok = t >= 0 && t < V;
  const size_t part = (size_t)row * parts;
  join_parts(mass + part, keys + part * top, parts, top,
             ok ? logits[(size_t)row * stride + t] : __uint_as_float(0x7fc00000u), row, out);
}

static int chunks_of(int V) { return (V + SCORE_CHUNK - 1) / SCORE_CHUNK; }

// bytes of scratch that mb_token_scores needs
MB_EXPORT long long mb_token_scores_scratch(int rows, int V, int top) {
  return (long long)rows * chunks_of(V) * (long long)(16 + 8 * top);
}

// For every row r of logits [rows, V] (`stride` values from row to row): logprobs[r] of tokens[r] (NaN
// where that is no token below V), entropy[r], and the `top` greatest values' ids and log
// probabilities. scratch: mb_token_scores_scratch bytes, 16-byte aligned.
MB_EXPORT int mb_token_scores(const float* logits, long long stride, int rows, int V,
                              const int* tokens, int top, float* logprobs, float* entropy,
                              int* top_ids, float* top_logprobs, void* scratch,
                              long long scratch_bytes, void* stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || top < 0 || top > MB_SCORES_TOP || top > V)
    MB_FAIL("mb_token_scores: %d alternatives of a vocabulary of %d", top, V);
  if (scratch_bytes < mb_token_scores_scratch(rows, V, top))
    MB_FAIL("mb_token_scores: %lld bytes of scratch", scratch_bytes);
  cudaStream_t s = (cudaStream_t)stream;
  const int parts = chunks_of(V);
  TopKey* keys = (TopKey*)scratch;
  Mass* mass = (Mass*)(keys + (size_t)rows * parts * top);
  mb_launch(score_chunks_kernel, dim3(rows, parts), dim3(SCORE_THREADS), 0, s, logits, (size_t)stride,
            V, SCORE_CHUNK, top, mass, keys);
  mb_launch(score_join_kernel, dim3(rows), dim3(128), 0, s, mass, keys, parts, top, logits,
            (size_t)stride, V, tokens, ScoreOut{logprobs, entropy, top_ids, top_logprobs});
  MB_CHECK_LAUNCH("mb_token_scores");
}
