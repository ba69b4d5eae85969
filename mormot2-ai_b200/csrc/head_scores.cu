// Log probabilities of given tokens, entropy and the greatest alternatives straight from the rows
// before the head: the product of rows [R, K] and the head [V, K] (bfloat16, float32 sums) on the
// fifth-generation tensor cores, whose results never leave the chip. What a row has to keep of its V
// logits is a mass (the maximum, S and T of scores.cuh) and `top` keys.
//
// A CTA pair (rank 0 issues tcgen05.mma.cta_group::2 for both) keeps 256 rows and walks a strip of
// the vocabulary in tiles of up to 256 ids; up to 128 rows each CTA walks by itself, in tiles of up to 128.
// 128 threads a CTA own a row each and fold a tile from tensor memory into their row's mass and keys while
// the next tile is multiplied. At the strip's end they leave both in memory; a warp a row joins the strips
// (head_join_kernel).
//
// The pairs that share a strip walk it side by side, so that its weights come from memory once and from
// L2 for all row blocks but the first: a band of b row blocks takes floor(pairs / b) strips. Rows are
// cut into bands such that few pairs idle (plan_bands).
//
// Bound: the tensor cores, from K of some 1,500 on (rows padded to 256; 151,936 ids, 5 alternatives: 1,024 rows of
// 4,096 values 804 us with the tensor pipe 98 % active, weights read once, 1.30 GB; 2,048 rows again and
// again 1.35 PFLOP/s under the power cap, on rows of few bits 1.53). Below that the four warps that read
// tensor memory: some 550 cycles for 32 ids of a row (the exponentials alone take 256), and the lists, some
// 110 instructions a value that goes in (1,024 values a row, 1,001 rows: 195 us without alternatives, 215 with 5,
// 270 with 20). Up to 128 rows the head's bytes (24 rows of 1,024 values: 52 us, 6.0 TB/s; of 4,096:
// 188, 6.6; 128 rows 55 and 214).
// Taken back: two such warps a quarter of the lanes, a tile each in turn (their lists see half the ids each,
// and together nearly twice the new values: 501 us, 656 with 20); ids in a log beside the values in
// registers (810 with 20: every value's way to the log is a branch); values held back in shared memory, 16 a
// row, and put in the lists by all rows at once (333 rows of 1,024 values with 20: 175 us against 172); a CTA by
// itself with tiles of 256 ids (128 rows of 2,048 values 124 us against 115, of 4,096 242 against 223); pairs that
// copy no rows beyond the last one (129 rows of 1,024 values 66 us against 64).
#include "scores.cuh"
#include "tc_common.cuh"

#include <initializer_list>

MB_DEFINE_LAST_ERROR

#define HS_THREADS 192
#define HS_BK 64
#define HS_HALF (128 * HS_BK * 2)            // 128 rows of an operand in a stage
#define HS_RING (12 * HS_HALF)               // of all stages
#define HS_STAGES 12                         // at most
#define HS_STRIPS 160                        // strips of a row at most
#define HS_BLOCKS 64                         // row blocks of a launch at most
#define HS_STAGED (4 * 32 * 128)             // 32 values of 32 rows for each epilogue warp
#define HS_SMEM (1024 + HS_RING + 256 + HS_STAGED)

// A CTA pair multiplies 256 rows with 256 ids, each CTA bringing half of both; a CTA by itself 128 with 128.
__host__ __device__ constexpr int block_rows_of(bool pair) { return pair ? 256 : 128; }

// A band: `blocks` row blocks from `first` on, each in `strips` strips of `width` ids, tiles of `tile`
struct HeadPlan {
  int bands, block_rows;
  int box, stages;           // rows of the head that a CTA copies for a tile, and stages of the ring
  int first[HS_BLOCKS], blocks[HS_BLOCKS], strips[HS_BLOCKS], width[HS_BLOCKS], tile[HS_BLOCKS];
  int part0[HS_BLOCKS];      // where a band's parts begin: [block][row][strips]
};

// The tiles of a pair (or of a CTA by itself), the same for all of its warps
struct HeadWalk {
  const HeadPlan& plan;
  int unit, limit, band, block, strip, n, end;
  __device__ HeadWalk(const HeadPlan& p, int unit_, int limit_) : plan(p), unit(unit_), limit(limit_), band(-1) {
    n = end = 0;
  }
  // its next strip; false when there is none
  __device__ __forceinline__ bool next_strip() {
    while (++band < plan.bands) {
      const int b = plan.blocks[band];
      if (unit >= b * plan.strips[band]) continue;
      block = unit % b;
      strip = unit / b;
      n = strip * plan.width[band];
      end = min(limit, n + plan.width[band]);
      return true;
    }
    return false;
  }
  __device__ __forceinline__ int row0() const { return (plan.first[band] + block) * plan.block_rows; }
  __device__ __forceinline__ int cols() const { return min(plan.tile[band], end - n); }
  __device__ __forceinline__ void step() { n += plan.tile[band]; }
};

// Notes of a row with lists of N places. Its strips share them: each leaves the greatest of its ids so far,
// of four groups apart, in notes of its own or, as a maximum, in some that others use too. Whatever is there, the
// greatest values of as many groups of ids, the `top`-th of them has `top` ids that are no less: no strip needs
// what is below it, and when a strip looks does not show in the results.
__host__ __device__ constexpr int notes_of(int n) { return n <= 8 ? 16 : n <= 16 ? 32 : 64; }

// A row's greatest values so far, in order, in registers: the last `top` of N places (what stands above
// them is never passed). A value goes in where it is greater, so the first of equals stays ahead.
template <int N> struct TopList {
  float v[N];
  int id[N];
  float bar;      // what a value has to pass
  __device__ __forceinline__ void clear(int top) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = i < N - top ? INFINITY : -INFINITY;
      id[i] = -1;
    }
    bar = -INFINITY;
  }
  // One of many groups' greatest values: in the end the least of v is below no more than top - 1 groups
  __device__ __forceinline__ void probe(float x) {
    x = fmaxf(x, -INFINITY);      // of nothing but NaN: none
#pragma unroll
    for (int k = N - 1; k > 0; --k) v[k] = fmaxf(v[k], fminf(v[k - 1], x));
    v[0] = fmaxf(v[0], x);
  }
  // The list anew, with a bar a little below that value: at least `top` values pass it
  __device__ __forceinline__ void start(int top) {
    const float least = v[N - 1];
    clear(top);
    raise(least);
  }
  __device__ __forceinline__ void raise(float least) {
    least = fminf(least, 3e38f);
    if (least > -INFINITY) bar = fmaxf(bar, least - 1e-6f * fabsf(least) - 1e-30f);
  }
  // A bar from the row's notes (0: none yet)
  __device__ __forceinline__ void look(const uint32_t* notes, int top) {
    float u[N];
#pragma unroll
    for (int k = 0; k < N; ++k) u[k] = k < N - top ? INFINITY : -INFINITY;
#pragma unroll
    for (int j0 = 0; j0 < notes_of(N); j0 += 16) {
      uint32_t place[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(place[j]) : "l"(notes + (j0 + j) * 256) : "memory");
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float x = place[j] == 0 ? -INFINITY : key_value((TopKey)place[j] << 32);
#pragma unroll
        for (int k = N - 1; k > 0; --k) u[k] = fmaxf(u[k], fminf(u[k - 1], x));
        u[0] = fmaxf(u[0], x);
      }
    }
    raise(u[N - 1]);
  }
  __device__ __forceinline__ void hush() { bar = INFINITY; }      // a row that is not there
  __device__ __forceinline__ void offer(float x, int i) {
    bool past[N];
#pragma unroll
    for (int k = 0; k < N; ++k) past[k] = x > v[k];
#pragma unroll
    for (int k = N - 1; k > 0; --k) {
      v[k] = past[k - 1] ? v[k - 1] : past[k] ? x : v[k];
      id[k] = past[k - 1] ? id[k - 1] : past[k] ? i : id[k];
    }
    v[0] = past[0] ? x : v[0];
    id[0] = past[0] ? i : id[0];
    bar = fmaxf(bar, v[N - 1]);
  }
  __device__ __forceinline__ void write(TopKey* keys, int top) const {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k >= N - top) keys[k - (N - top)] = id[k] < 0 ? 0 : key_of(v[k], id[k]);
  }
};
template <> struct TopList<0> {
  static constexpr float bar = 0.f;
  __device__ __forceinline__ void clear(int) {}
  __device__ __forceinline__ void probe(float) {}
  __device__ __forceinline__ void start(int) {}
  __device__ __forceinline__ void look(const uint32_t*, int) {}
  __device__ __forceinline__ void hush() {}
  __device__ __forceinline__ void offer(float, int) {}
  __device__ __forceinline__ void write(TopKey*, int) const {}
};

// 32 columns of this thread's lane. The load is one of a whole warp, and the code between two of them leaves lanes
// behind (rows that are not there, values that go into lists): they come together first.
__device__ __forceinline__ void load32(uint32_t taddr, float* x) {
  uint32_t a[16], b[16];
  __syncwarp();
  TMEM_LD16(a, 0);
  TMEM_LD16(b, 16);
  TMEM_HOLD16("tcgen05.wait::ld.sync.aligned;", a);
  TMEM_HOLD16("", b);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    x[j] = __uint_as_float(a[j]);
    x[16 + j] = __uint_as_float(b[j]);
  }
}
// cap tanh(x / cap). For |u| up to 1 the continued fraction u / (1 + u^2 / (3 + u^2 / (5 + ...)))
// (Lambert) cut behind the 9 gives u (945 + 105 u^2 + u^4) / (945 + 420 u^2 + 15 u^4), off by less than
// 4 units of 2^-24; beyond it the exponential's form is exact enough. With tanhf and a division 333 rows of
// 2,048 values took 957 us where this takes 210 (a division of 0 has a way of its own, which the rows that
// are not there took).
__device__ __forceinline__ float capped_small(float x, float cap, float by) {
  const float u = x * by, z = u * u;
  return cap * __fdividef(u * fmaf(z, z + 105.f, 945.f), fmaf(z, fmaf(z, 15.f, 420.f), 945.f));
}
__device__ __forceinline__ void shape32(float* x, float scale, float cap) {
  if (scale != 1.f) {
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] *= scale;
  }
  if (cap > 0.f) {
    const float by = 1.f / cap;
    bool small = true;
#pragma unroll
    for (int j = 0; j < 32; ++j) small = small && fabsf(x[j]) <= cap;
    if (__all_sync(0xffffffffu, small)) {
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] = capped_small(x[j], cap, by);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        x[j] = fabsf(x[j]) > cap ? cap * tanh_of_2xlog2e(x[j] * by * 2.8853900817779268f)
                                 : capped_small(x[j], cap, by);
    }
  }
}
// The greatest of each eight
__device__ __forceinline__ void max_eights(const float* x, float* m) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    m[g] = x[8 * g];
#pragma unroll
    for (int j = 1; j < 8; ++j) m[g] = fmaxf(m[g], x[8 * g + j]);
  }
}

// Rows that are copied for a tile of `rows`: by pairs all, those beyond the last one as zeros; by a CTA by itself
// no more than are there, where the copies' zeros take longer than the weights (1,024 values a row: 4 rows
// 82 us in a box of 128 rows, 61 in one of 8), and the stages lie that close together: up to 12 of them instead of
// 6 (24 rows of 4,096 values 203 -> 188 us). Behind its rows a tile holds whatever is there; nobody reads the
// products. Pairs multiply for longer than they copy, and zeros are what keeps the tensor cores coolest.
template <bool PAIR> __host__ __device__ __forceinline__ int box_rows(int rows) {
  return PAIR ? 128 : (rows + 7) & ~7;
}

template <int N, bool PAIR>
__global__ void __launch_bounds__(HS_THREADS, 1)
head_scores_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ HeadPlan plan, int rows, int limit, int K, float scale, float cap,
                   const int* __restrict__ tokens, int top, float* __restrict__ given, Mass* __restrict__ mass,
                   TopKey* __restrict__ keys, uint32_t* notes, int* __restrict__ error) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t bars = base + HS_RING;
  const uint32_t full0 = bars, empty0 = bars + 8 * HS_STAGES;
  const uint32_t acc_full0 = bars + 16 * HS_STAGES, acc_empty0 = acc_full0 + 16;
  const uint32_t slot = acc_empty0 + 16;
  const uint32_t staged = bars + 256;
  volatile uint32_t* slot_ptr = (volatile uint32_t*)(smem_raw + (slot - raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const int nkb = (K + HS_BK - 1) / HS_BK;
  const int row_bytes = box_rows<PAIR>(rows) * HS_BK * 2, id_bytes = (PAIR ? 128 : plan.box) * HS_BK * 2;
  const int stages = PAIR ? HS_RING / (2 * HS_HALF) : plan.stages;
  const uint32_t sA = base, sB = base + stages * row_bytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full0 + 8 * b, 1);
      mbar_init(acc_empty0 + 8 * b, PAIR ? 8 : 4);      // the epilogue warps (of both CTAs)
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    if (PAIR) tmem_alloc_pair(slot, 512); else tmem_alloc(slot, 512);
  }
  __syncwarp();      // the cluster's barrier takes whole warps too
  tc_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *slot_ptr;
  mb_grid_wait();
  mb_grid_launch_next();
  HeadWalk walk(plan, PAIR ? blockIdx.x >> 1 : blockIdx.x, limit);
  if (warp == 0) {
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      while (walk.next_strip()) {
        const int m0 = walk.row0() + (int)rank * 128;
        for (; walk.n < walk.end; walk.step()) {
          // each CTA of a pair holds half of the tile's ids (whole boxes are copied)
          const int n0 = walk.n + (int)rank * (((walk.cols() + 15) & ~15) >> 1);
          for (int i = 0; i < nkb; ++i) {
            mbar_wait(empty0 + 8 * s, ph ^ 1, error, 61);
            if (PAIR) {
              if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * (row_bytes + id_bytes));
              const uint32_t full_lead = cluster_addr_of(full0 + 8 * s, 0);
              tma_load_2d_pair(sA + s * row_bytes, &tmA, i * HS_BK, m0, full_lead);
              tma_load_2d_pair(sB + s * id_bytes, &tmB, i * HS_BK, n0, full_lead);
            } else {
              mbar_expect_tx(full0 + 8 * s, row_bytes + id_bytes);
              tma_load_2d(sA + s * row_bytes, &tmA, i * HS_BK, m0, full0 + 8 * s);
              tma_load_2d(sB + s * id_bytes, &tmB, i * HS_BK, n0, full0 + 8 * s);
            }
            if (++s == stages) { s = 0; ph ^= 1; }
          }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      int s = 0, it = 0;
      uint32_t ph = 0;
      while (walk.next_strip()) {
        for (; walk.n < walk.end; walk.step(), ++it) {
          const uint32_t idesc = umma_idesc_bf16(block_rows_of(PAIR), (walk.cols() + 15) & ~15);
          const int b = it & 1;
          mbar_wait(acc_empty0 + 8 * b, ((it >> 1) & 1) ^ 1, error, 62);
          tc_fence_after_sync();
          for (int i = 0; i < nkb; ++i) {
            mbar_wait(full0 + 8 * s, ph, error, 63);
            tc_fence_after_sync();
            const uint64_t da = umma_desc_k128(sA + s * row_bytes);
            const uint64_t db = umma_desc_k128(sB + s * id_bytes);
#pragma unroll
            for (int k = 0; k < HS_BK / 16; ++k) {
              if (PAIR) umma_bf16_pair(tmem + b * 256, da + 2 * k, db + 2 * k, idesc, (i | k) != 0);
              else umma_bf16(tmem + b * 256, da + 2 * k, db + 2 * k, idesc, (i | k) != 0);
            }
            if (PAIR) umma_commit_pair(empty0 + 8 * s, 3); else umma_commit(empty0 + 8 * s);
            if (++s == stages) { s = 0; ph ^= 1; }
          }
          if (PAIR) umma_commit_pair(acc_full0 + 8 * b, 3); else umma_commit(acc_full0 + 8 * b);
        }
      }
    }
  } else {
    const int q = warp & 3;
    const int lane_row = q * 32 + lane;
    const uint32_t mine = staged + (uint32_t)q * 4096 + lane * 4;
    const bool shaped = scale != 1.f || cap > 0.f;
    int it = 0;
    while (walk.next_strip()) {
      const int in_block = (int)rank * 128 + lane_row, row = walk.row0() + in_block;
      const int token = row < rows ? tokens[row] : -1;
      // The row's mass, S - 1 in place of S from the first value on: beside the likeliest token's 1 a tile of
      // less than 2^-24 would be lost, and of a nearly certain token all others are such tiles.
      float m = -INFINITY, s = 0.f, t = 0.f;
      TopList<N> list;
      list.clear(top);
      int seen = 0;                              // tiles of the strip
      float groups[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};      // the greatest of every fourth eight
      uint32_t* noted = nullptr;
      if (PAIR && notes != nullptr) noted = notes + (size_t)(row >> 8) * (256 * notes_of(N)) + (row & 255);
      auto note = [&]() {
        if (noted == nullptr || row >= rows) return;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          asm volatile("red.relaxed.gpu.global.max.u32 [%0], %1;"
                       ::"l"(noted + (walk.strip * 4 + g) % notes_of(N) * 256), "r"(key_place(groups[g]))
                       : "memory");
      };
      if (row >= rows) list.hush();
      const bool idle = walk.row0() + (int)rank * 128 + q * 32 >= rows;    // none of the warp's rows is there
      for (; walk.n < walk.end; walk.step(), ++it) {
        const int b = it & 1, cols = walk.cols();
        // looked at after 1, 2, 4, ... tiles, while the next one is multiplied
        if (PAIR && N > 0 && !idle && seen != 0 && noted != nullptr && (seen & (seen - 1)) == 0) {
          if (row < rows) list.look(noted, top);
          __syncwarp();
        }
        mbar_wait(acc_full0 + 8 * b, (it >> 1) & 1, error, 64);
        tc_fence_after_sync();
        float tile_s = 0.f, tile_t = 0.f;        // the tile's part, over the same maximum
        const uint32_t taddr = tmem + b * 256 + ((uint32_t)(q * 32) << 16);
        if (N > 0 && !idle && seen == 0) {
          // A strip's first tile is read ahead for a bar: the `top`-th of its eights' greatest values, or of its
          // fours' where the eights are few (8 rows of 512 values, 20 alternatives of 32,000 ids: 35 us, 31 so).
          // Without it the first values of all rows pass, one after another.
#pragma unroll 1
          for (int c = 0; c < cols; c += 32) {
            float x[32];
            load32(taddr + c, x);
            if (shaped) shape32(x, scale, cap);
#pragma unroll
            for (int g = 0; g < 8; g += 2) {
              float four[2];
#pragma unroll
              for (int e = 0; e < 2; ++e)
                four[e] = fmaxf(fmaxf(x[4 * (g + e)], x[4 * (g + e) + 1]),
                                fmaxf(x[4 * (g + e) + 2], x[4 * (g + e) + 3]));
              if (c + 4 * g + 8 > cols) continue;
              groups[g >> 1] = fmaxf(groups[g >> 1], fmaxf(four[0], four[1]));
              if (N <= 8 || cols >= 16 * top) {
                list.probe(fmaxf(four[0], four[1]));
              } else {
                list.probe(four[0]);
                list.probe(four[1]);
              }
            }
          }
          list.start(top);
          if (row >= rows) list.hush();
          if (PAIR) note();
        }
#pragma unroll 1
        for (int c = 0; c < (idle ? 0 : cols); c += 32) {
          float x[32];
          load32(taddr + c, x);
          const int n = min(32, cols - c), id0 = walk.n + c;
          if (shaped) shape32(x, scale, cap);
          if (n < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j >= n) x[j] = -INFINITY;
          }
          float eights[4];
          max_eights(x, eights);
          const float most = fmaxf(fmaxf(eights[0], eights[1]), fmaxf(eights[2], eights[3]));
          if (PAIR && N > 0 && noted != nullptr) {
#pragma unroll
            for (int g = 0; g < 4; ++g) groups[g] = fmaxf(groups[g], eights[g]);
          }
          const bool moved = most > m;
          if (moved) {
            const Mass row_part = mass_over({m, s + 1.f, t}, most), tile_part = mass_over({m, tile_s, tile_t}, most);
            m = most;
            s = row_part.s, t = row_part.t;
            tile_s = tile_part.s, tile_t = tile_part.t;
          }
          const float at = m == -INFINITY ? 0.f : m;
          float piece = 0.f;                     // where the maximum is new, its 1 is in here
          mass_add<32>(x, at, piece, tile_t);
          tile_s += moved ? piece - 1.f : piece;
          const unsigned off = (unsigned)token - (unsigned)id0;
          if (__any_sync(0xffffffffu, off < (unsigned)n)) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (off == (unsigned)j && j < n) given[row] = x[j];
          }
          if (N > 0 && __any_sync(0xffffffffu, most > list.bar)) {
            // Which values pass is a bit each; a lane takes its own one after another. They are read
            // again from shared memory, where a register could not be named by a number.
            unsigned pass = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + j * 128), "f"(x[j]) : "memory");
              if (x[j] > list.bar) pass |= 1u << j;
            }
            while (pass) {
              const int j = __ffs(pass) - 1;
              pass &= pass - 1;
              float y;
              asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(mine + j * 128) : "memory");
              list.offer(y, id0 + j);
            }
            __syncwarp();
          }
        }
        s += tile_s;
        t += tile_t;
        ++seen;
        if (PAIR && N > 0 && !idle && (seen & (seen - 1)) == 0) note();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (rank == 0) mbar_arrive(acc_empty0 + 8 * b);
          else mbar_arrive_cluster(cluster_addr_of(acc_empty0 + 8 * b, 0));
        }
      }
      if (row < rows) {
        const int strips = plan.strips[walk.band];
        const size_t part =
            plan.part0[walk.band] + ((size_t)walk.block * block_rows_of(PAIR) + in_block) * strips + walk.strip;
        mass[part] = {m, m == -INFINITY ? s - 1.f : s, t};      // as rest_join takes it (no value: no 1 either)
        list.write(keys + part * top, top);
      }
    }
  }
  // neither CTA of a pair leaves while the other may still read its shared memory or signal its barriers
  __syncwarp();
  tc_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();
  if (warp == 1) {
    if (PAIR) tmem_dealloc_pair(tmem, 512); else tmem_dealloc(tmem, 512);
  }
}

// A warp a row joins its strips: their masses, and `top` times the greatest of the heads of their keys,
// which are in order. A lane has the strips lane, lane + 32 and so on.
__global__ void __launch_bounds__(32)
head_join_kernel(const __grid_constant__ HeadPlan plan, const Mass* __restrict__ mass,
                 const TopKey* __restrict__ keys, int top, const float* __restrict__ given, int limit,
                 const int* __restrict__ tokens, ScoreOut out) {
  mb_grid_wait();
  mb_grid_launch_next();
  extern __shared__ TopKey sh_keys[];
  const int row = blockIdx.x, lane = threadIdx.x;
  const int token = tokens[row];
  const float logit = token >= 0 && token < limit ? given[row] : __uint_as_float(0x7fc00000u);
  int band = 0, block = row / plan.block_rows;
  while (band + 1 < plan.bands && block >= plan.first[band + 1]) ++band;
  block -= plan.first[band];
  const int strips = plan.strips[band];
  const size_t part = plan.part0[band] + ((size_t)block * plan.block_rows + row % plan.block_rows) * strips;
  for (int i = lane; i < strips * top; i += 32)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(sh_keys + i)), "l"(keys + part * top + i)
                 : "memory");
  Mass v[HS_STRIPS / 32];
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < HS_STRIPS / 32; ++i) {
    v[i] = lane + 32 * i < strips ? mass[part + lane + 32 * i] : rest_none();
    most = fmaxf(most, v[i].m);
  }
  most = warp_max(most);
  Mass all = {most, 0.f, 0.f};
  int tops = -1;
#pragma unroll
  for (int i = 0; i < HS_STRIPS / 32; ++i) {
    const bool top_one = v[i].m == most;
    const Mass p = top_one ? v[i] : mass_over({v[i].m, v[i].s + 1.f, v[i].t}, most);
    all.s += p.s, all.t += p.t;
    tops += __popc(__ballot_sync(0xffffffffu, top_one));
  }
  all.s = warp_sum(all.s) + (float)tops;
  all.t = warp_sum(all.t);
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
  TopKey mine = 0;
  if (top > 0) {
    int head[HS_STRIPS / 32];
    TopKey next[HS_STRIPS / 32], first = 0;      // of the lane's strips, and the greatest of those
#pragma unroll
    for (int i = 0; i < HS_STRIPS / 32; ++i) {
      head[i] = (lane + 32 * i) * top;
      next[i] = lane + 32 * i < strips ? sh_keys[head[i]] : 0;
      if (next[i] > first) first = next[i];
    }
    for (int j = 0; j < top; ++j) {
      const uint32_t place = (uint32_t)(first >> 32), best = __reduce_max_sync(0xffffffffu, place);
      const uint32_t id = __reduce_max_sync(0xffffffffu, place == best ? (uint32_t)first : 0u);
      if (id == 0) break;
      const TopKey key = (TopKey)best << 32 | id;
      if (lane == j) mine = key;
      if (first == key) {
        first = 0;
#pragma unroll
        for (int i = 0; i < HS_STRIPS / 32; ++i) {
          if (32 * i >= strips) break;
          if (next[i] == key) {
            ++head[i];
            next[i] = head[i] < (lane + 32 * i + 1) * top ? sh_keys[head[i]] : 0;
          }
          if (next[i] > first) first = next[i];
        }
      }
      __syncwarp();
    }
  }
  finish_row(all, logit, mine, top, row, out);
}

typedef void (*HeadKernel)(CUtensorMap, CUtensorMap, HeadPlan, int, int, int, float, float, const int*, int, float*,
                           Mass*, TopKey*, uint32_t*, int*);
// The kernel whose lists have room for `top` keys
#define HS_FORMS 9
static int head_form(int top) { return (top + 3) / 4; }
#define HS_ALL(PAIR_)                                                                                    \
  {head_scores_kernel<0, PAIR_>,  head_scores_kernel<4, PAIR_>,  head_scores_kernel<8, PAIR_>,           \
   head_scores_kernel<12, PAIR_>, head_scores_kernel<16, PAIR_>, head_scores_kernel<20, PAIR_>,          \
   head_scores_kernel<24, PAIR_>, head_scores_kernel<28, PAIR_>, head_scores_kernel<32, PAIR_>}
static HeadKernel head_kernel(bool pair, int form) {
  static const HeadKernel kernels[2][HS_FORMS] = {HS_ALL(false), HS_ALL(true)};
  return kernels[pair][form];
}
static cudaError_t allow_smem(bool pair, int form) {
  static unsigned long long done[2][HS_FORMS] = {};
  return mb_allow_smem((const void*)head_kernel(pair, form), HS_SMEM, &done[pair][form]);
}

// How many CTA pairs the device runs at once (0: the kernel cannot run here)
static int head_pairs(int sms) {
  static int pairs = -1;
  if (pairs >= 0) return pairs;
  if (allow_smem(true, HS_FORMS - 1) != cudaSuccess) {
    cudaGetLastError();
    return pairs = 0;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * sms);
  cfg.blockDim = dim3(HS_THREADS);
  cfg.dynamicSmemBytes = HS_SMEM;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, head_kernel(true, HS_FORMS - 1), &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  n = n > sms / 2 ? sms / 2 : n;
  return pairs = n > HS_STRIPS ? HS_STRIPS : n;
}

// Pairs, or CTAs by themselves for rows that one of them holds: half of a pair's tile would be empty, and
// its products take as long as the weights' way from memory. 5 and 20 alternatives, us in pairs and by themselves:
// 128 rows of 512 values 71 105 | 50 85, of 1,024 75 110 | 69 95, of 2,048 120 147 | 124 144, of 4,096
// 231 245 | 234 246.
static bool in_pairs(int rows) { return rows > block_rows_of(false); }
static int head_units(bool pair, int sms) {
  const int pairs = head_pairs(sms);
  return pair || pairs == 0 ? pairs : sms < HS_STRIPS ? sms : HS_STRIPS;
}

// Ids of a strip where `blocks` row blocks share the pairs (or CTAs), a multiple of 16
static int strip_width(int blocks, int units, int limit) {
  const int strips = units / blocks;
  return ((limit + strips - 1) / strips + 15) & ~15;
}

// Ids of a tile of a CTA by itself, a multiple of 16. All of a tile is copied, so it should not reach beyond the
// strip: 24 rows of 4,096 values, strips of 1,040 ids, in tiles of 128 (1,152 copied) 208 us, of 96 (1,056) 188. A
// tile itself costs as much as some 32,768 values of the head: of 512 values a row 31 and 36 us.
static int tile_of(int width, int K) {
  const int most = block_rows_of(false);
  int best = most;
  long long cost = 0;
  for (int t = most; t >= 64; t -= 16) {
    const long long c = (width + t - 1) / t * ((long long)t * K + 32768);
    if (t == most || c < cost) best = t, cost = c;
  }
  return best;
}

// Cuts a launch's row blocks into bands of at most `units` blocks such that the strips' widths add up
// to the least: the time of a band is that of its widest strip, and a strip's start and end (its first tile
// has nothing to overlap, its last one's values neither), which count as 512 ids. With 64 the 2,048 rows
// above took four bands of two blocks, which fill the pairs exactly and read the weights four times: 2,090 us
// where one band of eight takes 1,885, with 1,024 values 623 and 475.
static void plan_bands(HeadPlan& plan, int rows, int units, int limit, int K) {
  plan.block_rows = block_rows_of(in_pairs(rows));
  const int blocks = (rows + plan.block_rows - 1) / plan.block_rows;
  int best[HS_BLOCKS + 1], take[HS_BLOCKS + 1];
  best[0] = 0;
  for (int n = 1; n <= blocks; ++n) {
    best[n] = 0x7fffffff;
    for (int b = 1; b <= n && b <= units; ++b) {
      const int cost = best[n - b] + strip_width(b, units, limit) + 512;
      if (cost < best[n]) best[n] = cost, take[n] = b;
    }
  }
  plan.bands = 0;
  int first = 0, part = 0;
  for (int n = blocks; n > 0; n -= take[n]) {
    const int i = plan.bands++, b = take[n], width = strip_width(b, units, limit);
    plan.first[i] = first;
    plan.blocks[i] = b;
    plan.width[i] = width;
    plan.strips[i] = (limit + width - 1) / width;
    const int tiles = (width + plan.block_rows - 1) / plan.block_rows;
    plan.tile[i] = ((width + tiles - 1) / tiles + 15) & ~15;
    plan.part0[i] = part;
    first += b;
    part += b * plan.block_rows * plan.strips[i];
  }
  plan.box = 128;
  if (!in_pairs(rows)) {      // one band, for a launch of so few rows is one block
    plan.box = plan.tile[0] = tile_of(plan.width[0], K);
    const int fit = HS_RING / ((box_rows<false>(rows) + plan.box) * HS_BK * 2);
    plan.stages = fit < HS_STAGES ? fit : HS_STAGES;
  }
}
// Whether a row's strips are wide enough that what they note pays for a memset ahead of the kernel. 5 and 20
// alternatives, us without and with notes: 200 rows of 512 values, 151,936 ids (strips of 2,054) 69 107 | 63 104,
// 1,001 rows (8,450) 184 254 | 172 234, 400 rows and 65,536 ids (1,772) 58 93 | 53 90; of 1,024 values the first
// 77 113 | 75 109, the last 63 100 | 60 96. CTAs by themselves have narrower ones (8 rows of 1,024 values, 151,936
// ids 57 77 | 58 89).
static bool notes_pay(const HeadPlan& plan, bool pair, int top) {
  int width = 0;
  for (int i = 0; i < plan.bands; ++i) width = plan.width[i] > width ? plan.width[i] : width;
  return pair && top > 0 && width >= 1024;
}
static long long notes_bytes(int rows, int form) { return (rows + 255ll) / 256 * 1024 * notes_of(4 * form); }
static int parts_of(const HeadPlan& plan) {
  const int i = plan.bands - 1;
  return plan.part0[i] + plan.blocks[i] * plan.block_rows * plan.strips[i];
}

// Whether mb_head_scores takes operands of these sizes and alignments on this device.
MB_EXPORT int mb_head_scores_supported(const void* A, int lda, const void* W, int K, int sms) {
  return K > 0 && K % 8 == 0 && lda >= K && lda % 8 == 0 && ((uintptr_t)A & 15) == 0 && ((uintptr_t)W & 15) == 0 &&
         head_pairs(sms) > 0;
}

// bytes of scratch that mb_head_scores needs: what the larger of its two plans takes (that of whole
// launches, and that of the last one, which may be cut into more strips)
MB_EXPORT long long mb_head_scores_scratch(int rows, int limit, int top, int sms) {
  const int most = HS_BLOCKS * block_rows_of(true);
  if (head_pairs(sms) <= 0 || rows <= 0 || limit <= 0) return 0;
  long long parts = 0;
  for (const int n : {rows < most ? 0 : most, rows % most}) {
    if (n == 0) continue;
    HeadPlan plan;
    plan_bands(plan, n, head_units(in_pairs(n), sms), limit, 0);
    if (parts_of(plan) > parts) parts = parts_of(plan);
  }
  const int one = rows < most ? rows : most;
  return parts * (12 + 8 * top) + 4ll * one + (top > 0 ? notes_bytes(one, head_form(top)) : 0) + 16;
}

// For rows A [rows, K] (bfloat16, `lda` values from row to row) and a head W [V, K]: the scores of
// tokens[r] under the logits x = scale A W^T, or cap tanh(x / cap) where cap > 0, of the ids below
// `limit` <= V. Outputs as mb_token_scores. scratch: mb_head_scores_scratch bytes, 16-byte aligned.
MB_EXPORT int mb_head_scores(const void* A, int lda, const void* W, int rows, int limit, int K,
                             float scale, float cap, const int* tokens, int top, float* logprobs,
                             float* entropy, int* top_ids, float* top_logprobs, void* scratch,
                             long long scratch_bytes, int* error, int sms, void* stream) {
  if (rows <= 0) return 0;
  if (limit <= 0 || top < 0 || top > MB_SCORES_TOP || top > limit)
    MB_FAIL("mb_head_scores: %d alternatives of a vocabulary of %d", top, limit);
  if (!mb_head_scores_supported(A, lda, W, K, sms))
    MB_FAIL("mb_head_scores: rows of %d values, %d apart, are not taken", K, lda);
  if (scratch_bytes < mb_head_scores_scratch(rows, limit, top, sms))
    MB_FAIL("mb_head_scores: %lld bytes of scratch", scratch_bytes);
  const int form = head_form(top), most = HS_BLOCKS * block_rows_of(true);
  cudaStream_t s = (cudaStream_t)stream;
  for (int r0 = 0; r0 < rows; r0 += most) {
    const int n = rows - r0 < most ? rows - r0 : most;
    const bool pair = in_pairs(n);
    if (cudaError_t e = allow_smem(pair, form)) MB_FAIL("mb_head_scores: %s", cudaGetErrorString(e));
    const __nv_bfloat16* a = (const __nv_bfloat16*)A + (size_t)r0 * lda;
    HeadPlan plan = {};
    plan_bands(plan, n, head_units(pair, sms), limit, K);
    CUtensorMap tmA, tmB;
    if (!mb_make_map_bf16(&tmB, W, limit, K, K, plan.box, "mb_head_scores weight")) return -1;
    const int box = pair ? box_rows<true>(n) : box_rows<false>(n);
    if (!mb_make_map_bf16(&tmA, a, n, K, lda, box, "mb_head_scores input")) return -1;
    const size_t parts = parts_of(plan);
    TopKey* keys = (TopKey*)scratch;
    Mass* mass = (Mass*)(keys + parts * top);
    float* given = (float*)(mass + parts);
    uint32_t* notes = notes_pay(plan, pair, top) ? (uint32_t*)(given + n) : nullptr;
    if (notes != nullptr)
      if (cudaError_t e = cudaMemsetAsync(notes, 0, notes_bytes(n, form), s))
        MB_FAIL("mb_head_scores: %s", cudaGetErrorString(e));
    int used = 0;
    for (int i = 0; i < plan.bands; ++i)
      if (plan.blocks[i] * plan.strips[i] > used) used = plan.blocks[i] * plan.strips[i];
    const dim3 block(HS_THREADS);
    cudaError_t e =
        pair ? mb_launch_clusters(head_kernel(true, form), dim3(2 * used), block, HS_SMEM, s, 2, tmA, tmB,
                                  plan, n, limit, K, scale, cap, tokens + r0, top, given, mass, keys,
                                  notes, error)
             : mb_launch(head_kernel(false, form), dim3(used), block, HS_SMEM, s, tmA, tmB, plan, n, limit,
                         K, scale, cap, tokens + r0, top, given, mass, keys, notes, error);
    if (e != cudaSuccess) MB_FAIL("mb_head_scores: %s", cudaGetErrorString(e));
    const ScoreOut out = {logprobs + r0, entropy + r0, top_ids + (size_t)r0 * top,
                          top_logprobs + (size_t)r0 * top};
    int strips = 0;
    for (int i = 0; i < plan.bands; ++i) strips = plan.strips[i] > strips ? plan.strips[i] : strips;
    mb_launch(head_join_kernel, dim3(n), dim3(32), (size_t)strips * top * 8, s, plan, mass, keys, top, given, limit,
              tokens + r0, out);
  }
  MB_CHECK_LAUNCH("mb_head_scores");
}
