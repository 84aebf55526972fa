// Cross entropy of a large vocabulary straight from the hidden states, and its
// gradient, without the logits of all tokens ever being stored.
//
//   l_nv = x_n . w_v,  lse_n = log sum_v exp(l_nv),  loss_n = lse_n - l_n,t(n),
//   g_nv = (exp(l_nv - lse_n) - [v = t(n)]) dloss_n,
//   dx_n = sum_v g_nv w_v,  dw_v = sum_n g_nv x_n.
//
// Forward: one matrix product whose epilogue leaves each tile's row maximum
// and sum of exponentials; a second kernel joins them.  Backward: the
// vocabulary goes by in pieces; a piece's logits are computed again, turned
// into g in the product's epilogue and rounded once to the inputs' type, and
// two more products take g to dx (summed in fp32 over the pieces) and dw.  The
// largest entry of a row of g is nearly always the target's, so its rounding is
// nearly all of g's: what it took off is kept in fp32 and added to both
// gradients at the end (error of the gradients' 2-norm in bf16 2.5e-3 without and
// 1.7e-3 with it, as of rounding the result alone).
// Rows with the ignored target are left out of every product: the first kernel
// lists the others, and the products run over that list.
#include "clear_device.hpp"
#include "clear_host.hpp"

#include <algorithm>
#include <type_traits>

namespace clr {

// What the kernels share: the listed rows and their statistics.
struct LossDims {
  const void *hidden, *weight;
  const int64_t *targets;
  float *loss, *lse;
  const float *dloss;
  void *dhidden, *dweight;
  int *count;       // listed rows (unless `direct`, as all of the list)
  float *unit;      // [2] power of two that g carries, and its inverse
  int *row;         // [N] token of listed row
  int *place;       // [N] listed row of a token, -1 where ignored
  int *target;      // [N] of a listed row, -1 where it is no class
  float *hit;       // [N] logit at the target
  float2 *part;     // forward: [tiles][N] (maximum, sum of exp(logit - maximum))
  float *lse2, *dl; // backward: [N]
  float *rest;      // backward: [N] what rounding took off g at the target
  int2 *hits;       // backward: [N] (listed row, class) by the class's tile, in order
  int *hit_start;   // backward: [tiles + 1]
  void *x;          // the listed rows of hidden, [N][width]
  void *g;          // backward: [N][pitch] of one piece
  float *dx;        // backward: [splits][N][width]
  int64_t h_stride, w_stride, ignore;
  int tokens, vocab, width, pitch;
  int v0, v1;       // the piece
  int splits, accumulate;
  int direct;       // no list, rows are tokens
};

// A row's target where no list holds it.
struct Target {
  bool counts;  // not ignored
  int at;       // its class, -1 where it is none
};
__device__ __forceinline__ Target target_of(const LossDims &p, int token) {
  const int64_t t = p.targets[token];
  return {t != p.ignore, t >= 0 && t < p.vocab ? (int)t : -1};
}
__device__ __forceinline__ int rows_of(const LossDims &p) { return p.direct ? p.tokens : *p.count; }

// fp16 carries g times a power of two that takes the largest factor to [2^13,
// 2^14), so that small probabilities stay far from the smallest numbers.
template <class T> __device__ __forceinline__ int unit_log(float top) {
  if (!__is_same(T, _Float16) || !(top > 0.0f)) return 0;
  return 14 - min(max(ilogbf(fminf(top, 1e30f)) + 1, -100), 100);
}

constexpr int GEMM_K = 64;

// One operand of a product: R rows (M or N) at a time, K in steps of 64.
// Where K is contiguous an LDS tile is [R][64] and a lane reads its eight
// values at once; where the rows are contiguous ([K][R] in memory) the tile is
// [64][R] and transposing reads collect them.
template <class T, int R, bool COLUMNS, int THREADS> struct Operand {
  static constexpr int ELEMENTS = R * GEMM_K;
  static constexpr int EACH = ELEMENTS / 8 / THREADS;
  static constexpr int CHUNKS = COLUMNS ? R / 8 : GEMM_K / 8;
  uint32_t at[EACH];  // byte offset of each of the thread's chunks in a step
  const char *base;   // of the next step
  int row_bytes;      // COLUMNS: a row of memory, otherwise a step
  int left;           // k that are left

  static __device__ __forceinline__ int swz(int r) {
    // rows of 128 bytes read 16 at a time, or of 256 and more transposed
    return COLUMNS ? (r & 3) << 2 : (r >> 1) & 7;
  }
  static __device__ __forceinline__ int row_of(int i, int tid) { return (i * THREADS + tid) / CHUNKS; }
  static __device__ __forceinline__ int chunk_of(int i, int tid) {
    return ((i * THREADS + tid) % CHUNKS) ^ swz(row_of(i, tid));
  }

  // The tile's rows start at row0 and end below `rows`; k0 <= k < k1.  A tile's
  // step stays within 2 GB (256 rows of at most 2^20 values, which the host
  // checks), so 32-bit offsets from its base do.
  __device__ __forceinline__ void open(const T *x, int64_t stride, int row0, int rows, int k0,
                                       int k1, int tid) {
    left = k1 - k0;
    row_bytes = (int)((COLUMNS ? stride : GEMM_K) * (int64_t)sizeof(T));
    base = (const char *)(x + (COLUMNS ? k0 * stride + row0 : row0 * stride + k0));
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int r = row_of(i, tid), c = chunk_of(i, tid);
      const bool in = COLUMNS ? row0 + c * 8 < rows : row0 + r < rows;
      at[i] = in ? (uint32_t)((r * stride + c * 8) * (int64_t)sizeof(T)) : NOWHERE;
    }
  }

  // Copies the next step's tile (zeros from the last k on) and moves on.
  __device__ __forceinline__ void load(T *lds, int tid) {
    if (COLUMNS) {
      const auto buffer = buffer_of(base, (uint32_t)(min(max(left, 0), GEMM_K) * row_bytes));
#pragma unroll
      for (int i = 0; i < EACH; i++)
        copy_to_lds(buffer, at[i], lds + (i * THREADS + uniform(tid & ~63)) * 8);
    } else {
      const auto buffer = buffer_of(base, ANYWHERE);
      // the threads are a multiple of 16 rows apart: one chunk index for all
      static_assert(COLUMNS || THREADS / CHUNKS % 16 == 0, "the swizzle's period");
      const bool in = chunk_of(0, tid) * 8 < left;
#pragma unroll
      for (int i = 0; i < EACH; i++)
        copy_to_lds(buffer, in ? at[i] : NOWHERE, lds + (i * THREADS + uniform(tid & ~63)) * 8);
    }
    base += (int64_t)row_bytes * (COLUMNS ? GEMM_K : 1);
    left -= GEMM_K;
  }

  // Rows r0 + lane % 32, k = 16 s + 8 (lane / 32) + 0..7.
  static __device__ __forceinline__ typename Half<T>::x8 read(const T *lds, int r0, int s, int lane) {
    if (COLUMNS) {
      const int kr = 16 * s + 8 * (lane >> 5) + ((lane & 15) >> 2);
      const int col = r0 + (lane & 16) + (lane & 3) * 4;
      const int c = col >> 3;
      const T *a = lds + kr * R + ((c ^ swz(kr)) * 8) + (col & 7);
      const T *b = lds + (kr + 4) * R + ((c ^ swz(kr + 4)) * 8) + (col & 7);
      return join<T>(read_transposed(a), read_transposed(b));
    } else {
      const int r = r0 + (lane & 31);
      return *(const typename Half<T>::x8 *)(lds + r * GEMM_K + (((2 * s + (lane >> 5)) ^ swz(r)) * 8));
    }
  }
};

// A block's tile of a product: BM x BN over WM x WN waves.
template <class T, int BM, int BN, int WM, int WN, bool CM, bool CN> struct Product {
  static constexpr int THREADS = 64 * WM * WN;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  static constexpr int M = BM, N = BN, WAVES_M = WM, WAVES_N = WN;
  using A = Operand<T, BM, CM, THREADS>;
  using B = Operand<T, BN, CN, THREADS>;

  // A wave's share of the buffers, for its results.
  static __device__ __forceinline__ T *slab(int wave, T *a0, T *b0, T *a1, T *b1) {
    constexpr int OWN = (BM / WM) * (BN / WN);
    constexpr int IN_A = A::ELEMENTS / OWN, IN_B = B::ELEMENTS / OWN;
    static_assert(2 * (IN_A + IN_B) >= WM * WN, "the results fit the buffers");
    if (wave < IN_B) return b0 + wave * OWN;
    wave -= IN_B;
    if (wave < IN_B) return b1 + wave * OWN;
    wave -= IN_B;
    return wave < IN_A ? a0 + wave * OWN : a1 + (wave - IN_A) * OWN;
  }
  struct alignas(8) Four { T v[4]; };
  static __device__ __forceinline__ Four four(const f32x16 &x, int q, float f) {
    Four y;
#pragma unroll
    for (int e = 0; e < 4; e++) y.v[e] = (T)(x[4 * q + e] * f);
    return y;
  }

  // `start` may set the sums' beginnings while the first tiles are under way.
  template <class F>
  static __device__ __forceinline__ void run(A &a, B &b, int steps, T *a0, T *b0, T *a1, T *b1,
                                             f32x16 (&acc)[TM][TN], F &&start) {
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int m0 = wave / WN * (BM / WM), n0 = wave % WN * (BN / WN);
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
    // Two sets of operand registers: 16 k are read while the 16 before them
    // multiply.  The fences keep the reads of all four from being drawn
    // together, which the registers cannot hold.
    typename Half<T>::x8 af[2][TM], bf[2][TN];
    auto read = [&](const T *at, const T *bt, int s) {
#pragma unroll
      for (int i = 0; i < TM; i++) af[s & 1][i] = A::read(at, m0 + 32 * i, s, lane);
#pragma unroll
      for (int j = 0; j < TN; j++) bf[s & 1][j] = B::read(bt, n0 + 32 * j, s, lane);
    };
    auto multiply = [&](int s) {
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
          acc[i][j] = Half<T>::mma(af[s & 1][i], bf[s & 1][j], acc[i][j]);
    };
    constexpr int LAST = GEMM_K / 16 - 1;
    static_assert(LAST % 2 == 1, "the next step's first operands go where the last ones are not");
    constexpr int READS = CM + CN + 2 > 2 ? 2 : 1;
    // The buffers change hands before a step's last products: those still
    // multiply while the next step's first operands are on their way.
    auto step = [&](T *at, T *bt, const T *an, const T *bn) {
#pragma unroll
      for (int s = 0; s < LAST; s++) {
        __builtin_amdgcn_sched_barrier(0);
        read(at, bt, s + 1);
        multiply(s);
        interleave<TM + TN, READS, READS>();
      }
      tile_barrier();
      __builtin_amdgcn_sched_barrier(0);
      read(an, bn, 0);
      a.load(at, tid), b.load(bt, tid);
      multiply(LAST);
      // one copy behind each product: issued together they keep the matrix
      // units waiting (logits of 4096 x 128256 x 4096: 3.07 against 2.96 ms)
      __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
      for (int i = 0; i < TM * TN; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
        __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // Loads past the end bring zeros, and an odd number of steps is made even
    // with one of zeros: the loop has one body and no branch.
    if (steps <= 0) return;
    a.load(a0, tid), b.load(b0, tid);
    start();
    tile_barrier();
    a.load(a1, tid), b.load(b1, tid);
    read(a0, b0, 0);
    for (int i = 0; i < steps; i += 2) {
      step(a0, b0, a1, b1);
      step(a1, b1, a0, b0);
    }
    wait_global<0>();  // no copy into LDS outlives its block
  }
};

// A wave's MR x 32 TN results as rows of memory: result columns are memory rows
// of MR values.  A lane holds four values of a row, which stored as they are
// would touch 64 rows an instruction, 8 bytes each; they go through the wave's
// part of LDS (the operands' buffers, free by now) into stores of whole rows.
// values(i, j, q) gives the four at rows 32 i + 8 q + 4 (lane / 32) of column
// 32 j + lane % 32; target(column, row) the address of eight, or null.
template <class T, int MR, int TN, class V, class P>
__device__ __forceinline__ void store_rows(T *slab, int lane, V &&values, P &&target) {
  struct alignas(16) Eight { T v[8]; };
  constexpr int CHUNKS = MR / 8, ROW = MR * 2;
  char *s = (char *)slab;
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int i = 0; i < MR / 32; i++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int row = 32 * j + (lane & 31), chunk = (4 * i + q) ^ (row & (CHUNKS - 1));
        *(decltype(values(i, j, q)) *)(s + row * ROW + chunk * 16 + (lane >> 5) * 8) = values(i, j, q);
      }
  __builtin_amdgcn_wave_barrier();
  wait_lds();
#pragma unroll
  for (int k = 0; k < 32 * TN * CHUNKS / 64; k++) {
    const int row = (k * 64 + lane) / CHUNKS, c = lane & (CHUNKS - 1);
    T *to = target(row, 8 * c);
    if (to) *(Eight *)to = *(const Eight *)(s + row * ROW + ((c ^ (row & (CHUNKS - 1))) * 16));
  }
}

// Tile of a block: each XCD (blocks go to the eight in turn) takes one run of
// tiles, in columns of four, so that its L2 serves four rows of tiles at a time.
__device__ __forceinline__ void tile_of(int id, int mt, int nt, int &m, int &n) {
  const int total = mt * nt;
  const int xcd = id & 7, q = total >> 3, r = total & 7;
  const int lin = xcd * q + min(xcd, r) + (id >> 3);
  const int g = lin / (4 * nt), in = lin - g * 4 * nt;
  const int gm = min(4, mt - 4 * g);
  m = 4 * g + in % gm;
  n = in / gm;
}

// Lists the rows that count, gathers their hidden states, and writes what the
// others get.  A block takes some tokens, up to 64 at a time, and counts those
// before them itself, so the list has one order and needs no second launch.
constexpr int LIST_ROWS = 64, LIST_THREADS = 256;

// The backward pass's blocks behind them take a tile of classes each, and list
// the rows whose target lies in it.
__device__ __forceinline__ void list_hits(const LossDims &p, int tile, int size, int tiles) {
  constexpr int WAVES = LIST_THREADS / 64;
  __shared__ int sums[2][WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int v0 = tile * size;
  const uint64_t below = (1ull << lane) - 1;
  int n = 0;
#pragma unroll 4
  for (int i = tid; i < p.tokens; i += LIST_THREADS) {
    const Target t = target_of(p, i);
    n += t.counts && t.at >= 0 && t.at < v0;
  }
  for (int x = 1; x < 64; x <<= 1) n += __shfl_xor(n, x, 64);
  if (lane == 0) sums[0][wave] = n;
  __syncthreads();
  int at = 0, row = 0;  // places of the next hit and of the next listed row
  for (int w = 0; w < WAVES; w++) at += sums[0][w];
  if (tid == 0) p.hit_start[tile] = at;
  for (int first = 0; first < p.tokens; first += LIST_THREADS) {
    const int i = first + tid;
    Target t = {false, -1};
    if (i < p.tokens) t = target_of(p, i);
    const bool hit = t.counts && t.at >= v0 && t.at < v0 + size;
    const uint64_t rows = __ballot(t.counts), hits = __ballot(hit);
    __syncthreads();
    if (lane == 0) sums[0][wave] = __popcll(rows), sums[1][wave] = __popcll(hits);
    __syncthreads();
    int r = row, h = at;
    for (int w = 0; w < WAVES; w++) {
      if (w < wave) r += sums[0][w], h += sums[1][w];
      row += sums[0][w], at += sums[1][w];
    }
    if (hit) p.hits[h + __popcll(hits & below)] = make_int2(r + __popcll(rows & below), t.at);
  }
  if (tile == tiles - 1 && tid == 0) p.hit_start[tiles] = at;
}

template <class T, bool BACKWARD>
__global__ __launch_bounds__(LIST_THREADS) void loss_list_kernel(LossDims p, int rows, int lists,
                                                                 int size) {
  if (BACKWARD && (int)blockIdx.x >= lists) {
    list_hits(p, blockIdx.x - lists, size, gridDim.x - lists);
    return;
  }
  __shared__ int before[LIST_THREADS / 64];
  __shared__ float tops[LIST_THREADS / 64];
  __shared__ int where[LIST_ROWS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int begin = blockIdx.x * rows, end = min(begin + rows, p.tokens);
  int n = 0;
  float top = 0.0f;
  // the last block counts everything, and finds the largest factor
  const bool last = (int)blockIdx.x == lists - 1;
#pragma unroll 4
  for (int i = tid; i < (last ? p.tokens : begin); i += LIST_THREADS) {
    const bool in = p.targets[i] != p.ignore;
    n += in && i < begin;
    if (BACKWARD && last && in) top = fmaxf(top, fabsf(p.dloss[i]));
  }
  for (int x = 1; x < 64; x <<= 1) {
    n += __shfl_xor(n, x, 64);
    top = fmaxf(top, __shfl_xor(top, x, 64));
  }
  if (lane == 0) before[tid >> 6] = n, tops[tid >> 6] = top;
  __syncthreads();
  n = 0;
  for (int w = 0; w < LIST_THREADS / 64; w++) n += before[w], top = fmaxf(top, tops[w]);
  for (int first = begin; first < end; first += LIST_ROWS) {
    const int here = min(end - first, LIST_ROWS);
    if (tid < 64) {
      const int i = first + lane;
      const bool there = lane < here;
      const int64_t t = there ? p.targets[i] : p.ignore;
      const bool in = t != p.ignore;
      const uint64_t votes = __ballot(in);
      const int at = n + __popcll(votes & ((1ull << lane) - 1));
      if (there) {
        where[lane] = in ? at : -1;
        if (BACKWARD) p.place[i] = in ? at : -1;
        const bool is_class = t >= 0 && t < p.vocab;
        if (in) {
          p.row[at] = i;
          p.target[at] = is_class ? (int)t : -1;
          if (BACKWARD) {
            p.lse2[at] = p.lse[i] * LOG2E;
            p.dl[at] = is_class ? p.dloss[i] : NAN;
          } else {
            p.hit[at] = NAN;
          }
        } else if (!BACKWARD) {
          p.loss[i] = 0.0f, p.lse[i] = 0.0f;
        }
      }
      n += __popcll(votes);
    }
    __syncthreads();
    struct alignas(16) Chunk { T v[8]; };
    const int chunks = p.width / 8;
    // consecutive chunks of consecutive rows, four under way a thread
#pragma unroll 4
    for (int i = tid; i < here * chunks; i += LIST_THREADS) {
      const int r = i / chunks, c = i - r * chunks;
      if (where[r] >= 0)
        ((Chunk *)((T *)p.x + (int64_t)where[r] * p.width))[c] =
            ((const Chunk *)((const T *)p.hidden + (int64_t)(first + r) * p.h_stride))[c];
    }
    __syncthreads();
  }
  if (last && tid == 0) {
    *p.count = n;
    if (BACKWARD) {
      const int e = unit_log<T>(top);
      p.unit[0] = ldexpf(1.0f, e), p.unit[1] = ldexpf(1.0f, -e);
    }
  }
}

// Logits of a tile, rows over the vocabulary and columns over the listed rows:
// a column's maximum and sum are taken within a lane.  GRAD: into g; otherwise
// into (maximum, sum) and the target's logit.
//
// 4096 x 128256 x 4096, a tenth ignored, bf16: 2.96 ms, 1.36 PFLOP/s over whole
// tiles, as a library product of 8192^3 (1.38).  The matrix units are busy 74%
// of the cycles and the clock falls to 1.5 GHz: bound by power.  128 tokens: the
// weights' 1.05 GB in 190 us, 5.5 TB/s.
template <class T, int BM, int BN, int WM, int WN, bool GRAD, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void loss_logits_kernel(LossDims p, int mt, int nt) {
  using P = Product<T, BM, BN, WM, WN, false, false>;
  __shared__ __attribute__((aligned(16))) T a0[P::A::ELEMENTS], b0[P::B::ELEMENTS];
  __shared__ __attribute__((aligned(16))) T a1[P::A::ELEMENTS], b1[P::B::ELEMENTS];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
  int m, n;
  tile_of(blockIdx.x, mt, nt, m, n);
  const int count = DIRECT ? p.tokens : *p.count;
  if (n * BN >= count) return;
  float unit = 1.0f;
  if (GRAD && DIRECT) {
    // every wave finds the largest factor; the hidden states that the gradient's
    // products read are shared out over the blocks, without what ignored rows hold
    float top = 0.0f;
    for (int i = lane; i < p.tokens; i += 64)
      if (target_of(p, i).counts) top = fmaxf(top, fabsf(p.dloss[i]));
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const int e = unit_log<T>(top);
    unit = ldexpf(1.0f, e);
    if (blockIdx.x == 0 && tid == 0) p.unit[0] = unit, p.unit[1] = ldexpf(1.0f, -e);
    const int chunks = p.width / 8;
    for (int i = blockIdx.x * P::THREADS + tid; i < p.tokens * chunks; i += gridDim.x * P::THREADS) {
      const int r = i / chunks, c = i - r * chunks;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (target_of(p, r).counts)
        x = ((const uint4 *)((const T *)p.hidden + (int64_t)r * p.h_stride))[c];
      ((uint4 *)p.x)[i] = x;
    }
  } else if (GRAD) {
    unit = p.unit[0];
  }
  typename P::A a;
  typename P::B b;
  a.open((const T *)p.weight, p.w_stride, p.v0 + m * BM, p.v1, 0, p.width, tid);
  b.open((const T *)(DIRECT ? p.hidden : p.x), DIRECT ? p.h_stride : p.width, n * BN, count, 0,
         p.width, tid);
  f32x16 acc[P::TM][P::TN];
  P::run(a, b, (p.width + GEMM_K - 1) / GEMM_K, a0, b0, a1, b1, acc, [] {});
  const int row0 = m * BM + wave / WN * (BM / WM) + 4 * h;  // of the piece
#pragma unroll
  for (int j = 0; j < P::TN; j++) {
    const int col = n * BN + wave % WN * (BN / WN) + 32 * j + (lane & 31);
    const bool there = col < count;
    Target t = {there, -1};
    if (there && DIRECT) t = target_of(p, col);
    else if (there) t.at = p.target[col];
    const int target = t.at >= 0 ? t.at - p.v0 : -1;
    if (GRAD) {
      float lse2 = 0.0f, dl = 0.0f;
      if (t.counts && DIRECT) lse2 = p.lse[col] * LOG2E, dl = t.at >= 0 ? p.dloss[col] : NAN;
      else if (t.counts) lse2 = p.lse2[col], dl = p.dl[col];
      dl *= unit;
      float here = 0.0f;  // g at the target
#pragma unroll
      for (int i = 0; i < P::TM; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int v = row0 + 32 * i + 8 * (e >> 2) + (e & 3);
          float y = exp2_fast(fmaf(acc[i][j][e], LOG2E, -lse2));
          y = (y - (v == target ? 1.0f : 0.0f)) * dl;
          here = v == target ? y : here;
          // beyond the vocabulary, and in ignored rows: zeros
          acc[i][j][e] = (!DIRECT || t.counts) && p.v0 + v < p.v1 ? y : 0.0f;
        }
      // the lane that holds the target's row: its place from row0 has no bit 2
      const int place = target - row0;
      if (t.counts && t.at >= 0 && place >= 0 && place < BM / WM && !(place & 4))
        p.rest[col] = here - (float)(T)here;
    } else {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < P::TM; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int v = row0 + 32 * i + 8 * (e >> 2) + (e & 3);
          if (v == target) p.hit[col] = acc[i][j][e];
          acc[i][j][e] = p.v0 + v < p.v1 ? acc[i][j][e] : -INFINITY;
          top = fmaxf(top, acc[i][j][e]);
        }
      top = halves_max(top);
      const float shift = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < P::TM; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) sum += exp2_fast((acc[i][j][e] - shift) * LOG2E);
      sum = halves_sum(sum);
      if (there && h == 0)
        p.part[(int64_t)(m * WM + wave / WN) * p.tokens + col] = make_float2(top, sum);
    }
  }
  if (GRAD) {
    tile_barrier();
    T *slab = P::slab(wave, a0, b0, a1, b1);
    T *g = (T *)p.g;
    const int c0 = n * BN + wave % WN * (BN / WN), v0 = m * BM + wave / WN * (BM / WM);
    store_rows<T, BM / WM, P::TN>(
        slab, lane,
        [&](int i, int j, int q) { return P::four(acc[i][j], q, 1.0f); },
        [&](int col, int v) {
          return c0 + col < count ? g + (int64_t)(c0 + col) * p.pitch + v0 + v : nullptr;
        });
  }
}

// Joins the tiles' statistics of a few listed rows: the tiles are shared out
// over the threads of a row, four loads under way each.
constexpr int JOIN_THREADS = 1024;

__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  // nothing so far, or NaN: the sums pass as they are
  return make_float2(m, (a.x == -INFINITY ? a.y : a.y * exp2_fast((a.x - m) * LOG2E)) +
                            (b.x == -INFINITY ? b.y : b.y * exp2_fast((b.x - m) * LOG2E)));
}

template <int JOIN_ROWS>
__global__ __launch_bounds__(JOIN_THREADS) void loss_join_kernel(LossDims p, int tiles) {
  constexpr int JOIN_PARTS = JOIN_THREADS / JOIN_ROWS;
  __shared__ float2 s[JOIN_PARTS][JOIN_ROWS];
  const int r = threadIdx.x % JOIN_ROWS, part = threadIdx.x / JOIN_ROWS;
  const int count = rows_of(p);
  const int col = blockIdx.x * JOIN_ROWS + r;
  if (blockIdx.x * JOIN_ROWS >= count) return;
  float2 x = make_float2(-INFINITY, 0.0f);
  if (col < count)
    for (int t = part; t < tiles; t += 4 * JOIN_PARTS) {
      float2 y[4];
#pragma unroll
      for (int i = 0; i < 4; i++)
        y[i] = t + i * JOIN_PARTS < tiles ? p.part[(int64_t)(t + i * JOIN_PARTS) * p.tokens + col]
                                          : make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int i = 0; i < 4; i++) x = join_stats(x, y[i]);
    }
  s[part][r] = x;
  for (int half = JOIN_PARTS / 2; half > 0; half /= 2) {
    __syncthreads();
    if (part < half) s[part][r] = x = join_stats(x, s[part + half][r]);
  }
  if (part != 0 || col >= count) return;
  // the maximum is a logit, not scaled: what is left of it behind the target's
  // logit is exact
  const float log_sum = logf(x.y), lse = x.x + log_sum;
  if (p.direct) {
    const Target t = target_of(p, col);
    p.lse[col] = t.counts ? lse : 0.0f;
    p.loss[col] = !t.counts ? 0.0f : t.at >= 0 ? (x.x - p.hit[col]) + log_sum : NAN;
    return;
  }
  const int token = p.row[col];
  p.lse[token] = lse;
  p.loss[token] = (x.x - p.hit[col]) + log_sum;
}

// dx of a tile over a share of the piece's vocabulary: rows over the width,
// columns over the listed rows.
template <class P, class T>
__device__ __forceinline__ void dx_tile(const LossDims &p, int m, int n, int split, T *a0, T *b0,
                                        T *a1, T *b1) {
  constexpr int BM = P::M, BN = P::N, WM = P::WAVES_M, WN = P::WAVES_N;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
  const int count = rows_of(p);
  if (n * BN >= count) return;
  const int all = p.v1 - p.v0;
  const int steps = (all + GEMM_K - 1) / GEMM_K, share = (steps + p.splits - 1) / p.splits;
  const int k0 = min(split * share * GEMM_K, all), k1 = min(k0 + share * GEMM_K, all);
  typename P::A a;
  typename P::B b;
  a.open((const T *)p.weight + (int64_t)p.v0 * p.w_stride, p.w_stride, m * BM, p.width, k0, k1, tid);
  // columns of g from the piece's end up to the next multiple of 8 are zeros
  b.open((const T *)p.g, p.pitch, n * BN, count, k0, k1, tid);
  f32x16 acc[P::TM][P::TN];
  P::run(a, b, (k1 - k0 + GEMM_K - 1) / GEMM_K, a0, b0, a1, b1, acc, [] {});
  const int row0 = m * BM + wave / WN * (BM / WM) + 4 * h;
#pragma unroll
  for (int j = 0; j < P::TN; j++) {
    const int col = n * BN + wave % WN * (BN / WN) + 32 * j + (lane & 31);
    if (col >= count) continue;
    float *out = p.dx + ((int64_t)split * p.tokens + col) * p.width;
#pragma unroll
    for (int i = 0; i < P::TM; i++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int d = row0 + 32 * i + 8 * q;
        if (d >= p.width) continue;
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = acc[i][j][4 * q + e];
        if (p.accumulate) x += *(const f32x4 *)(out + d);
        *(f32x4 *)(out + d) = x;
      }
  }
}

// dw of a tile: rows over the width, columns over the piece's vocabulary.
template <class P, class T>
__device__ __forceinline__ void dw_tile(const LossDims &p, int m, int n, T *a0, T *b0, T *a1, T *b1) {
  constexpr int BM = P::M, BN = P::N, WM = P::WAVES_M, WN = P::WAVES_N;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int count = rows_of(p);
  typename P::A a;
  typename P::B b;
  a.open((const T *)p.x, p.width, m * BM, p.width, 0, count, tid);
  b.open((const T *)p.g, p.pitch, n * BN, p.v1 - p.v0, 0, count, tid);
  f32x16 acc[P::TM][P::TN];
  const int v0 = p.v0 + n * BN + wave % WN * (BN / WN), d0 = m * BM + wave / WN * (BM / WM);
  P::run(a, b, (count + GEMM_K - 1) / GEMM_K, a0, b0, a1, b1, acc, [&] {
    // What rounding took off g at the targets among the wave's columns, row by
    // row in order: two lanes hold a column.
    const int tile = p.v0 / BN + n;
    const int begin = p.direct ? 0 : p.hit_start[tile];
    const int end = p.direct ? p.tokens : p.hit_start[tile + 1];
    for (int first = begin; first < end; first += 64) {
      int row = 0, col = -1;
      if (first + lane < end && !p.direct) {
        const int2 x = p.hits[first + lane];
        row = x.x, col = x.y - v0;
      } else if (first + lane < end) {
        row = first + lane;
        const Target t = target_of(p, row);
        if (t.counts && t.at >= 0) col = t.at - v0;
      }
      uint64_t hits = __ballot(col >= 0 && col < BN / WN);
      // each lane takes the first hit of each of its columns, all at once; what
      // hits a column again waits for the next turn, and so does the rest when
      // eight have (4096 x 128256 x 4096 with all tokens of one class: 23 ms
      // against 31 where the rest goes on; of many classes 10.2 ms either way)
      while (hits) {
        uint64_t later = 0;
        int waiting = 0, mine[P::TN];
#pragma unroll
        for (int j = 0; j < P::TN; j++) mine[j] = -1;
        while (hits && waiting < 8) {
          const int from = __ffsll((unsigned long long)hits) - 1;
          hits &= hits - 1;
          const int r = __builtin_amdgcn_readlane(row, from);
          const int c = __builtin_amdgcn_readlane(col, from);
          bool taken = false;
#pragma unroll
          for (int j = 0; j < P::TN; j++)
            if (c == 32 * j + (lane & 31)) {
              taken = mine[j] >= 0;
              mine[j] = taken ? mine[j] : r;
            }
          if (__any(taken)) later |= 1ull << from, waiting++;
        }
        hits |= later;
#pragma unroll
        for (int j = 0; j < P::TN; j++) {
          if (mine[j] < 0) continue;
          const float rest = p.rest[mine[j]];
          const T *x = (const T *)p.x + (int64_t)mine[j] * p.width + d0 + 4 * (lane >> 5);
          const int left = p.width - d0 - 4 * (lane >> 5);
#pragma unroll
          for (int i = 0; i < P::TM; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
              typename P::Four y = {};
              if (32 * i + 8 * q < left) y = *(const typename P::Four *)(x + 32 * i + 8 * q);
#pragma unroll
              for (int e = 0; e < 4; e++)
                acc[i][j][4 * q + e] = fmaf(rest, (float)y.v[e], acc[i][j][4 * q + e]);
            }
        }
      }
    }
  });
  tile_barrier();
  const float f = p.unit[1];
  store_rows<T, BM / WM, P::TN>(
      P::slab(wave, a0, b0, a1, b1), lane,
      [&](int i, int j, int q) { return P::four(acc[i][j], q, f); },
      [&](int v, int d) {
        return v0 + v < p.v1 && d0 + d < p.width
                   ? (T *)p.dweight + (int64_t)(v0 + v) * p.width + d0 + d : nullptr;
      });
}

// Both gradients' products of a piece in one launch: dx has few tiles with a
// long sum, which come first, and dw's many short ones fill the machine beside
// and behind them.  Neither needs a transposed copy: the operands' rows lie
// along the result's, and LDS is read transposed.
//
// A quarter of 128256 classes, 4096 x 4096: 2.0 TFLOP over whole tiles in 1.53
// ms, 1.3 PFLOP/s, of which the targets' remainders take 0.04 ms.  Bound by
// power like the logits.
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void loss_grads_kernel(LossDims p, int dt, int nt, int vt) {
  using X = Product<T, BM, BN, WM, WN, true, false>;
  using W = Product<T, BM, BN, WM, WN, true, true>;
  __shared__ __attribute__((aligned(16))) T a0[X::A::ELEMENTS], b0[X::B::ELEMENTS];
  __shared__ __attribute__((aligned(16))) T a1[X::A::ELEMENTS], b1[X::B::ELEMENTS];
  const int xs = dt * nt, id = blockIdx.x;
  int m, n;
  if (id < xs * p.splits) {
    tile_of(id % xs, dt, nt, m, n);
    dx_tile<X>(p, m, n, id / xs, a0, b0, a1, b1);
  } else {
    tile_of(id - xs * p.splits, dt, vt, m, n);
    dw_tile<W>(p, m, n, a0, b0, a1, b1);
  }
}

// The splits' sum, in order, with what g's rounding took off at the target,
// rounded once; zeros for ignored tokens.
template <class T> __global__ __launch_bounds__(256) void loss_dx_join_kernel(LossDims p) {
  struct alignas(8) Four { T v[4]; };
  const int quads = p.width / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t token = i / quads;
  if (token >= p.tokens) return;
  const int d = (int)(i - token * quads) * 4;
  const int at = !p.direct ? p.place[token] : target_of(p, (int)token).counts ? (int)token : -1;
  f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
  if (at >= 0) {
#pragma unroll 4
    for (int s = 0; s < p.splits; s++)
      x += *(const f32x4 *)(p.dx + ((int64_t)s * p.tokens + at) * p.width + d);
  }
  if (at >= 0) {
    const Target t = target_of(p, (int)token);
    if (t.at >= 0) {
      const Four w = *(const Four *)((const T *)p.weight + t.at * p.w_stride + d);
      const float r = p.rest[at];
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = fmaf(r, (float)w.v[e], x[e]);
    }
  }
  Four y;
  const float f = p.unit[1];
#pragma unroll
  for (int e = 0; e < 4; e++) y.v[e] = (T)(x[e] * f);
  *(Four *)((T *)p.dhidden + token * p.width + d) = y;
}

// --------------------------------------------------------------------- host

struct LossPlan {
  bool big;        // 256 x 256 tiles
  int tile;
  int classes;     // of a tile in the forward pass
  int piece;       // classes of a piece
  int splits;
  int64_t bytes;
};

template <class F> static void carve(LossDims &p, char *base, int64_t &used, F &&body) {
  auto take = [&](auto *&ptr, int64_t n) {
    using E = std::remove_reference_t<decltype(*ptr)>;
    ptr = (E *)(base + used);
    used += ceil_div(n * (int64_t)sizeof(E), 256) * 256;
  };
  body(take);
}

static LossPlan plan_loss(const clear_loss_args &a, bool backward, LossDims &p, char *base) {
  require(a.type == CLEAR_BF16 || a.type == CLEAR_FP16, "loss: type is bf16 or fp16");
  require(a.tokens >= 0 && a.vocab >= 1 && a.width >= 8 && a.width % 8 == 0,
          "loss: at least one class, and a width that is a multiple of 8");
  const int64_t most = (int64_t)1 << 30;
  require(a.tokens <= most && a.vocab <= most && a.width <= 1 << 20, "loss: too large");
  p = {};
  p.hidden = a.hidden, p.weight = a.weight, p.targets = (const int64_t *)a.targets;
  p.loss = (float *)a.loss, p.lse = (float *)a.lse, p.dloss = (const float *)a.dloss;
  p.dhidden = a.dhidden, p.dweight = a.dweight;
  p.h_stride = a.h_stride, p.w_stride = a.w_stride, p.ignore = a.ignore_index;
  p.tokens = (int)a.tokens, p.vocab = (int)a.vocab, p.width = (int)a.width;
  LossPlan plan = {};
  // 256 x 256 tiles move half the operand bytes of 128 x 128 ones through LDS,
  // but need enough of them to fill the machine
  plan.big = a.tokens > 128 && ceil_div(a.vocab, 256) * ceil_div(a.tokens, 256) >= 256;
  plan.tile = plan.big ? 256 : 128;
  const int64_t n = a.tokens > 0 ? a.tokens : 1;
  const int64_t small_tiles = ceil_div(a.vocab, 128) * ceil_div(n, 128);
  // One tile of tokens: leaving rows out would save no product, so the list and
  // its launch are left out (64 x 4099 x 256 with gradients: 42 us with a list,
  // 35 without).  The forward pass does without while its products are shorter
  // than what the list takes, sooner where all tiles run at once (two a CU), 0
  // to 0.6 of the tokens ignored: 600 x 6000 x 2000 40-36 us with it, 31 without;
  // 250 x 12920 x 3176 65-67 and 67; 500 x 20000 x 512 (628 tiles) 29-20 and 25.
  // The backward pass needs the list for the targets' remainders too (300 x 3000
  // x 3000 with 0.6 ignored: 67 us with it, 83 without).
  p.direct = a.tokens <= 128 ||
             (!backward && !plan.big &&
              a.tokens * a.vocab <= ((int64_t)1 << (small_tiles <= 512 ? 33 : 31)) / a.width);
  // Tiles fewer than the CUs are bound by a step's latency, which half a tile's
  // copies and products shorten: 5 x 15061 x 4000 63 us whole, 57 in halves; 300 x
  // 2000 x 3000 46 and 31; as many as the CUs (128 x 32000 x 4096): 79 and 77.
  plan.classes = p.direct && !backward && small_tiles < 256 ? 64 : plan.tile;
  // A piece's g takes up to 256 MB, and from 32768 tokens on 8 KB a token: fewer
  // than 4096 classes would have dx's sums read and written for too few products.
  // All pieces have about the same size.
  const int64_t most_piece = std::max<int64_t>(4096, ((int64_t)1 << 27) / n / 256 * 256);
  const int64_t pieces = ceil_div(a.vocab, most_piece);
  plan.piece = (int)(ceil_div(ceil_div(a.vocab, pieces), 256) * 256);
  p.pitch = plan.piece;
  // dx has few tiles and a long sum: shared out until the machine is full
  const int64_t tiles = ceil_div(a.width, plan.tile) * ceil_div(n, plan.tile);
  const int64_t steps = ceil_div(std::min<int64_t>(plan.piece, a.vocab), GEMM_K);
  const int64_t full = plan.big ? 256 : 512;
  plan.splits = (int)std::max<int64_t>(1, std::min<int64_t>(full / tiles, steps / 4));
  p.splits = plan.splits;
  int64_t used = 0;
  carve(p, base, used, [&](auto &&take) {
    uint16_t *x, *g;
    take(p.count, 1), take(p.unit, 2), take(p.row, n), take(p.target, n), take(x, n * a.width);
    p.x = x;
    if (!backward) {
      take(p.hit, n);
      take(p.part, ceil_div(a.vocab, plan.classes) * 2 * n);
    } else {
      take(p.place, n), take(p.lse2, n), take(p.dl, n), take(p.rest, n), take(p.hits, n);
      take(p.hit_start, ceil_div(a.vocab, plan.tile) + 1);
      take(g, n * plan.piece);
      p.g = g;
      take(p.dx, (int64_t)plan.splits * n * a.width);
    }
  });
  plan.bytes = used;
  return plan;
}

static unsigned loss_grid(int64_t n) {
  require(n < (int64_t)1 << 31, "loss: too many blocks");
  return (unsigned)n;
}

// Tokens of a list block: from 1024 on about a thousand blocks, each of which reads
// all targets before its own, so that the reads grow with the tokens alone
// (forward pass of 2^20 x 500 x 64: 0.93 ms; 17.5 at 16 tokens a block, whose
// reads grow with the tokens' square).
template <class T, bool BACKWARD> static void loss_list(const LossDims &p, int tile, hipStream_t st) {
  if (p.direct) return;
  const int rows = std::max(1, p.tokens / 1024);
  const int lists = (int)ceil_div(p.tokens, rows);
  const int64_t tiles = BACKWARD ? ceil_div(p.vocab, tile) : 0;
  loss_list_kernel<T, BACKWARD>
      <<<loss_grid(lists + tiles), LIST_THREADS, 0, st>>>(p, rows, lists, tile);
  launched();
}

template <class T, int BM, int TILE, int WM, int WN, bool GRAD>
static void loss_logits(const LossDims &p, int mt, int nt, hipStream_t st) {
  const unsigned n = loss_grid((int64_t)mt * nt);
  if constexpr (TILE == 128) {
    if (p.direct) {
      loss_logits_kernel<T, BM, TILE, WM, WN, GRAD, true><<<n, 64 * WM * WN, 0, st>>>(p, mt, nt);
      launched();
      return;
    }
  }
  if constexpr (BM == TILE) {
    loss_logits_kernel<T, BM, TILE, WM, WN, GRAD, false><<<n, 64 * WM * WN, 0, st>>>(p, mt, nt);
    launched();
  }
}

// Tiles of BM classes and TILE tokens; BM below TILE only without a list.
template <class T, int BM, int TILE, int WM, int WN>
static void loss_forward_go(LossDims &p, hipStream_t st) {
  loss_list<T, false>(p, TILE, st);
  p.v0 = 0, p.v1 = p.vocab;
  const int mt = (int)ceil_div(p.vocab, BM), nt = (int)ceil_div(p.tokens, TILE);
  loss_logits<T, BM, TILE, WM, WN, false>(p, mt, nt, st);
  // few tokens: more threads a row, which the narrower loads pay for
  if (p.tokens < 2048)
    loss_join_kernel<4><<<loss_grid(ceil_div(p.tokens, 4)), JOIN_THREADS, 0, st>>>(p, mt * WM);
  else
    loss_join_kernel<16><<<loss_grid(ceil_div(p.tokens, 16)), JOIN_THREADS, 0, st>>>(p, mt * WM);
  launched();
}

template <class T, int TILE, int WM, int WN>
static void loss_backward_go(LossDims &p, int piece, hipStream_t st) {
  loss_list<T, true>(p, TILE, st);
  const int dt = (int)ceil_div(p.width, TILE), nt = (int)ceil_div(p.tokens, TILE);
  for (int64_t v = 0; v < p.vocab; v += piece) {
    p.v0 = (int)v, p.v1 = (int)std::min<int64_t>(v + piece, p.vocab);
    p.accumulate = v > 0;
    const int vt = (int)ceil_div(p.v1 - p.v0, TILE);
    loss_logits<T, TILE, TILE, WM, WN, true>(p, vt, nt, st);
    loss_grads_kernel<T, TILE, TILE, WM, WN>
        <<<loss_grid((int64_t)dt * nt * p.splits + (int64_t)dt * vt), 64 * WM * WN, 0, st>>>(
            p, dt, nt, vt);
    launched();
  }
  loss_dx_join_kernel<T>
      <<<loss_grid(ceil_div((int64_t)p.tokens * (p.width / 4), 256)), 256, 0, st>>>(p);
  launched();
}

template <class T> static void loss_go(const LossPlan &plan, LossDims &p, bool backward, hipStream_t st) {
  if (plan.big) {
    if (backward) loss_backward_go<T, 256, 2, 4>(p, plan.piece, st);
    else loss_forward_go<T, 256, 256, 2, 4>(p, st);
  } else {
    if (backward) loss_backward_go<T, 128, 2, 2>(p, plan.piece, st);
    else if (plan.classes == 64) loss_forward_go<T, 64, 128, 2, 2>(p, st);
    else loss_forward_go<T, 128, 128, 2, 2>(p, st);
  }
}

static void loss_call(const clear_loss_args *args, bool backward, void *stream) {
  require(args, "loss: no arguments");
  const clear_loss_args &a = *args;
  LossDims p;
  const LossPlan plan = plan_loss(a, backward, p, (char *)a.workspace);
  if (p.tokens == 0 && !backward) return;
  require(a.weight && (p.tokens == 0 || (a.hidden && a.targets && a.lse)), "loss: null tensor");
  require(a.h_stride >= a.width && a.h_stride <= 1 << 21 && a.w_stride >= a.width &&
              a.w_stride <= 1 << 21 &&
              a.width <= 1 << 20, "loss: strides");
  require(aligned(a.hidden, 16) && aligned(a.weight, 16) && a.h_stride % 8 == 0 &&
              a.w_stride % 8 == 0, "loss: rows start at multiples of 16 bytes");
  require(a.workspace && aligned(a.workspace, 256) && a.workspace_bytes >= plan.bytes,
          "loss: the workspace is too small or misaligned");
  if (backward)
    require(a.dweight && (p.tokens == 0 || (a.dloss && a.dhidden)) && aligned(a.dhidden, 16) &&
                aligned(a.dweight, 16), "loss: null or misaligned gradient");
  else
    require(a.loss, "loss: null output");
  require(p.tokens > 0, "loss: the backward pass needs at least one token");
  hipStream_t st = (hipStream_t)stream;
  if (a.type == CLEAR_BF16) loss_go<__bf16>(plan, p, backward, st);
  else loss_go<_Float16>(plan, p, backward, st);
}

}  // namespace clr

using namespace clr;

extern "C" int clear_loss_workspace(const clear_loss_args *args, int64_t backward, int64_t *bytes) {
  return guarded([&] {
    require(args && bytes, "loss: no arguments");
    LossDims p;
    *bytes = plan_loss(*args, backward != 0, p, nullptr).bytes;
  });
}

extern "C" int clear_loss_forward(const clear_loss_args *args, void *stream) {
  return guarded([&] { loss_call(args, false, stream); });
}

extern "C" int clear_loss_backward(const clear_loss_args *args, void *stream) {
  return guarded([&] { loss_call(args, true, stream); });
}
