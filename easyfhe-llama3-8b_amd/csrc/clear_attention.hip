// Grouped attention of the clear decoder and its gradient.
//
//   s_ij = scale q_i . k_j,  p_ij = exp(s_ij - lse_i) over the visible j,
//   o_i = sum_j p_ij v_j,    delta_i = do_i . o_i,
//   ds_ij = p_ij (do_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i,
//   dv_j = sum_i p_ij do_i.
//
// No score is stored: the forward pass carries a running maximum and sum per
// query, the backward pass computes the probabilities again from lse.
// Statistics and sums are fp32.  p and ds are rounded to the inputs' type, once
// each, as operands of the second products: the matrix units take 16-bit operands
// at sixteen times the rate of fp32's, and either of them in two 16-bit pieces
// would add a quarter to a third to the products.  Error against 64 bits (2-norm,
// rounding the result alone and here), bf16: outputs 1.6e-3 and 1.9e-3 to 2.1e-3,
// with gradients 1.7e-3 and 2.4e-3; fp16 with gradients 2.1e-4 and 3.0e-4.
#include "clear_device.hpp"
#include "clear_host.hpp"

#include <algorithm>

namespace clr {

struct AttnDims {
  const void *q, *k, *v;
  void *out;
  float *lse;
  const int *kv_lens, *q_start;
  const void *dout;
  void *dq, *dk, *dv;
  float *stat;  // backward: [B, H, Tq] of lse in powers of two, then of delta
  float *part;  // split forward: partial outputs, then (maximum, sum)
                // split backward: [parts][2][B, Tk, Hk, D] of dk and dv
  float *dq_part;  // [dq_parts][B, Tq, H, D]
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, o_sb, o_st, o_sh;
  int batch, tq, tk, heads, kv_heads, group, dim, causal;
  int splits, split_keys, parts, dq_parts;
  float scale, scale2;  // scale2: into powers of two
};

__device__ __forceinline__ int visible_len(const AttnDims &p, int b) {
  return p.kv_lens ? min(max(p.kv_lens[b], 0), p.tk) : p.tk;
}
// Query i sees keys up to i + offset (kept where i + offset cannot overflow: the
// host sees to it that queries and keys together leave a tile below 2^31).
__device__ __forceinline__ int causal_offset(const AttnDims &p, int b) {
  return p.q_start ? min(max(p.q_start[b], -p.tq), p.tk) : p.tk - p.tq;
}

// LDS tiles hold PITCH elements a row (the head padded to 64 or 128).
template <int DP> struct Tile {
  static constexpr int PITCH = DP <= 64 ? 64 : 128;
  static constexpr int CHUNKS = PITCH / 8;
  static __device__ __forceinline__ int at(int r, int c) { return c ^ swizzle<2 * PITCH>(r); }
};

// Copies of ROWS rows of a [row][dim] matrix into LDS by THREADS threads, with
// zeros for rows from `hi` on and for the head's padding.  The lanes' offsets
// are the same for every tile; the descriptor's size ends it at row hi.
template <class T, int DP, int ROWS, int THREADS> struct Rows {
  using L = Tile<DP>;
  static constexpr int EACH = ROWS * L::CHUNKS / THREADS;
  const T *base;
  int64_t stride;
  uint32_t at[EACH];

  __device__ __forceinline__ void open(const T *x, int64_t st, int dim, int tid) {
    base = x, stride = st;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int r = (i * THREADS + tid) / L::CHUNKS;
      const int c = L::at(r, (i * THREADS + tid) % L::CHUNKS);
      at[i] = c * 8 < dim ? (uint32_t)((r * st + c * 8) * (int64_t)sizeof(T)) : NOWHERE;
    }
  }
  __device__ __forceinline__ void load(int64_t offset, int row0, int hi, T *lds, int tid) const {
    const int rows = min(max(hi - row0, 0), ROWS);
    const Buffer b = buffer_of(base + offset + row0 * stride,
                               (uint32_t)(rows * stride * (int64_t)sizeof(T)));
#pragma unroll
    for (int i = 0; i < EACH; i++)
      copy_to_lds(b, at[i], lds + (i * THREADS + uniform(tid & ~63)) * 8);
  }
};

// A lane's byte offsets for the two kinds of reads.  Chunk indices enter a
// tile's addresses by XOR below the row's bits, so one offset and a constant
// give every address; `renew` at the head of a step keeps the compiler from
// holding all of them in registers through the loop, which spills.
template <class T, int DP> struct Reads {
  using L = Tile<DP>;
  using X8 = typename Half<T>::x8;
  uint32_t row, col;

  __device__ __forceinline__ void open(int lane) {
    const int c = lane & 31, h = lane >> 5;
    row = c * 2 * L::PITCH + L::at(c, h) * 16;
    const int r = 4 * h + ((lane & 15) >> 2), chunk = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    col = r * 2 * L::PITCH + L::at(r, chunk) * 16 + (lane & 1) * 8;
  }
  __device__ __forceinline__ void renew() { asm volatile("" : "+v"(row), "+v"(col)); }

  // Row r0 + lane % 32 (r0 a multiple of 32), elements 16 s + 8 (lane / 32) + 0..7.
  __device__ __forceinline__ X8 rows(const T *tile, int r0, int s) const {
    return *(const X8 *)((const char *)tile + r0 * 2 * L::PITCH + (row ^ (32 * s)));
  }
  // A operand of the second product: column d0 + lane % 32 of rows
  // r0 + 4h + 0..3 and r0 + 8 + 4h + 0..3, r0 a multiple of 16.
  __device__ __forceinline__ X8 columns(const T *tile, int r0, int d0) const {
    const char *t = (const char *)tile + r0 * 2 * L::PITCH;
    return join<T>(read_transposed(t + (col ^ (2 * d0))),
                   read_transposed(t + 16 * L::PITCH + (col ^ (2 * d0) ^ 32)));
  }
};

// B operand over the head of one row: elements 16 s + 8 h + 0..7, zeros outside.
template <class T, int DP>
__device__ __forceinline__ void row_operand(typename Half<T>::x8 (&f)[DP / 16], const T *row,
                                            bool there, int dim, int h) {
#pragma unroll
  for (int s = 0; s < DP / 16; s++) {
    const int d = 16 * s + 8 * h;
    typename Half<T>::x8 z;
#pragma unroll
    for (int j = 0; j < 8; j++) z[j] = (T)0.0f;
    f[s] = there && d < dim ? *(const typename Half<T>::x8 *)(row + d) : z;
  }
}

// ------------------------------------------------------------------ forward

// A probability enters the second product rounded to the inputs' type, as 2^UP
// times its power relative to a maximum that lags by up to 2^SLACK.  fp16 has no
// numbers below 2^-25: carried up to its largest ones, powers down to 2^-38 of a
// row's largest count, so that 2^20 small ones are not lost behind one key with
// most of the mass.  (Relative to the maximum alone, as bf16 takes them, 40000
// keys of 2^-26 round to an output of 0 in place of 6e-4.)
template <class T> struct Powers;
template <> struct Powers<__bf16> { static constexpr float SLACK = 8.0f, UP = 0.0f; };
template <> struct Powers<_Float16> { static constexpr float SLACK = 2.0f, UP = 13.0f; };

// Running softmax of one query column over 32 RS keys, and the output's update.
template <class T, int DP, int RS> struct Running {
  f32x16 o[DP / 32];
  float m, l;  // o and l carry 2^UP until `finish`, which puts it into m

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < DP / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    m = -INFINITY, l = 0.0f;
  }
  __device__ __forceinline__ void finish() { l = halves_sum(l), m -= Powers<T>::UP; }

  // The K and V tiles' first row is key0, and the column sees keys below
  // `limit` (`masked`, the same for the wave) or all of them.
  __device__ __forceinline__ void step(const typename Half<T>::x8 (&qf)[DP / 16], const T *kt,
                                       const T *vt, Reads<T, DP> &rd, int key0, int limit,
                                       bool masked, float scale2, int lane) {
    const int h = lane >> 5;
    rd.renew();
    f32x16 s[RS];
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < RS; r++)
#pragma unroll
      for (int i = 0; i < 16; i++) s[r][i] = 0.0f;
#pragma unroll
    for (int d = 0; d < DP / 16; d++)
#pragma unroll
      for (int r = 0; r < RS; r++)
        s[r] = Half<T>::mma(rd.rows(kt, 32 * r, d), qf[d], s[r]);
    interleave<RS * DP / 16, 4, 1>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    // the products and the softmax between them keep to their places: drawn
    // together they need more registers than two waves a SIMD leave
    __builtin_amdgcn_sched_barrier(0);
    if (masked) {
#pragma unroll
      for (int r = 0; r < RS; r++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int key = key0 + 32 * r + 8 * (i >> 2) + 4 * h + (i & 3);
          s[r][i] = key < limit ? s[r][i] : -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int r = 0; r < RS; r++)
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, s[r][i]);
    top = halves_max(top) * scale2;
    // The maximum only has to keep the powers in range: it moves when the new one
    // is more than the slack above, so most steps leave the outputs as they are.
    if (__any(top > m + Powers<T>::SLACK)) {
      const float next = fmaxf(m, top);
      const float f = m == -INFINITY ? 0.0f : exp2_fast(m - next);
      l *= f;
#pragma unroll
      for (int d = 0; d < DP / 32; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] *= f;
      m = next;
    }
    const float shift = m == -INFINITY ? 0.0f : m - Powers<T>::UP;
    auto powers = [&](int r) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        s[r][i] = exp2_fast(fmaf(s[r][i], scale2, -shift));
        sum += s[r][i];
      }
      l += sum;
    };
    // the powers of the next 32 keys are taken while those before them multiply
    powers(0);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int r = 0; r < RS; r++) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const auto pf = narrow<T>(s[r], 8 * k);
#pragma unroll
        for (int d = 0; d < DP / 32; d++)
          o[d] = Half<T>::mma(rd.columns(vt, 32 * r + 16 * k, 32 * d), pf, o[d]);
      }
      if (r + 1 < RS) {
        powers(r + 1);
        interleave<2 * DP / 32, 4, 2, 48 * 32 / (2 * DP)>();
      } else {
        interleave<2 * DP / 32, 4, 2>();
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
  }
};

// log sum_j exp(s_j) of a row from its running maximum and sum (both in powers of
// two).  The sum is 0 only where the row sees nothing, or nothing but scores of
// -inf; NaN scores leave the maximum alone, so it is the sum that tells of them.
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.0f ? -INFINITY : (m + __log2f(l)) * LN2;
}

// Four output elements 8 b + 4 h + 0..3 of each 32, rounded once.
template <class T, int DP>
__device__ __forceinline__ void store_columns(T *row, const f32x16 (&o)[DP / 32], float f, int dim,
                                              int h) {
  struct alignas(8) Four { T v[4]; };
#pragma unroll
  for (int d = 0; d < DP / 32; d++)
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const int at = 32 * d + 8 * b + 4 * h;
      if (at < dim) {
        Four x;
#pragma unroll
        for (int j = 0; j < 4; j++) x.v[j] = (T)(o[d][4 * b + j] * f);
        *(Four *)(row + at) = x;
      }
    }
}

// The same four in fp32, unscaled.
template <int DP>
__device__ __forceinline__ void store_sums(float *row, const f32x16 (&o)[DP / 32], int dim, int h) {
#pragma unroll
  for (int d = 0; d < DP / 32; d++)
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const int at = 32 * d + 8 * b + 4 * h;
      f32x4 x;
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = o[d][4 * b + j];
      if (at < dim) *(f32x4 *)(row + at) = x;
    }
}

constexpr int FWD_WAVES = 4, FWD_ROWS = 32 * FWD_WAVES, FWD_KEYS = 64;

// Many queries: a block takes 128 queries of one head, a wave 32 of them as
// columns, and 64 keys at a time go through LDS in two buffers.  Two blocks
// share a CU: one's products run beside the other's powers, and waves that
// multiply go first.
//
// 2 x 4096 causal tokens, 32 and 8 heads of 128, bf16: 275 GFLOP in 275-290 us,
// 0.95-1.0 PFLOP/s (a library product of 8192^3: 1.38).  The matrix units are
// busy 48% of the cycles, the vector unit about as long (a power is a quarter
// of the rate of other instructions); the clock is at 1.85 GHz of 2.4 under
// this load.  Heads of 64 have as many powers for half the products: the vector
// unit bounds them.
template <class T, int DP>
__global__ __launch_bounds__(64 * FWD_WAVES, 2) void attention_forward_kernel(AttnDims p) {
  using L = Tile<DP>;
  __shared__ __attribute__((aligned(16))) T k0[FWD_KEYS * L::PITCH], k1[FWD_KEYS * L::PITCH];
  __shared__ __attribute__((aligned(16))) T v0[FWD_KEYS * L::PITCH], v1[FWD_KEYS * L::PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
  // Blocks of one key head differ by a multiple of B Hk: with eight XCDs taking
  // blocks in turn they mostly share an L2, and the longest rows come first.
  const int pairs = p.batch * p.kv_heads;
  const int pair = blockIdx.x % pairs, split = blockIdx.x / pairs % p.splits;
  const int rest = blockIdx.x / pairs / p.splits;
  const int b = pair / p.kv_heads, kvh = pair % p.kv_heads;
  const int tiles = (p.tq + FWD_ROWS - 1) / FWD_ROWS;
  const int q0 = (tiles - 1 - rest / p.group) * FWD_ROWS;
  const int head = kvh * p.group + rest % p.group;
  const int qi = q0 + wave * 32 + (lane & 31);
  const int len = visible_len(p, b), off = causal_offset(p, b);
  const int begin = split * p.split_keys;
  if (p.splits > 1 && begin >= len) return;  // the join leaves these splits out
  const bool there = qi < p.tq;
  const int limit = p.causal ? max(0, min(len, qi + off + 1)) : len;
  const int last = min(q0 + FWD_ROWS, p.tq) - 1;
  const int end = min(p.causal ? max(0, min(len, last + off + 1)) : len, begin + p.split_keys);
  // all queries of the wave see keys below `open`
  const int open = p.causal ? min(len, q0 + wave * 32 + off + 1) : len;
  // and none of them sees keys from `closed` on
  const int closed = p.causal ? min(len, q0 + wave * 32 + 31 + off + 1) : len;
  typename Half<T>::x8 qf[DP / 16];
  row_operand<T, DP>(qf, (const T *)p.q + b * p.q_sb + (int64_t)qi * p.q_st + head * p.q_sh, there,
                     p.dim, h);
  const T *kb = (const T *)p.k + b * p.k_sb + kvh * p.k_sh;
  const T *vb = (const T *)p.v + b * p.v_sb + kvh * p.v_sh;
  Running<T, DP, 2> run;
  run.clear();
  Reads<T, DP> rd;
  rd.open(lane);
  Rows<T, DP, FWD_KEYS, 64 * FWD_WAVES> krows, vrows;
  krows.open(kb, p.k_st, p.dim, tid), vrows.open(vb, p.v_st, p.dim, tid);
  auto load = [&](int key, T *k, T *v) {
    krows.load(0, key, end, k, tid), vrows.load(0, key, end, v, tid);
  };
  auto use = [&](int key, const T *k, const T *v) {
    if (key >= closed) return;
    run.step(qf, k, v, rd, key, min(limit, end), key + FWD_KEYS > min(open, end), p.scale2, lane);
  };
  if (begin < end) load(begin, k0, v0);
  for (int key = begin; key < end; key += 2 * FWD_KEYS) {
    tile_barrier();
    if (key + FWD_KEYS < end) load(key + FWD_KEYS, k1, v1);
    use(key, k0, v0);
    tile_barrier();
    if (key + 2 * FWD_KEYS < end) load(key + 2 * FWD_KEYS, k0, v0);
    if (key + FWD_KEYS < end) use(key + FWD_KEYS, k1, v1);
  }
  if (!there) return;
  run.finish();
  const float l = run.l;
  if (p.splits > 1) {
    const int64_t rows = (int64_t)p.batch * p.tq * p.heads;
    const int64_t row = ((int64_t)b * p.tq + qi) * p.heads + head;
    if (h == 0)
      ((float2 *)(p.part + p.splits * rows * p.dim))[split * rows + row] = make_float2(run.m, l);
    store_sums<DP>(p.part + (split * rows + row) * p.dim, run.o, p.dim, h);
    return;
  }
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  store_columns<T, DP>((T *)p.out + ((int64_t)(b * (int64_t)p.tq + qi) * p.heads + head) * p.dim,
                       run.o, f, p.dim, h);
  if (h == 0)
    p.lse[((int64_t)b * p.heads + head) * p.tq + qi] = row_lse(run.m, l);
}

// Few queries: the queries of a group's heads are packed into the 32 columns,
// and the keys are shared out, first over blocks, then over a block's waves.
// Each wave streams its own keys through its own part of LDS, 32 at a time in
// two buffers, and waits for no other until the end, where the four partial
// results are joined in LDS.  The columns that no query fills cost matrix time
// that the memory's leaves free.
//
// One token of 16 sequences, caches of up to 16384 filled to about half, 8 key
// heads of 128: about 540 MB in 100-115 us, 4.9-5.3 TB/s, as fast as a copy.
constexpr int FEW_WAVES = 4, FEW_KEYS = 32;

template <class T, int DP>
__global__ __launch_bounds__(64 * FEW_WAVES, 1) void attention_few_kernel(AttnDims p) {
  using L = Tile<DP>;
  constexpr int N = FEW_KEYS * L::PITCH;
  constexpr int COPIES = 2 * FEW_KEYS * L::CHUNKS / 64;
  __shared__ __attribute__((aligned(16))) T k0[FEW_WAVES * N], k1[FEW_WAVES * N];
  __shared__ __attribute__((aligned(16))) T v0[FEW_WAVES * N], v1[FEW_WAVES * N];
  __shared__ float2 ml[FEW_WAVES][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
  const int pairs = p.batch * p.kv_heads;
  const int pair = blockIdx.x % pairs, split = blockIdx.x / pairs;
  const int b = pair / p.kv_heads, kvh = pair % p.kv_heads;
  const int column = blockIdx.y * 32 + (lane & 31);
  const int qi = column / p.group, head = kvh * p.group + column % p.group;
  const bool there = qi < p.tq;
  const int len = visible_len(p, b), off = causal_offset(p, b);
  const int begin = split * p.split_keys;
  if (p.splits > 1 && begin >= len) return;  // the join leaves these splits out
  const int limit = p.causal ? max(0, min(len, qi + off + 1)) : len;
  const int last = min((int)(blockIdx.y * 32 + 31) / p.group, p.tq - 1);
  const int end = min(begin + p.split_keys, p.causal ? max(0, min(len, last + off + 1)) : len);
  const int first = min((int)(blockIdx.y * 32) / p.group, p.tq - 1);
  const int open = p.causal ? min(len, first + off + 1) : len;
  typename Half<T>::x8 qf[DP / 16];
  row_operand<T, DP>(qf, (const T *)p.q + b * p.q_sb + (int64_t)qi * p.q_st + head * p.q_sh, there,
                     p.dim, h);
  const T *kb = (const T *)p.k + b * p.k_sb + kvh * p.k_sh;
  const T *vb = (const T *)p.v + b * p.v_sb + kvh * p.v_sh;
  Running<T, DP, 1> run;
  run.clear();
  Reads<T, DP> rd;
  rd.open(lane);
  T *kw0 = k0 + wave * N, *kw1 = k1 + wave * N, *vw0 = v0 + wave * N, *vw1 = v1 + wave * N;
  Rows<T, DP, FEW_KEYS, 64> krows, vrows;
  krows.open(kb, p.k_st, p.dim, lane), vrows.open(vb, p.v_st, p.dim, lane);
  auto load = [&](int key, T *k, T *v) {
    krows.load(0, key, end, k, lane), vrows.load(0, key, end, v, lane);
  };
  auto use = [&](int key, const T *k, const T *v) {
    run.step(qf, k, v, rd, key, min(limit, end), key + FEW_KEYS > min(open, end), p.scale2, lane);
  };
  constexpr int STEP = FEW_WAVES * FEW_KEYS;
  int key = begin + wave * FEW_KEYS;
  if (key < end) load(key, kw0, vw0);
  for (; key + STEP < end; key += 2 * STEP) {
    wait_lds();
    load(key + STEP, kw1, vw1);
    wait_global<COPIES>();
    use(key, kw0, vw0);
    wait_lds();
    if (key + 2 * STEP < end) {
      load(key + 2 * STEP, kw0, vw0);
      wait_global<COPIES>();
    } else {
      wait_global<0>();
    }
    use(key + STEP, kw1, vw1);
  }
  if (key < end) {
    wait_global<0>();
    use(key, kw0, vw0);
  }
  // Join: every wave's outputs relative to the common maximum.
  run.finish();
  if (h == 0) ml[wave][lane & 31] = make_float2(run.m, run.l);
  __syncthreads();
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int w = 0; w < FEW_WAVES; w++) m = fmaxf(m, ml[w][lane & 31].x);
#pragma unroll
  for (int w = 0; w < FEW_WAVES; w++) {
    const float2 x = ml[w][lane & 31];
    l += x.x == -INFINITY ? x.y : x.y * exp2_fast(x.x - m);  // x.y: 0, or NaN
  }
  const float mine = run.m == -INFINITY ? 0.0f : exp2_fast(run.m - m);
  // The waves' 32 x DP outputs: k0 and v0 are free, one wave needs DP / 32
  // tiles of 4 KB, and two waves fit each array.
  constexpr int WAVE_FLOATS = 32 * DP;
  static_assert(2 * WAVE_FLOATS * 4 <= (int)sizeof(k0), "two waves' outputs fit one array");
  auto slab = [&](int w) { return (float *)(w < 2 ? k0 : v0) + (w & 1) * WAVE_FLOATS; };
  float *own = slab(wave);
#pragma unroll
  for (int d = 0; d < DP / 32; d++)
#pragma unroll
    for (int bq = 0; bq < 4; bq++) {
      f32x4 x;
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = run.o[d][4 * bq + j] * mine;
      // [32 d + 8 bq + 4 h .. + 3][column], columns of quads side by side
      *(f32x4 *)(own + ((d * 8 + bq * 2 + h) * 32 + (lane & 31)) * 4) = x;
    }
  __syncthreads();
  const int quads = DP / 4;
  for (int i = tid; i < quads * 32; i += 64 * FEW_WAVES) {
    const int c = i & 31, quad = i >> 5;
    f32x4 x = *(const f32x4 *)(slab(0) + i * 4);
#pragma unroll
    for (int w = 1; w < FEW_WAVES; w++) x += *(const f32x4 *)(slab(w) + i * 4);
    const int col = blockIdx.y * 32 + c, q = col / p.group, hd = kvh * p.group + col % p.group;
    if (q >= p.tq || quad * 4 >= p.dim) continue;
    const int64_t row = ((int64_t)b * p.tq + q) * p.heads + hd;
    // c is this thread's own column as lane & 31 is: m and l are that column's
    if (p.splits == 1) {
      struct alignas(8) Four { T v[4]; } y;
      const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int j = 0; j < 4; j++) y.v[j] = (T)(x[j] * f);
      *(Four *)((T *)p.out + row * p.dim + quad * 4) = y;
    } else {
      const int64_t rows = (int64_t)p.batch * p.tq * p.heads;
      *(f32x4 *)(p.part + (split * rows + row) * p.dim + quad * 4) = x;
    }
  }
  if (tid < 32 && there) {
    const int64_t row = ((int64_t)b * p.tq + qi) * p.heads + head;
    if (p.splits == 1) {
      p.lse[((int64_t)b * p.heads + head) * p.tq + qi] = row_lse(m, l);
    } else {
      const int64_t rows = (int64_t)p.batch * p.tq * p.heads;
      float2 *stats = (float2 *)(p.part + p.splits * rows * p.dim);
      stats[split * rows + row] = make_float2(m, l);
    }
  }
}

// The splits' partial outputs of one row, in order; a wave a row (6 us for 512
// rows of 16 splits).
template <class T>
__global__ __launch_bounds__(64) void attention_join_kernel(AttnDims p) {
  const int64_t rows = (int64_t)p.batch * p.tq * p.heads;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const float2 *stats = (const float2 *)(p.part + p.splits * rows * p.dim);
  const int head = (int)(row % p.heads);
  const int64_t bq = row / p.heads;
  const int b = (int)(bq / p.tq), qi = (int)(bq % p.tq);
  // splits from the sequence's length on have seen nothing
  const int splits = min(p.splits, (visible_len(p, b) + p.split_keys - 1) / p.split_keys);
  float m = -INFINITY, l = 0.0f;
  for (int s = lane; s < splits; s += 64) m = fmaxf(m, stats[s * rows + row].x);
  for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  for (int s = lane; s < splits; s += 64) {
    const float2 t = stats[s * rows + row];
    l += t.x == -INFINITY ? t.y : t.y * exp2_fast(t.x - m);  // t.y: 0, or NaN
  }
  for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x, 64);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int d = 2 * lane; d < p.dim; d += 128) {
    float a0 = 0.0f, a1 = 0.0f;
#pragma unroll 4
    for (int s = 0; s < splits; s++) {
      const float t = stats[s * rows + row].x;
      const float f = t == -INFINITY ? 0.0f : exp2_fast(t - m);
      const float2 x = *(const float2 *)(p.part + (s * rows + row) * p.dim + d);
      a0 += x.x * f, a1 += x.y * f;
    }
    T *y = (T *)p.out + row * p.dim + d;
    y[0] = (T)(a0 * inv), y[1] = (T)(a1 * inv);
  }
  if (lane == 0)
    p.lse[((int64_t)b * p.heads + head) * p.tq + qi] = row_lse(m, l);
}

// ----------------------------------------------------------------- backward

constexpr int BWD_WAVES = 4;

// The backward kernels carry p times 2^15: fp16 then keeps small probabilities
// away from its smallest numbers, and fp32's power is not cut off at 2^-126.
// A score gradient keeps the factor in bf16, whose range allows it, and loses
// it in fp16, where do . v decides its size.
constexpr float P_LOG = 15.0f, P_UP = 32768.0f;
template <class T> struct Carried;
template <> struct Carried<__bf16> {
  static constexpr float DOWN = 1.0f, LEFT = 1.0f / P_UP;
  static constexpr bool ENDS = false;
};
template <> struct Carried<_Float16> {
  static constexpr float DOWN = 1.0f / P_UP, LEFT = 1.0f;
  static constexpr bool ENDS = true;
};

// In fp16 a score gradient may be beyond the largest number where the sums that
// it goes into, times the scale, are not: a column's sums are then infinite or
// NaN in every element (infinity times 0 is NaN), so one of them tells.  The
// block takes such columns again, in units of 2^13 and at last of 2^26, which
// hold any do . v of fp16 operands (128 x 2^32, twice).  What that loses, below
// 2^-12 of a number beyond 2^16 (2 of one beyond 2^29), is less than the large
// one's rounding.
constexpr float FEWER = 1.0f / 8192.0f, FEWEST = FEWER * FEWER;

// Whether a column of the block is lost, the same for all of its lanes; those lanes
// whose own is get the next unit.
template <int WAVES> __device__ __forceinline__ bool lost_columns(float sum, float &unit, int *votes) {
  const bool lost = !(halves_sum(sum * 0.0f) == 0.0f) && unit > FEWEST;
  votes[threadIdx.x >> 6] = __any(lost);
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) any |= votes[w];
  unit *= lost ? FEWER : 1.0f;
  return uniform(any) != 0;
}

// block(dims, thread, block, unit, again) until it returns false.  Nearly every
// call takes nothing again and should not pay for it with registers: its arguments
// and its place are hidden from the compiler, which would keep what follows from
// them for the next time.  5 x 1003 uneven tokens with 12 heads of 64, forward and
// backward, of four sets of lengths: 52-83 us without any of this, 53-84 with it,
// 53-94 where nothing is hidden (a block less a CU); 2 x 4096 causal tokens of 32
// and 8 heads of 128 1.304, 1.310 and 1.34 ms; 4 x 128 of them 44, 46 and 47 us.
template <class T, class F> __device__ __forceinline__ void blocks(const AttnDims &p, F &&block) {
  float unit = 1.0f;
  if constexpr (!Carried<T>::ENDS) {
    block(p, (int)threadIdx.x, (int)blockIdx.x, unit, false);
  } else {
    for (bool again = false;; again = true) {
      // the kernel's one argument
      typedef const __attribute__((address_space(4))) AttnDims *Argument;
      Argument a = (Argument)__builtin_amdgcn_kernarg_segment_ptr();
      int thread = threadIdx.x, index = blockIdx.x;
      asm volatile("" : "+s"(a), "+v"(thread), "+s"(index));
      if (__builtin_expect(!block(*(const AttnDims *)a, thread, index, unit, again), 1)) break;
    }
  }
}

// dq of 128 queries of one head, and each query's (lse, delta) for the keys'
// gradients.  The columns are queries, so both statistics are the lane's own.
// Delta is taken from the rounded output, which is what the forward pass
// leaves: off by half a step over the root of the number of keys that share the
// row's mass.  Tiles that see up to 128 keys, where this counts, have all of
// them in LDS at once and take delta_i = sum_j p_ij do_i . v_j first: 24 causal
// tokens in bf16, error of dq and dk 2.9e-3 without and 2.3e-3 with (the score
// gradients' and the result's own rounding), for 3 us more where no query sees
// more keys (128 causal tokens, 32 and 8 heads of 128: 29.5 and 32.4 us of
// backward pass), nothing at 600 and more.  Keys go by 64 in two halves: one's
// scores multiply while the other's gradients are taken.
//
// 2 x 4096 causal tokens, 32 and 8 heads of 128, bf16: 412 GFLOP in 370 us, 1.1
// PFLOP/s, the matrix units busy 60% of the cycles at 1.75 GHz (one half at a
// time: 421 us).
template <class T, int DP>
__device__ __forceinline__ bool dq_block(const AttnDims &p, int tid, int block, float &unit) {
  using L = Tile<DP>;
  constexpr int ROWS = 32 * BWD_WAVES, KEYS = 64;
  __shared__ __attribute__((aligned(16))) T k0[KEYS * L::PITCH], k1[KEYS * L::PITCH];
  __shared__ __attribute__((aligned(16))) T v0[KEYS * L::PITCH], v1[KEYS * L::PITCH];
  const int lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5, c = lane & 31;
  const int pairs = p.batch * p.kv_heads;
  const int pair = block % pairs, part = block / pairs % p.dq_parts;
  const int rest = block / pairs / p.dq_parts;
  const int b = pair / p.kv_heads, kvh = pair % p.kv_heads;
  const int tiles = (p.tq + ROWS - 1) / ROWS;
  const int q0 = (tiles - 1 - rest / p.group) * ROWS;
  const int head = kvh * p.group + rest % p.group;
  const int qi = q0 + wave * 32 + c;
  const int len = visible_len(p, b), off = causal_offset(p, b);
  const bool there = qi < p.tq;
  const int limit = p.causal ? max(0, min(len, qi + off + 1)) : len;
  const int last = min(q0 + ROWS, p.tq) - 1;
  // the part's share of all keys
  const int share = ((p.tk + KEYS - 1) / KEYS + p.dq_parts - 1) / p.dq_parts * KEYS;
  const int begin = part * share;
  const int all = p.causal ? max(0, min(len, last + off + 1)) : len;
  const int end = min(all, begin + share);
  const bool few = all <= 2 * KEYS && end == all && begin == 0;
  const int open = p.causal ? min(len, q0 + wave * 32 + off + 1) : len;
  const int closed = p.causal ? min(len, q0 + wave * 32 + 31 + off + 1) : len;
  // a query that sees nothing takes no part: its dout may hold anything
  const bool live = there && limit > 0;
  typename Half<T>::x8 qf[DP / 16], df[DP / 16];
  row_operand<T, DP>(qf, (const T *)p.q + b * p.q_sb + (int64_t)qi * p.q_st + head * p.q_sh, live,
                     p.dim, h);
  row_operand<T, DP>(df, (const T *)p.dout + b * p.o_sb + (int64_t)qi * p.o_st + head * p.o_sh,
                     live, p.dim, h);
  float delta = 0.0f;
  const T *orow = (const T *)p.out + ((int64_t)(b * (int64_t)p.tq + qi) * p.heads + head) * p.dim;
#pragma unroll
  for (int s = 0; s < DP / 16; s++) {
    const int d = 16 * s + 8 * h;
    if (live && d < p.dim) {
      const auto o8 = *(const typename Half<T>::x8 *)(orow + d);
#pragma unroll
      for (int j = 0; j < 8; j++) delta = fmaf((float)o8[j], (float)df[s][j], delta);
    }
  }
  const int64_t at = ((int64_t)b * p.heads + head) * p.tq + qi;
  // nor does one that sees nothing but scores of -inf, whose output is 0 as well
  const float lse = live ? p.lse[at] : -INFINITY;
  const float lse2 = lse == -INFINITY ? INFINITY : fmaf(lse, LOG2E, -P_LOG);
  const T *kb = (const T *)p.k + b * p.k_sb + kvh * p.k_sh;
  const T *vb = (const T *)p.v + b * p.v_sb + kvh * p.v_sh;
  f32x16 dq[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) dq[d][i] = 0.0f;
  Rows<T, DP, KEYS, 64 * BWD_WAVES> krows, vrows;
  krows.open(kb, p.k_st, p.dim, tid), vrows.open(vb, p.v_st, p.dim, tid);
  auto load = [&](int key, T *k, T *v) {
    krows.load(0, key, end, k, tid), vrows.load(0, key, end, v, tid);
  };
  Reads<T, DP> rd;
  rd.open(lane);
  if (begin < end) load(begin, k0, v0);
  if (few) {
    if (KEYS < end) load(KEYS, k1, v1);
    tile_barrier();
    delta = 0.0f;
#pragma unroll 1
    for (int key = 0; key < min(closed, end); key += 32) {
      const T *k = (key < KEYS ? k0 : k1) + key % KEYS * L::PITCH;
      const T *v = (key < KEYS ? v0 : v1) + key % KEYS * L::PITCH;
      rd.renew();
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; i++) s[i] = 0.0f, dp[i] = 0.0f;
#pragma unroll
      for (int d = 0; d < DP / 16; d++) {
        s = Half<T>::mma(rd.rows(k, 0, d), qf[d], s);
        dp = Half<T>::mma(rd.rows(v, 0, d), df[d], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const bool seen = key + 8 * (i >> 2) + 4 * h + (i & 3) < min(limit, end);
        const float x = exp2_fast(fmaf(s[i], p.scale2, -lse2)) * dp[i];
        delta += seen ? x : 0.0f;
      }
    }
    delta *= 1.0f / P_UP;
  }
  delta = halves_sum(delta) * Carried<T>::DOWN;
  if (there && h == 0 && part == 0) {
    const int64_t n = (int64_t)p.batch * p.heads * p.tq;
    p.stat[at] = lse2, p.stat[n + at] = delta;
  }
  // the score gradients' unit, which is 1 unless they are taken again
  const float down = Carried<T>::DOWN * unit, shift = delta * unit;
  auto use = [&](int key, const T *k, const T *v) {
    if (key >= closed) return;
    rd.renew();
    f32x16 s[2], dp[2];
    auto scores = [&](int r) {
#pragma unroll
      for (int i = 0; i < 16; i++) s[r][i] = 0.0f, dp[r][i] = 0.0f;
#pragma unroll
      for (int d = 0; d < DP / 16; d++) {
        s[r] = Half<T>::mma(rd.rows(k, 32 * r, d), qf[d], s[r]);
        dp[r] = Half<T>::mma(rd.rows(v, 32 * r, d), df[d], dp[r]);
      }
    };
    auto gradients = [&](int r) {
#pragma unroll
      for (int i = 0; i < 16; i++)
        s[r][i] = exp2_fast(fmaf(s[r][i], p.scale2, -lse2)) * fmaf(dp[r][i], down, -shift);
    };
    auto add = [&](int r) {
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        const auto sf = narrow<T>(s[r], 8 * kk);
#pragma unroll
        for (int d = 0; d < DP / 32; d++)
          dq[d] = Half<T>::mma(rd.columns(k, 32 * r + 16 * kk, 32 * d), sf, dq[d]);
      }
    };
    static_assert(KEYS == 64, "two halves");
    __builtin_amdgcn_sched_barrier(0);
    scores(0);
    interleave<DP / 8, 4, 1>();
    __builtin_amdgcn_sched_barrier(0);
    // the second half's products run while the first one's gradients are taken
    scores(1);
    gradients(0);
    interleave<DP / 8, 4, 1, 64 * 8 / DP>();
    __builtin_amdgcn_sched_barrier(0);
    if (key + KEYS > min(open, end)) {
#pragma unroll
      for (int i = 0; i < 16; i++) {
        s[0][i] = key + 8 * (i >> 2) + 4 * h + (i & 3) < min(limit, end) ? s[0][i] : 0.0f;
        // a hidden key's score leaves no power to take
        s[1][i] = key + 32 + 8 * (i >> 2) + 4 * h + (i & 3) < min(limit, end) ? s[1][i] : -INFINITY;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    add(0);
    gradients(1);
    interleave<DP / 16, 4, 2, 64 * 16 / DP>();
    __builtin_amdgcn_sched_barrier(0);
    add(1);
    interleave<DP / 16, 4, 2>();
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int key = begin; key < end; key += 2 * KEYS) {
    tile_barrier();
    if (key + KEYS < end && !few) load(key + KEYS, k1, v1);
    use(key, k0, v0);
    tile_barrier();
    if (key + 2 * KEYS < end) load(key + 2 * KEYS, k0, v0);
    if (key + KEYS < end) use(key + KEYS, k1, v1);
  }
  if constexpr (Carried<T>::ENDS) {
    __shared__ int votes[BWD_WAVES];
    const float used = unit;
    if (lost_columns<BWD_WAVES>(dq[0][0], unit, votes)) return true;
    if (p.dq_parts > 1) {
#pragma unroll
      for (int d = 0; d < DP / 32; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) dq[d][i] *= 1.0f / used;
    }
  }
  if (there && p.dq_parts > 1) {
    const int64_t rows = (int64_t)p.batch * p.tq * p.heads;
    store_sums<DP>(p.dq_part + (part * rows + ((int64_t)b * p.tq + qi) * p.heads + head) * p.dim, dq,
                   p.dim, h);
    return false;
  }
  if (there)
    store_columns<T, DP>((T *)p.dq + ((int64_t)(b * (int64_t)p.tq + qi) * p.heads + head) * p.dim,
                         dq, p.scale * Carried<T>::LEFT / unit, p.dim, h);
  return false;
}

template <class T, int DP>
__global__ __launch_bounds__(64 * BWD_WAVES, 2) void attention_dq_kernel(AttnDims p) {
  blocks<T>(p, [](const AttnDims &a, int tid, int block, float &unit, bool) {
    return dq_block<T, DP>(a, tid, block, unit);
  });
}

// dk and dv of 32 WAVES keys of one key head: the columns are keys, and the group's
// queries go by 64 at a time, so the sum over shared heads stays in registers
// and has one order.  Two sets of WAVES waves take 32 of the 64 queries each,
// which puts two waves on a SIMD while one block has the CU to itself: blocks
// of very different lengths (a causal mask) are then handed out longest first
// to whichever CU is free.  The sets' sums are joined in LDS at the end.
//
// The same sizes: 550 GFLOP in 580-610 us, 0.9-0.95 PFLOP/s, the matrix units
// busy 45% of the cycles at 1.7 GHz.  On four waves with the operands of k and v
// in registers one wave a SIMD took 866 us; with v read from LDS 512 registers
// a SIMD do for two.  dq has a kernel of its own, which computes scores and
// probabilities a second time (7 products in place of 5): adding up dq over the
// key tiles would need atomics, whose order changes results.
//
// Few key tiles (short sequences, few key heads) would leave most CUs without
// a block: the queries are then shared out over `parts` blocks a tile, whose
// fp32 sums a second kernel adds in order.
template <class T, int DP, int WAVES>
__device__ __forceinline__ bool dkv_block(const AttnDims &p, int tid, int block, float &unit, bool again) {
  using L = Tile<DP>;
  constexpr int COLS = 32 * WAVES, ROWS = 64, THREADS = 128 * WAVES;
  __shared__ __attribute__((aligned(16))) T q0[ROWS * L::PITCH], q1[ROWS * L::PITCH];
  __shared__ __attribute__((aligned(16))) T d0[ROWS * L::PITCH], d1[ROWS * L::PITCH];
  __shared__ __attribute__((aligned(16))) T vt[COLS * L::PITCH];
  __shared__ __attribute__((aligned(16))) float st0[2 * 64], st1[2 * 64];
  const int set = uniform(tid / (64 * WAVES)), lane = tid & 63, wave = uniform(tid >> 6) & (WAVES - 1), h = lane >> 5, c = lane & 31;
  const int pairs = p.batch * p.kv_heads;
  const int pair = block % pairs;
  const int b = pair / p.kv_heads, kvh = pair % p.kv_heads;
  const int part = block / pairs % p.parts;
  const int first_key = block / pairs / p.parts * COLS;  // the longest first
  const int key = first_key + wave * 32 + c;
  const int len = visible_len(p, b), off = causal_offset(p, b);
  const bool there = key < len;
  typename Half<T>::x8 kf[DP / 16];
  row_operand<T, DP>(kf, (const T *)p.k + b * p.k_sb + (int64_t)key * p.k_st + kvh * p.k_sh, there,
                     p.dim, h);
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) dk[d][i] = 0.0f, dv[d][i] = 0.0f;
  // queries that see a key of this block, and the first that sees any key
  const int lo = p.causal ? max(0, -off) : 0;
  const int from = p.causal ? max(lo, first_key - off) : 0;
  const int to = first_key < len ? p.tq : 0;
  const int per_head = to > from ? (to - from + ROWS - 1) / ROWS : 0;
  const int all_steps = per_head * p.group, share = (all_steps + p.parts - 1) / p.parts;
  const int first_step = min(part * share, all_steps);
  const int steps = min(share, all_steps - first_step);
  const int64_t n = (int64_t)p.batch * p.heads * p.tq;
  Rows<T, DP, ROWS, THREADS> qrows, drows;
  qrows.open((const T *)p.q + b * p.q_sb, p.q_st, p.dim, tid);
  drows.open((const T *)p.dout + b * p.o_sb, p.o_st, p.dim, tid);
  // the next step's head of the group and first row
  int load_head = steps > 0 ? first_step / per_head : 0;
  int load_row = from + (first_step - load_head * per_head) * ROWS, use_row = load_row;
  auto load = [&](T *qt, T *dt, float *st) {
    const int head = kvh * p.group + load_head;
    qrows.load(head * p.q_sh, load_row, p.tq, qt, tid);
    drows.load(head * p.o_sh, load_row, p.tq, dt, tid);
    if (set == 0 && wave < 2) {
      // queries from tq on: zeros in q, dout and both statistics add nothing
      const Buffer s =
          buffer_of(p.stat + wave * n + ((int64_t)b * p.heads + head) * p.tq + load_row,
                    (uint32_t)min(p.tq - load_row, ROWS) * 4);
      copy_to_lds4(s, lane * 4, st + wave * 64);
    }
    load_row += ROWS;
    if (load_row >= p.tq) load_row = from, load_head++;
  };
  Reads<T, DP> rd;
  rd.open(lane);
  auto use = [&](const T *qt, const T *dt, const float *st) {
    rd.renew();
    const int row0 = use_row;
    use_row = use_row + ROWS >= p.tq ? from : use_row + ROWS;
    const int r = set;
    // unless the wave's first key is behind every query of these rows
    if (!p.causal || first_key + wave * 32 <= row0 + 32 * r + 31 + off) {
      f32x16 s, dp;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 16; i++) s[i] = 0.0f, dp[i] = 0.0f;
#pragma unroll
      for (int d = 0; d < DP / 16; d++) {
        s = Half<T>::mma(rd.rows(qt, 32 * r, d), kf[d], s);
        dp = Half<T>::mma(rd.rows(dt, 32 * r, d),
                          rd.rows(vt + wave * 32 * L::PITCH, 0, d), dp);
      }
      interleave<DP / 8, 6, 2>();
      __builtin_amdgcn_sched_barrier(0);
      const bool all = !p.causal || first_key + wave * 32 + 31 <= row0 + 32 * r + off;
#pragma unroll
      for (int bq = 0; bq < 4; bq++) {
        const f32x4 ls = *(const f32x4 *)(st + 32 * r + 8 * bq + 4 * h);
        const f32x4 dl = *(const f32x4 *)(st + 64 + 32 * r + 8 * bq + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int i = 4 * bq + j;
          float e = exp2_fast(fmaf(s[i], p.scale2, -ls[j]));
          if (!all) e = key <= row0 + 32 * r + 8 * bq + 4 * h + j + off ? e : 0.0f;
          dp[i] = e * fmaf(dp[i], Carried<T>::DOWN, -dl[j]);
          s[i] = e;
        }
      }
      if (Carried<T>::ENDS && again) {
#pragma unroll
        for (int i = 0; i < 16; i++) dp[i] *= unit;
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        const auto pf = narrow<T>(s, 8 * kk);
        const auto sf = narrow<T>(dp, 8 * kk);
#pragma unroll
        for (int d = 0; d < DP / 32; d++) {
          dv[d] = Half<T>::mma(rd.columns(dt, 32 * r + 16 * kk, 32 * d), pf, dv[d]);
          dk[d] = Half<T>::mma(rd.columns(qt, 32 * r + 16 * kk, 32 * d), sf, dk[d]);
        }
      }
      interleave<DP / 8, 4, 2>();
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Both sets do the same between two barriers.  The first goes first where
  // they meet, so one's products run beside the other's powers.
  if (set == 0) __builtin_amdgcn_s_setprio(1);
  if (steps > 0) {
    Rows<T, DP, COLS, THREADS> vrows;
    vrows.open((const T *)p.v + b * p.v_sb + kvh * p.v_sh, p.v_st, p.dim, tid);
    vrows.load(0, first_key, len, vt, tid);
    load(q0, d0, st0);
  }
  for (int i = 0; i < steps; i += 2) {
    tile_barrier();
    if (i + 1 < steps) load(q1, d1, st1);
    use(q0, d0, st0);
    tile_barrier();
    if (i + 2 < steps) load(q0, d0, st0);
    if (i + 1 < steps) use(q1, d1, st1);
  }
  if constexpr (Carried<T>::ENDS) {
    __shared__ int votes[2 * WAVES];
    const float used = unit;
    // columns from the sequence's length on hold what nobody reads
    if (lost_columns<2 * WAVES>(there ? dk[0][0] : 0.0f, unit, votes)) return true;
    if (again) {
#pragma unroll
      for (int d = 0; d < DP / 32; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) dk[d][i] *= 1.0f / used;
    }
  }
  // dk, then dv, from the second set to the first through the row buffers'
  // space; q0 .. d1 are one set's 4 waves x 32 keys x DP floats at DP = PITCH.
  auto slab = [&](int w) { return (float *)(w == 0 ? q0 : w == 1 ? q1 : w == 2 ? d0 : d1); };
  static_assert(32 * DP * 4 <= (int)sizeof(q0), "a wave's sums fit one buffer");
#pragma unroll
  for (int which = 0; which < 2; which++) {
    f32x16(&sum)[DP / 32] = which ? dv : dk;
    __syncthreads();
    if (set == 1) {
#pragma unroll
      for (int d = 0; d < DP / 32; d++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          f32x4 x;
#pragma unroll
          for (int j = 0; j < 4; j++) x[j] = sum[d][4 * q + j];
          *(f32x4 *)(slab(wave) + ((d * 4 + q) * 64 + lane) * 4) = x;
        }
    }
    __syncthreads();
    if (set == 0) {
#pragma unroll
      for (int d = 0; d < DP / 32; d++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const f32x4 x = *(const f32x4 *)(slab(wave) + ((d * 4 + q) * 64 + lane) * 4);
#pragma unroll
          for (int j = 0; j < 4; j++) sum[d][4 * q + j] += x[j];
        }
    }
  }
  if (set == 1 || key >= p.tk) return false;
  const int64_t row = ((int64_t)b * p.tk + key) * p.kv_heads + kvh;
  if (!there) {  // keys beyond the sequence's length have had no part
#pragma unroll
    for (int d = 0; d < DP / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) dk[d][i] = 0.0f, dv[d][i] = 0.0f;
  }
  if (p.parts > 1) {
    const int64_t rows = (int64_t)p.batch * p.tk * p.kv_heads;
    float *out = p.part + (2 * part * rows + row) * p.dim;
    store_sums<DP>(out, dk, p.dim, h), store_sums<DP>(out + rows * p.dim, dv, p.dim, h);
    return false;
  }
  store_columns<T, DP>((T *)p.dk + row * p.dim, dk, p.scale * Carried<T>::LEFT, p.dim, h);
  store_columns<T, DP>((T *)p.dv + row * p.dim, dv, 1.0f / P_UP, p.dim, h);
  return false;
}

template <class T, int DP, int WAVES>
__global__ __launch_bounds__(128 * WAVES, 2) void attention_dkv_kernel(AttnDims p) {
  blocks<T>(p, [](const AttnDims &a, int tid, int block, float &unit, bool again) {
    return dkv_block<T, DP, WAVES>(a, tid, block, unit, again);
  });
}

// The sum of the parts' [parts][stride] values, in order, times f, rounded once.
template <class T>
__global__ __launch_bounds__(256) void attention_parts_kernel(const float *part, int parts,
                                                              int64_t stride, int64_t n, float f,
                                                              void *out) {
  struct alignas(8) Four { T v[4]; };
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int i = 0; i < parts; i++) x += *(const f32x4 *)(part + i * stride + at);
  Four y;
#pragma unroll
  for (int j = 0; j < 4; j++) y.v[j] = (T)(x[j] * f);
  *(Four *)((T *)out + at) = y;
}

// --------------------------------------------------------------------- host

static AttnDims attention_dims(const clear_attention_args &a) {
  require(a.type == CLEAR_BF16 || a.type == CLEAR_FP16, "attention: type is bf16 or fp16");
  require(a.batch >= 0 && a.q_tokens >= 0 && a.kv_tokens >= 0, "attention: negative size");
  require(a.kv_heads >= 1 && a.heads >= 1 && a.heads % a.kv_heads == 0,
          "attention: the query heads are a multiple of the key heads");
  require(a.dim >= 8 && a.dim <= 128 && a.dim % 8 == 0,
          "attention: the head is a multiple of 8, at most 128");
  // FLT_MIN: below it the scale has fewer bits in fp32, or is 0
  require(a.scale >= 1.1754943508222875e-38 && a.scale < 1e30,
          "attention: the scale is positive and finite in fp32");
  const int64_t most = (int64_t)1 << 30;
  require(a.batch <= most && a.q_tokens <= most && a.kv_tokens <= most && a.heads <= 1 << 16 &&
              a.batch * a.heads <= most && a.q_tokens + a.kv_tokens <= 2 * most - 256,
          "attention: too large");
  AttnDims p = {};
  p.q = a.q, p.k = a.k, p.v = a.v, p.out = a.out, p.lse = (float *)a.lse;
  p.kv_lens = (const int *)a.kv_lens, p.q_start = (const int *)a.q_start;
  p.dout = a.dout, p.dq = a.dq, p.dk = a.dk, p.dv = a.dv;
  p.q_sb = a.q_sb, p.q_st = a.q_st, p.q_sh = a.q_sh;
  p.k_sb = a.k_sb, p.k_st = a.k_st, p.k_sh = a.k_sh;
  p.v_sb = a.v_sb, p.v_st = a.v_st, p.v_sh = a.v_sh;
  p.o_sb = a.o_sb, p.o_st = a.o_st, p.o_sh = a.o_sh;
  p.batch = (int)a.batch, p.tq = (int)a.q_tokens, p.tk = (int)a.kv_tokens;
  p.heads = (int)a.heads, p.kv_heads = (int)a.kv_heads, p.group = (int)(a.heads / a.kv_heads);
  p.dim = (int)a.dim, p.causal = a.causal != 0;
  p.scale = (float)a.scale, p.scale2 = (float)(a.scale * 1.4426950408889634);
  p.splits = 1, p.split_keys = p.tk > 0 ? p.tk : 1, p.parts = p.dq_parts = 1;
  return p;
}

// Offsets inside a tile have 32 bits, and a tile's end is found by its row
// stride: rows do not overlap and are at most 2^23 elements apart.
static void check_rows(const void *x, int64_t sb, int64_t st, int64_t sh, int64_t rows, int64_t dim) {
  const bool used = rows > 0;
  require(!used || x, "attention: null tensor");
  require(!used || (aligned(x, 16) && sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0),
          "attention: rows start at multiples of 16 bytes");
  require(!used || (st >= dim && st <= 1 << 23), "attention: stride of the tokens");
}

// Which kernel: each takes the keys past 32 packed columns, or past 128 queries
// of one head, in about the same time, so the fewer passes win; one pass is
// always packed, since its keys are shared out over the waves too.  8 sequences,
// 16000 keys, 8 key heads of 128, packed and by heads: 8 queries of 32 heads
// (1 and 4 passes) 110 and 300 us, 16 (2 and 4) 207 and 297, 32 (4 and 4) 386
// and 300, 33 queries of 8 heads (2 and 1) 196 and 103.
static bool few_queries(const AttnDims &p) {
  const int64_t packed = ceil_div((int64_t)p.tq * p.group, 32);
  return packed <= 1 || packed < p.group * ceil_div(p.tq, 128);
}

static int64_t query_blocks(const AttnDims &p) {
  return (int64_t)p.batch * p.heads * ceil_div(p.tq, 128);
}
static int64_t key_blocks(const AttnDims &p, int keys) {
  return (int64_t)p.batch * p.kv_heads * ceil_div(p.tk, keys);
}

// Into how many blocks the sum behind a tile is split: where the tiles are
// fewer than the CUs and the sum is long, as many as give two a CU, of four
// steps or more each.  The join costs a launch and the fp32 sums' way through
// memory.  Backward pass of 1500 tokens with 32 and 8 heads of 128: 213 us
// whole, 123 in parts; of 3 x 700 tokens with 8 heads (11 steps behind 144
// tiles): 41 whole, 46 in parts.  Forward pass of 3000 tokens with one head: 56
// and 22 us; of 1003 tokens with 12 heads (16 steps): 16 and 21.
static int parts_of(int64_t blocks, int64_t steps, int64_t least) {
  if (blocks == 0 || blocks >= 256 || steps < least) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(512 / blocks, steps / 4));
}
static void plan_parts(AttnDims &p) {
  const int64_t blocks = key_blocks(p, 128);
  p.parts = parts_of(blocks, p.group * ceil_div(p.tq, 64), blocks <= 64 ? 8 : 16);
  p.dq_parts = parts_of(query_blocks(p), ceil_div(p.tk, 64), 16);
}

// Keys a block takes where there are few queries: enough blocks for the
// machine, none below 256 keys (the join costs a launch and a round trip).
static void plan_splits(AttnDims &p) {
  if (!few_queries(p)) {
    const int64_t tiles = ceil_div(p.tk, FWD_KEYS);
    const int64_t share = ceil_div(tiles, parts_of(query_blocks(p), tiles, 24));
    p.split_keys = (int)std::max<int64_t>(share * FWD_KEYS, FWD_KEYS);
    p.splits = (int)std::max<int64_t>(ceil_div(p.tk, p.split_keys), 1);
    return;
  }
  const int64_t blocks = (int64_t)p.batch * p.kv_heads * ceil_div((int64_t)p.tq * p.group, 32);
  if (blocks == 0) return;
  const int64_t want = ceil_div(1024, blocks);
  int64_t keys = ceil_div(ceil_div(p.tk, want), 128) * 128;
  keys = keys < 256 ? 256 : keys;
  p.splits = (int)(p.tk > 0 ? ceil_div(p.tk, keys) : 1);
  p.split_keys = (int)keys;
}

static int64_t forward_bytes(const AttnDims &p) {
  if (p.splits == 1) return 0;
  const int64_t rows = (int64_t)p.batch * p.tq * p.heads;
  return p.splits * rows * (p.dim + 2) * (int64_t)sizeof(float);
}

static int64_t stat_bytes(const AttnDims &p) {
  return ceil_div(2 * (int64_t)p.batch * p.heads * p.tq * (int64_t)sizeof(float), 16) * 16;
}
static int64_t backward_bytes(const AttnDims &p) {
  const int64_t sums = (int64_t)p.batch * p.tk * p.kv_heads * p.dim * (int64_t)sizeof(float);
  const int64_t dq = (int64_t)p.batch * p.tq * p.heads * p.dim * (int64_t)sizeof(float);
  return stat_bytes(p) + (p.parts > 1 ? 2 * p.parts * sums : 0) +
         (p.dq_parts > 1 ? p.dq_parts * dq : 0);
}

static unsigned blocks_of(int64_t n) {
  require(n < (int64_t)1 << 31, "attention: too many blocks");
  return (unsigned)n;
}

template <class T, int DP> static void forward_go(const AttnDims &p, hipStream_t st) {
  const int64_t pairs = (int64_t)p.batch * p.kv_heads;
  auto join = [&] {
    if (p.splits == 1) return;
    attention_join_kernel<T><<<blocks_of((int64_t)p.batch * p.tq * p.heads), 64, 0, st>>>(p);
    launched();
  };
  if (few_queries(p)) {
    const dim3 grid(blocks_of(pairs * p.splits), (unsigned)ceil_div((int64_t)p.tq * p.group, 32));
    attention_few_kernel<T, DP><<<grid, 64 * FEW_WAVES, 0, st>>>(p);
    launched();
    join();
    return;
  }
  const unsigned n = blocks_of(query_blocks(p) * p.splits);
  attention_forward_kernel<T, DP><<<n, 64 * FWD_WAVES, 0, st>>>(p);
  launched();
  join();
}

template <class T, int DP> static void backward_go(const AttnDims &p, hipStream_t st) {
  auto add = [&](const float *part, int parts, int64_t stride, int64_t n, float f, void *out) {
    attention_parts_kernel<T><<<blocks_of(ceil_div(n / 4, 256)), 256, 0, st>>>(part, parts, stride,
                                                                              n, f, out);
    launched();
  };
  if (p.tq > 0) {
    attention_dq_kernel<T, DP>
        <<<blocks_of(query_blocks(p) * p.dq_parts), 64 * BWD_WAVES, 0, st>>>(p);
    launched();
    const int64_t m = (int64_t)p.batch * p.tq * p.heads * p.dim;
    if (p.dq_parts > 1) add(p.dq_part, p.dq_parts, m, m, p.scale * Carried<T>::LEFT, p.dq);
  }
  if (p.tk > 0) {
    // Narrow heads leave room for several blocks a CU: halves of a tile even out
    // what the CUs get (5 x 1003 tokens of 12 heads of 64, uneven lengths: the
    // whole backward pass 80 -> 66 us).
    const bool halves = DP <= 64 && p.parts == 1 && key_blocks(p, 128) < 1024;
    if (!halves)
      attention_dkv_kernel<T, DP, 4><<<blocks_of(key_blocks(p, 128) * p.parts), 512, 0, st>>>(p);
    else if constexpr (DP <= 64)
      attention_dkv_kernel<T, DP, 2><<<blocks_of(key_blocks(p, 64)), 256, 0, st>>>(p);
    launched();
    if (p.parts > 1) {
      const int64_t m = (int64_t)p.batch * p.tk * p.kv_heads * p.dim;
      add(p.part, p.parts, 2 * m, m, p.scale * Carried<T>::LEFT, p.dk);
      add(p.part + m, p.parts, 2 * m, m, 1.0f / P_UP, p.dv);
    }
  }
}

template <bool BACKWARD, class T> static void dispatch(const AttnDims &p, hipStream_t st) {
  // the head padded to the next size a kernel is built for
  if (p.dim <= 64) BACKWARD ? backward_go<T, 64>(p, st) : forward_go<T, 64>(p, st);
  else if (p.dim <= 96) BACKWARD ? backward_go<T, 96>(p, st) : forward_go<T, 96>(p, st);
  else BACKWARD ? backward_go<T, 128>(p, st) : forward_go<T, 128>(p, st);
}

}  // namespace clr

using namespace clr;

extern "C" int clear_attention_workspace(const clear_attention_args *args, int64_t backward,
                                         int64_t *bytes) {
  return guarded([&] {
    require(args && bytes, "attention: no arguments");
    AttnDims p = attention_dims(*args);
    if (!backward) plan_splits(p);
    if (backward) plan_parts(p);
    *bytes = backward ? backward_bytes(p) : forward_bytes(p);
  });
}

extern "C" int clear_attention_forward(const clear_attention_args *args, void *stream) {
  return guarded([&] {
    require(args, "attention: no arguments");
    const clear_attention_args &a = *args;
    AttnDims p = attention_dims(a);
    if (p.batch == 0 || p.tq == 0) return;
    check_rows(a.q, a.q_sb, a.q_st, a.q_sh, p.tq, p.dim);
    check_rows(a.k, a.k_sb, a.k_st, a.k_sh, p.tk, p.dim);
    check_rows(a.v, a.v_sb, a.v_st, a.v_sh, p.tk, p.dim);
    require(a.out && a.lse && aligned(a.out, 16), "attention: null or misaligned output");
    plan_splits(p);
    const int64_t need = forward_bytes(p);
    require(need <= a.workspace_bytes && (need == 0 || (a.workspace && aligned(a.workspace, 16))),
            "attention: the workspace is too small");
    p.part = (float *)a.workspace;
    hipStream_t st = (hipStream_t)stream;
    a.type == CLEAR_BF16 ? dispatch<false, __bf16>(p, st) : dispatch<false, _Float16>(p, st);
  });
}

extern "C" int clear_attention_backward(const clear_attention_args *args, void *stream) {
  return guarded([&] {
    require(args, "attention: no arguments");
    const clear_attention_args &a = *args;
    AttnDims p = attention_dims(a);
    if (p.batch == 0 || (p.tq == 0 && p.tk == 0)) return;
    check_rows(a.q, a.q_sb, a.q_st, a.q_sh, p.tq, p.dim);
    check_rows(a.dout, a.o_sb, a.o_st, a.o_sh, p.tq, p.dim);
    check_rows(a.k, a.k_sb, a.k_st, a.k_sh, p.tk, p.dim);
    check_rows(a.v, a.v_sb, a.v_st, a.v_sh, p.tk, p.dim);
    require(p.tq == 0 || (a.out && a.lse && a.dq && aligned(a.out, 16) && aligned(a.dq, 16)),
            "attention: null or misaligned tensor");
    require(p.tk == 0 || (a.dk && a.dv && aligned(a.dk, 16) && aligned(a.dv, 16)),
            "attention: null or misaligned gradient");
    plan_parts(p);
    const int64_t need = backward_bytes(p);
    require(need <= a.workspace_bytes && (need == 0 || (a.workspace && aligned(a.workspace, 16))),
            "attention: the workspace is too small");
    p.stat = (float *)a.workspace;
    p.part = (float *)((char *)a.workspace + stat_bytes(p));
    p.dq_part = p.part;
    if (p.parts > 1) p.dq_part += 2 * p.parts * (int64_t)p.batch * p.tk * p.kv_heads * p.dim;
    hipStream_t st = (hipStream_t)stream;
    a.type == CLEAR_BF16 ? dispatch<true, __bf16>(p, st) : dispatch<true, _Float16>(p, st);
  });
}
