// Attention of a few query rows over the paged 8-bit cache (tokens one at a
// time, drafts being checked, many query heads on one kv head).
//
// Mathematics.  With S^T = K Q^T (keys x rows) and O^T = V^T P^T, keys are the
// long dimension of both products' A operands (mma.sync m16n8k16, f16 with
// f32 sums), and the query rows of a kv head -- new tokens x query heads that
// share it -- are the narrow N, 8 to a step, so one token of 8 shared heads
// wastes nothing.  e4m3 codes are exact in f16; a page's scales 2^e never
// touch the codes: K's goes into the factor that takes scores to log2 units,
// V's into the exponent of p (moving O's unit when it strays more than 2^6
// from it).  A query row is scaled by a power of two so that its largest
// element lies in [1, 2) before it becomes f16: a bf16 row is exact down to
// 2^-14 of that element and rounded by at most 2^-25 of it below.  Scores,
// maxima, sums and O are f32; p is rounded to f16 (2^-12 relative), the only
// rounding of width before the output's.
//
// No operand goes through shared memory.  The order of a contraction's terms
// is free, so each lane's 16 consecutive bytes of a key serve as its shares
// of four k-steps, and of a value row as the rows 2i, 2i+1 of D / 16 m-tiles:
// every load is 8 or 16 bytes and a warp's cover whole 64-128-byte pieces of rows.
//
// Bound by memory: codes are read once per kv head.  The visible 64-key
// chunks of all (sequence, head, row block) lie on one line that the grid
// cuts into equal parts, so uneven lengths balance and one long sequence
// fills the GPU.  A part that covers a segment only partly leaves (m, l, O)
// in the workspace; the last of the segment's parts to arrive joins them in
// the parts' order, so results do not depend on which came last.
#include <cuda_bf16.h>

#include "kv8.cuh"
#include "kv8_attend.cuh"

namespace kv8 {
namespace {

constexpr int THREADS = 128, WARPS = 4;
constexpr float LAZY = 8.0f;  // log2 units that scores may pass the reference before O moves
constexpr int UNIT_LAZY = 6;  // the same for V's exponent: p stays below 2^14 in f16
constexpr float NONE = -1e30f;

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// The geometry of one (sequence, head, row block) and of its chunk line.
struct Segment {
  int b, head, start, n, len;  // n new tokens, rows from `start`; len keys
  int rows, row0;              // rows of the kv head, first row of this block
  Span span;
};

// Codes and exponents of 16 keys, as a lane holds them: K rows g and g + 8
// (16 bytes at 64 j + 16 q), V rows 2q, 2q+1, 2q+8, 2q+9 (D / 8 bytes at
// g D / 8), with g = lane / 4, q = lane % 4.
template <int D>
struct Tile {
  uint32_t k[2][D / 16], v[4][D / 32];
  int ek, ev, key0;
  bool dead;  // the page number was bad: every key hidden
};

template <int D>
__device__ __forceinline__ void load_tile(Tile<D> &t, const AttendParams &p, const Segment &g,
                                          int key0, int page, int lane) {
  t.key0 = key0;
  t.dead = page < 0 || page >= p.s.pages;
  if (t.dead) {
    report(p.s.status, STATUS_PAGE);
    page = 0;
  }
  const int64_t unit = int64_t(page) * 2 * p.s.kv_heads + g.head;
  t.ek = p.exps[unit];
  t.ev = p.exps[unit + p.s.kv_heads];
  const int slot = key0 & ((1 << p.s.page_shift) - 1);
  const uint8_t *k = p.codes + ((unit << p.s.page_shift) + slot) * D;
  const uint8_t *v = k + ((int64_t(p.s.kv_heads) << p.s.page_shift) * D);
  const int gr = lane >> 2, q = lane & 3;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(k + (gr + 8 * i) * D + 64 * j + 16 * q));
      t.k[i][4 * j] = w.x, t.k[i][4 * j + 1] = w.y, t.k[i][4 * j + 2] = w.z, t.k[i][4 * j + 3] = w.w;
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint8_t *at = v + (2 * q + (i & 1) + 8 * (i >> 1)) * D + gr * (D / 8);
    if constexpr (D == 64) {
      const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(at));
      t.v[i][0] = w.x, t.v[i][1] = w.y;
    } else {
      const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(at));
      t.v[i][0] = w.x, t.v[i][1] = w.y, t.v[i][2] = w.z, t.v[i][3] = w.w;
    }
  }
}

// What a warp carries over its tiles, for rows 2q, 2q+1 of each 8-row block.
template <int D, int NT>
struct State {
  float o[D / 16][NT][4];
  float m[NT][2], l[NT][2];
  float mult[NT][2];  // scale * log2(e) * the row's power of two
  int pos[NT][2];     // position of the row's token, -1: no such row
  int unit;           // O is in units of 2^unit
};

template <int D, int NT>
__device__ __forceinline__ void scale_o(State<D, NT> &st, const float (&f)[NT][2]) {
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      st.o[i][t][0] *= f[t][0], st.o[i][t][2] *= f[t][0];
      st.o[i][t][1] *= f[t][1], st.o[i][t][3] *= f[t][1];
    }
}

template <int D, int NT, typename Q>
__device__ __forceinline__ void tile_step(State<D, NT> &st, Tile<D> &t, const AttendParams &p,
                                          const Segment &g, const Q &query, int lane) {
  const int gr = lane >> 2, q = lane & 3;
  // ---- S^T = K Q^T ----
  float s[NT][4] = {};
#pragma unroll
  for (int w = 0; w < D / 16; ++w) {
    const uint32_t a[4] = {e4m3x2_f16x2(t.k[0][w]), e4m3x2_f16x2(t.k[1][w]),
                           e4m3x2_f16x2(t.k[0][w] >> 16), e4m3x2_f16x2(t.k[1][w] >> 16)};
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const uint2 b = query(w, i);
      mma(s[i], a, b.x, b.y);
    }
  }
  const float mk = pow2(t.ek);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[i][c] *= st.mult[i][c & 1] * mk;
  // ---- hidden keys: only in tiles that some row does not see whole ----
  const bool masked = t.dead || !g.span.all_see(t.key0, t.key0 + 15);
  uint32_t nan_at[4] = {};  // bit d: value d of the lane's V row i is NaN
  bool any_nan = false;
  if (masked) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (t.dead || !g.span.sees(st.pos[i][c & 1], t.key0 + gr + 8 * (c >> 1))) s[i][c] = -INFINITY;
    // A hidden key has p = 0, but 0 * NaN is NaN: values no row sees become
    // zero, and a NaN that only some rows see is taken out here and put into
    // those rows' sums below.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool seen = !t.dead && g.span.any_sees(t.key0 + 2 * q + (i & 1) + 8 * (i >> 1));
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        if (!seen) t.v[i][w] = 0;
        const uint32_t bad = nan_bytes(t.v[i][w]);
        if (bad != 0) {
          t.v[i][w] &= ~((bad >> 7) * 0xffu);
#pragma unroll
          for (int j = 0; j < 4; ++j) nan_at[i] |= ((bad >> (8 * j + 7)) & 1u) << (4 * w + j);
        }
      }
    }
    any_nan = __any_sync(0xffffffffu, (nan_at[0] | nan_at[1] | nan_at[2] | nan_at[3]) != 0);
  }
  // ---- running maxima, kept while no score passes them by more than LAZY ----
  bool grow = false;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) grow |= s[i][c] > st.m[i][c & 1] + LAZY;
  const bool move = t.ev - st.unit > UNIT_LAZY || st.unit - t.ev > UNIT_LAZY;
  if (__any_sync(0xffffffffu, grow) || move) {
    float f[NT][2];
    const float unit = move ? pow2(st.unit - t.ev) : 1.0f;
    if (move) st.unit = t.ev;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = fmaxf(s[i][c], s[i][c + 2]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        top = fmaxf(top, st.m[i][c]);
        f[i][c] = exp2_fast(st.m[i][c] - top);
        st.m[i][c] = top;
        st.l[i][c] *= f[i][c];
        f[i][c] *= unit;
      }
    scale_o(st, f);
  }
  // ---- p = 2^(s - m) in units of 2^(unit - ev); P^T by 8 x 8 transposes ----
  const float dev = float(t.ev - st.unit), undo = pow2(st.unit - t.ev);
  uint32_t b[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    float e[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) e[c] = exp2_fast(s[i][c] - (st.m[i][c & 1] - dev));
    st.l[i][0] = fmaf(e[0] + e[2], undo, st.l[i][0]);
    st.l[i][1] = fmaf(e[1] + e[3], undo, st.l[i][1]);
    const __half2 lo = __floats2half2_rn(e[0], e[1]), hi = __floats2half2_rn(e[2], e[3]);
    b[i][0] = transpose8x8(*reinterpret_cast<const uint32_t *>(&lo));
    b[i][1] = transpose8x8(*reinterpret_cast<const uint32_t *>(&hi));
  }
  // ---- O^T += V^T P^T ----
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const uint32_t sel = i & 1 ? 0x7362 : 0x5140;  // (key 2q, key 2q+1) of two neighbouring d
    const uint32_t x = __byte_perm(t.v[0][i / 2], t.v[1][i / 2], sel);
    const uint32_t y = __byte_perm(t.v[2][i / 2], t.v[3][i / 2], sel);
    const uint32_t a[4] = {e4m3x2_f16x2(x), e4m3x2_f16x2(x >> 16), e4m3x2_f16x2(y), e4m3x2_f16x2(y >> 16)};
#pragma unroll
    for (int r = 0; r < NT; ++r) mma(st.o[i][r], a, b[r][0], b[r][1]);
  }
  if (any_nan) {
    uint32_t rows[NT][2] = {};  // bit d: the row sees a NaN in value d
    for (int from = 0; from < 4; ++from)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t bits = __shfl_sync(0xffffffffu, nan_at[i], (lane & ~3) | from);
        const int key = t.key0 + 2 * from + (i & 1) + 8 * (i >> 1);
#pragma unroll
        for (int r = 0; r < NT; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (g.span.sees(st.pos[r][c], key)) rows[r][c] |= bits;
      }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (rows[r][c & 1] >> (2 * i + (c >> 1)) & 1u) st.o[i][r][c] = NAN;
  }
}

// One row's share of a lane: Q[64 j + 16 q .. + 15] for each j, scaled into
// f16; returns the row's exponent (row = f16 row * 2^exponent).
template <int D, typename T>
__device__ __forceinline__ int query_row(uint32_t (&f)[D / 8], const T *row, int q) {
  float x[D / 4];
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (row != nullptr) w = *reinterpret_cast<const uint4 *>(row + 64 * j + 16 * q + 8 * h);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) unpack2<T>(u[i], x[16 * j + 8 * h + 2 * i], x[16 * j + 8 * h + 2 * i + 1]);
    }
#pragma unroll
  for (int i = 0; i < D / 4; ++i) amax = fabsf(x[i]) < INFINITY ? fmaxf(amax, fabsf(x[i])) : amax;
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const int e = row_exponent(amax);
  const float by = pow2(-e);
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const __half2 h = __floats2half2_rn(x[2 * i] * by, x[2 * i + 1] * by);
    f[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  return e;
}

// Shared memory: first the joined rows of the four warps, over the staged queries.
template <int D, int NT>
constexpr int SMEM_JOIN = WARPS * 8 * NT * (D + 8) * 4;
static_assert(SMEM_JOIN<64, 1> >= 1 * 32 * 64 / 8 * 4, "the staged queries fit under the join");

template <int D, int NT, typename T>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 4 : NT == 2 ? 3 : 2)
rows_kernel(const AttendParams p) {
  constexpr int ROWS = 8 * NT, LD = D + 8;
  extern __shared__ __align__(16) uint8_t dyn[];
  float *const join = reinterpret_cast<float *>(dyn);
  __shared__ float sm_m[WARPS][ROWS], sm_l[WARPS][ROWS], weight[WARPS][ROWS], row_l[ROWS], row_m[ROWS];
  __shared__ int sm_unit[WARPS], row_exp[ROWS];
  __shared__ unsigned ticket;
  __shared__ unsigned scan[WARPS];
  uint32_t *const line = reinterpret_cast<uint32_t *>(dyn + SMEM_JOIN<D, NT>);  // [seqs + 1]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gr = lane >> 2, q = lane & 3;
  const Seqs &s = p.s;

  // ---- the line of chunks: where each sequence starts ----
  {
    const int per = (s.seqs + THREADS - 1) / THREADS, b0 = min(tid * per, s.seqs), b1 = min(b0 + per, s.seqs);
    unsigned sum = 0;
    for (int b = b0; b < b1; ++b) {
      int start, n, len;
      lengths(s, b, start, n, len);
      if (n * p.group > p.row_limit) n = 0;
      unsigned c = 0;
      if (n > 0) c = unsigned(Span(p, len - n, len - 1).chunks) * ((n * p.group + ROWS - 1) / ROWS) * s.kv_heads;
      line[b] = c;
      sum += c;
    }
    unsigned at = sum;
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, at, d);
      if (lane >= d) at += u;
    }
    if (lane == 31) scan[warp] = at;
    __syncthreads();
    for (int w = 0; w < warp; ++w) at += scan[w];
    at -= sum;
    for (int b = b0; b < b1; ++b) {
      const unsigned c = line[b];
      line[b] = at;
      at += c;
    }
    if (tid == THREADS - 1) line[s.seqs] = at;
    __syncthreads();
  }
  const uint64_t total = line[s.seqs];
  const uint64_t N = gridDim.x < total ? gridDim.x : total;  // every part has a chunk
  if (blockIdx.x >= N) return;
  const unsigned from = unsigned(blockIdx.x * total / N), to = unsigned((blockIdx.x + 1) * total / N);

  for (unsigned pos = from; pos < to;) {
    // ---- the segment at `pos` ----
    Segment g;
    {
      int lo = 0, hi = s.seqs - 1;  // last b with line[b] <= pos (empty ones come before it)
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (line[mid] <= pos) lo = mid; else hi = mid - 1;
      }
      g.b = lo;
    }
    lengths(s, g.b, g.start, g.n, g.len);
    g.span = Span(p, g.len - g.n, g.len - 1);
    g.rows = g.n * p.group;
    const int chunks = g.span.chunks;
    const unsigned rel = pos - line[g.b], hr = rel / chunks;
    const int c0 = rel - hr * chunks, c1 = int(min(unsigned(chunks), c0 + (to - pos)));
    g.head = hr % s.kv_heads;
    g.row0 = hr / s.kv_heads * ROWS;
    const unsigned seg0 = pos - c0;
    pos += c1 - c0;
    // rows of this block see only part of the sequence's keys
    const int t0 = g.row0 / p.group, t1 = min(g.row0 + ROWS, g.rows) - 1;
    g.span.first = g.len - g.n + t0;
    g.span.last = g.len - g.n + t1 / p.group;

    // ---- queries ----
    State<D, NT> st;
    uint32_t own[NT == 1 ? D / 8 : 1];
    uint32_t *const staged = reinterpret_cast<uint32_t *>(dyn);
    const auto row_at = [&](int r, int64_t ts, int64_t hs) {
      const int i = (g.row0 + r) / p.group, h = g.head * p.group + (g.row0 + r) - i * p.group;
      return (g.start + i) * ts + h * hs;
    };
    if constexpr (NT == 1) {
      const T *row = gr + g.row0 < g.rows ? static_cast<const T *>(p.q) + row_at(gr, p.q_ts, p.q_hs) : nullptr;
      const int e = query_row<D>(own, row, q);
      st.mult[0][0] = p.scale_log2 * pow2(__shfl_sync(0xffffffffu, e, 8 * q));
      st.mult[0][1] = p.scale_log2 * pow2(__shfl_sync(0xffffffffu, e, 8 * q + 4));
    } else {
      __syncthreads();  // the last segment's join is read
      for (int i = warp; i < NT; i += WARPS) {
        const int r = 8 * i + gr;
        uint32_t f[D / 8];
        const T *row = r + g.row0 < g.rows ? static_cast<const T *>(p.q) + row_at(r, p.q_ts, p.q_hs) : nullptr;
        const int e = query_row<D>(f, row, q);
        if (q == 0) row_exp[r] = e;
#pragma unroll
        for (int w = 0; w < D / 16; ++w)
          *reinterpret_cast<uint2 *>(&staged[((w * NT + i) * 32 + lane) * 2]) = make_uint2(f[2 * w], f[2 * w + 1]);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) st.mult[i][c] = p.scale_log2 * pow2(row_exp[8 * i + 2 * q + c]);
    }
    const auto query = [&](int w, int i) {
      if constexpr (NT == 1)
        return make_uint2(own[2 * w], own[2 * w + 1]);
      else
        return *reinterpret_cast<const uint2 *>(&staged[((w * NT + i) * 32 + lane) * 2]);
    };
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = g.row0 + 8 * i + 2 * q + c;
        st.pos[i][c] = r < g.rows ? g.len - g.n + r / p.group : -1;
        st.m[i][c] = NONE;
        st.l[i][c] = 0.0f;
      }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) st.o[i][t][c] = 0.0f;
    st.unit = 0;

    // ---- this warp's quarter of the part, 16 keys a tile, one tile ahead ----
    const int tiles = c1 - c0, first_tile = 4 * c0 + warp * tiles;
    const int *row = s.table + int64_t(g.b) * s.width;
    const auto key_of = [&](int i) { return g.span.key0((first_tile + i) >> 2) + 16 * ((first_tile + i) & 3); };
    const auto page_of = [&](int i) { return i < tiles ? row[key_of(i) >> s.page_shift] : 0; };
    Tile<D> a, b;
    int page = page_of(1);
    load_tile(a, p, g, key_of(0), page_of(0), lane);
    st.unit = a.ev;
    for (int i = 0; i < tiles; i += 2) {
      if (i + 1 < tiles) load_tile(b, p, g, key_of(i + 1), page, lane);
      page = page_of(i + 2);
      if (g.span.wanted(a.key0, a.key0 + 15)) tile_step(st, a, p, g, query, lane);
      if (i + 1 < tiles) {
        if (i + 2 < tiles) load_tile(a, p, g, key_of(i + 2), page, lane);
        page = page_of(i + 3);
        if (g.span.wanted(b.key0, b.key0 + 15)) tile_step(st, b, p, g, query, lane);
      }
    }

    // ---- join the warps ----
    __syncthreads();  // staged queries and the last join are read
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float l = st.l[i][c];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int r = 8 * i + 2 * q + c;
        if (gr == 0) sm_m[warp][r] = st.m[i][c], sm_l[warp][r] = l;
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
          *reinterpret_cast<float2 *>(&join[(warp * ROWS + r) * LD + gr * (D / 8) + 2 * j]) =
              make_float2(st.o[j][i][c], st.o[j][i][c + 2]);
      }
    if (lane == 0) sm_unit[warp] = st.unit;
    __syncthreads();
    if (tid < ROWS) {
      float m = NONE, l = 0.0f;
      for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sm_m[w][tid]);
      for (int w = 0; w < WARPS; ++w) {
        const float f = exp2_fast(sm_m[w][tid] - m);
        l += f * sm_l[w][tid];
        weight[w][tid] = f * pow2(sm_unit[w]);
      }
      row_m[tid] = m;
      row_l[tid] = l;
    }
    __syncthreads();
    const bool whole = c1 - c0 == chunks;
    const int rows = min(ROWS, g.rows - g.row0);
    const auto store = [&](int r, int d, const float (&x)[8], float l) {
      const float by = l == 0.0f ? 0.0f : 1.0f / l;
      uint4 w;
      w.x = pack2<T>(x[0] * by, x[1] * by);
      w.y = pack2<T>(x[2] * by, x[3] * by);
      w.z = pack2<T>(x[4] * by, x[5] * by);
      w.w = pack2<T>(x[6] * by, x[7] * by);
      *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + row_at(r, p.o_ts, p.o_hs) + d) = w;
    };
    // partial results: two slots a CTA (a segment it ends, one it begins)
    float *const slot = p.partial + (int64_t(blockIdx.x) * 2 + (c0 == 0)) * ROWS * (D + 2);
    for (int i = tid; i < rows * (D / 8); i += THREADS) {
      const int r = i / (D / 8), d = i % (D / 8) * 8;
      float x[8] = {};
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = weight[w][r];
        const float4 u = *reinterpret_cast<const float4 *>(&join[(w * ROWS + r) * LD + d]);
        const float4 v = *reinterpret_cast<const float4 *>(&join[(w * ROWS + r) * LD + d + 4]);
        x[0] += f * u.x, x[1] += f * u.y, x[2] += f * u.z, x[3] += f * u.w;
        x[4] += f * v.x, x[5] += f * v.y, x[6] += f * v.z, x[7] += f * v.w;
      }
      if (whole) {
        store(r, d, x, row_l[r]);
      } else {
        __stcg(reinterpret_cast<float4 *>(slot + r * D + d), make_float4(x[0], x[1], x[2], x[3]));
        __stcg(reinterpret_cast<float4 *>(slot + r * D + d + 4), make_float4(x[4], x[5], x[6], x[7]));
      }
    }
    if (whole) continue;
    if (tid < ROWS) {
      __stcg(slot + ROWS * D + tid, row_m[tid]);
      __stcg(slot + ROWS * D + ROWS + tid, row_l[tid]);
    }
    // ---- the last part of the segment to arrive joins all of them ----
    const unsigned part0 = unsigned(((uint64_t(seg0) + 1) * N - 1) / total);
    const unsigned part1 = unsigned(((uint64_t(seg0) + chunks) * N - 1) / total);
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      ticket = atomicAdd(p.counters + part0, 1u);
      if (ticket == part1 - part0) p.counters[part0] = 0;
      __threadfence();
    }
    __syncthreads();
    if (ticket != part1 - part0) continue;
    const auto part_slot = [&](unsigned c) {
      return p.partial + (int64_t(c) * 2 + (c == part0)) * ROWS * (D + 2);
    };
    for (int i = tid; i < rows * (D / 8); i += THREADS) {
      const int r = i / (D / 8), d = i % (D / 8) * 8;
      float m = NONE, l = 0.0f, x[8] = {};
      for (unsigned c = part0; c <= part1; ++c) m = fmaxf(m, __ldcg(part_slot(c) + ROWS * D + r));
      for (unsigned c = part0; c <= part1; ++c) {
        const float *at = part_slot(c);
        const float f = exp2_fast(__ldcg(at + ROWS * D + r) - m);
        l += f * __ldcg(at + ROWS * D + ROWS + r);
        const float4 u = __ldcg(reinterpret_cast<const float4 *>(at + r * D + d));
        const float4 v = __ldcg(reinterpret_cast<const float4 *>(at + r * D + d + 4));
        x[0] += f * u.x, x[1] += f * u.y, x[2] += f * u.z, x[3] += f * u.w;
        x[4] += f * v.x, x[5] += f * v.y, x[6] += f * v.z, x[7] += f * v.w;
      }
      store(r, d, x, l);
    }
  }
}

template <int D, int NT, typename T>
cudaError_t launch(const AttendParams &p, int grid, int device, cudaStream_t stream) {
  const int smem = SMEM_JOIN<D, NT> + (p.s.seqs + 1) * 4;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        rows_kernel<D, NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
        SMEM_JOIN<D, NT> + (EMMY_KV8_MAX_SEQS + 1) * 4);
    if (e != cudaSuccess) return e;
  }
  rows_kernel<D, NT, T><<<grid, THREADS, smem, stream>>>(p);
  return cudaGetLastError();
}

template <int D, typename T>
cudaError_t launch_nt(const AttendParams &p, int nt, int grid, int device, cudaStream_t stream) {
  switch (nt) {
    case 1: return launch<D, 1, T>(p, grid, device, stream);
    case 2: return launch<D, 2, T>(p, grid, device, stream);
    default: return launch<D, 4, T>(p, grid, device, stream);
  }
}

}  // namespace

// 8-row blocks a CTA takes together, for the rows of the largest sequence.
int rows_blocks(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

// CTAs that fill the GPU, as the launch bounds allow them.
int rows_grid(int nt, int device) { return sm_count(device) * (nt == 1 ? 4 : nt == 2 ? 3 : 2); }

uint64_t rows_partial_bytes(int nt, int head_dim, int device) {
  return uint64_t(rows_grid(nt, device)) * 2 * 8 * nt * (head_dim + 2) * 4;
}

cudaError_t rows_attend(const AttendParams &p, int nt, int head_dim, bool bf16, int device,
                        cudaStream_t stream) {
  // no more CTAs than chunks that the table could hold
  const int64_t most = ((int64_t(p.s.width) << p.s.page_shift) >> 6) * p.s.seqs * p.s.kv_heads *
                       ((int64_t(p.most_rows) + 8 * nt - 1) / (8 * nt));
  int grid = rows_grid(nt, device);
  if (most < grid) grid = int(most);
  if (grid < 1) return cudaSuccess;
  if (head_dim == 64)
    return bf16 ? launch_nt<64, __nv_bfloat16>(p, nt, grid, device, stream)
                : launch_nt<64, __half>(p, nt, grid, device, stream);
  return bf16 ? launch_nt<128, __nv_bfloat16>(p, nt, grid, device, stream)
              : launch_nt<128, __half>(p, nt, grid, device, stream);
}

}  // namespace kv8
