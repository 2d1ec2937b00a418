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
// maxima, sums and O are f32; p is rounded to f16, because both products are
// f16's: by up to 2^-11 of it, and where it is below 2^-14 by up to 2^-25 of its
// unit, which is at most 2^6 of the row's (V's exponent may stray by so much).
// Their sum l is of the weights before that rounding -- of those after it would
// cost a conversion a weight -- so an f16 output differs from f32 arithmetic's
// in its last bit (2.4e-4 from 64 bits where f32 weights are 2.1e-4, very long
// keys), and many small weights beside a large one lose bits that l has.
//
// The order of a contraction's terms is free, so a lane's 16 consecutive bytes
// of a key serve as its shares of four k-steps, and of a value row as the rows
// 2i, 2i+1 of D / 16 m-tiles: codes go from shared memory to MMA fragments by
// 8- and 16-byte loads and one conversion, with no shuffles.  A fifth warp
// brings 64-key chunks of K and V by TMA, several ahead: the bytes in flight
// that HBM's latency asks for cost no registers.  The TMA's swizzle spreads
// the rows that the lanes of a load read over all banks.
//
// Bound by memory: codes are read once for each block of up to 16 rows of a kv
// head, by neighbours, so from memory once.  A segment -- one sequence, kv head
// and block of rows -- is cut into about as many parts of 64-key chunks as its
// share of a target number of parts, a CTA a part, so uneven lengths balance and
// one long sequence fills the GPU, while a segment of about a part's length
// stays whole and needs no join.  Parts of a cut segment leave (m, l, O) in
// the workspace; up to ONE_LEVEL of them are joined by the last to arrive, in
// their order, more in groups by the last of each group and then the groups by
// the last of those, so results do not depend on the order of arrival.  Where
// there are few segments, clusters of CTAs join their parts first, each a share
// of the rows' values out of the others' shared memory: a short segment is one
// cluster and needs neither the workspace nor its round trips to L2, a long one
// leaves a result a cluster there.
#include <cuda_bf16.h>

#include <cuda.h>  // CUtensorMap

#include "kv8_async.cuh"
#include "kv8_attend.cuh"

namespace kv8 {
namespace {

constexpr int WARPS = 4, THREADS = 160, ALL_WARPS = 5;  // four that compute, one that loads
constexpr float LAZY = 8.0f;  // log2 units that scores may pass the reference before O moves
// Parts of a segment that one CTA joins at once, or up to ONE_LEVEL where that
// leaves one level (one level | two, us: 23 results 33.5 | 35.0, 28 results 17.6 |
// 18.5, 52 results 23.5 | 21.5).
constexpr int GROUP = 16, ONE_LEVEL = 24;
constexpr int MOST_CLUSTER = 8;
constexpr int UNIT_LAZY = 6;  // the same for V's exponent: p stays below 2^14 in f16

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
  int row0, rows;              // first row of the kv head, and how many, at most 8 NT
  int part, parts, slot0;      // this CTA's part, of how many; workspace slot of part 0
  Span span;
};

// What goes with a chunk of codes.
struct ChunkInfo {
  int key0, ek, ev, dead;
};

// Shared memory: the ring of chunks (K rows, then V rows; the join of the warps
// once the loop is over), then the staged queries.
template <int D, int NT>
struct Layout {
  static constexpr int CHUNK = 2 * 64 * D;
  static constexpr int STAGES = 64 * 1024 / CHUNK;
  static constexpr int QUERIES = STAGES * CHUNK, END = QUERIES + NT * 16 * D;
  static constexpr int DYN = END + 1024;  // the swizzle repeats every 1 KB
  static constexpr int LD = D + 4;        // floats of a row of the join
  static_assert((WARPS * LD + D) * 8 * NT * 4 <= QUERIES, "the join and a cluster's part fit over the ring");
  static_assert(2 * 64 * 8 * NT * 4 <= QUERIES, "so do the maxima and sums of 64 parts");
};

__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap *map, int row, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst),
      "l"(map), "r"(0), "r"(row), "r"(smem_addr(bar))
      : "memory");
}

// Codes of 16 keys as a lane holds them, g = lane / 4, q = lane % 4: K rows g
// and g + 8 (D / 4 bytes at q D / 4), V rows 2q, 2q+1, 2q+8, 2q+9 (D / 8 bytes
// at g D / 8).  The swizzle exchanges a row's 16-byte pieces: by row & 7 in
// rows of 128 bytes, by row / 2 & 3 in rows of 64.
template <int D>
__device__ __forceinline__ void load_k(uint32_t (&k)[2][D / 16], const uint8_t *rows, int gr, int q) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const int piece = D == 128 ? (2 * q + j) ^ gr : q ^ (gr >> 1 & 3);
      const uint4 w = *reinterpret_cast<const uint4 *>(rows + (gr + 8 * i) * D + 16 * piece);
      k[i][4 * j] = w.x, k[i][4 * j + 1] = w.y, k[i][4 * j + 2] = w.z, k[i][4 * j + 3] = w.w;
    }
}
template <int D>
__device__ __forceinline__ void load_v(uint32_t (&v)[4][D / 32], const uint8_t *rows, int gr, int q) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 2 * q + (i & 1);  // row & 7
    const uint8_t *row = rows + (r + 8 * (i >> 1)) * D;
    if constexpr (D == 64) {
      const uint2 w = *reinterpret_cast<const uint2 *>(row + 16 * ((gr >> 1) ^ q) + 8 * (gr & 1));
      v[i][0] = w.x, v[i][1] = w.y;
    } else {
      const uint4 w = *reinterpret_cast<const uint4 *>(row + 16 * (gr ^ r));
      v[i][0] = w.x, v[i][1] = w.y, v[i][2] = w.z, v[i][3] = w.w;
    }
  }
}

// What a warp carries over its tiles, for rows 2q, 2q+1 of each 8-row block.
template <int D, int NT>
struct State {
  float o[D / 16][NT][4];
  float m[NT][2], l[NT][2];
  int unit;           // O is in units of 2^unit
  bool big;           // some row's maximum is
};

// Scores in log2 units -> weights, b = P^T as B fragments; moves the maxima
// and O where it must.
template <int D, int NT>
__device__ __forceinline__ void softmax_step(State<D, NT> &st, float (&s)[NT][4], uint32_t (&b)[NT][2], int ev) {
  bool grow = false;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) grow |= s[i][c] > st.m[i][c & 1] + LAZY;
  const bool move = ev - st.unit > UNIT_LAZY || st.unit - ev > UNIT_LAZY || (st.big && ev != st.unit);
  if (__any_sync(0xffffffffu, grow) || move) {
    bool big = false;
    float f[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
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
        big |= is_big(top);
      }
    }
    st.big = __any_sync(0xffffffffu, big);
    float unit = 1.0f;
    if (move || st.big) {
      unit = pow2(st.unit - ev);
      st.unit = ev;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        st.o[j][i][0] *= f[i][0] * unit, st.o[j][i][2] *= f[i][0] * unit;
        st.o[j][i][1] *= f[i][1] * unit, st.o[j][i][3] *= f[i][1] * unit;
      }
  }
  // p = 2^(s - m) in units of 2^(unit - ev); P^T by 8 x 8 transposes
  const float dev = float(ev - st.unit), undo = pow2(st.unit - ev);
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
}

// O^T += V^T P^T of 16 keys.
template <int D, int NT>
__device__ __forceinline__ void pv_step(State<D, NT> &st, const uint32_t (&v)[4][D / 32], const uint32_t (&b)[NT][2]) {
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const uint32_t sel = i & 1 ? 0x7362 : 0x5140;  // (key 2q, key 2q+1) of two neighbouring d
    const uint32_t x = __byte_perm(v[0][i / 2], v[1][i / 2], sel);
    const uint32_t y = __byte_perm(v[2][i / 2], v[3][i / 2], sel);
    const uint32_t a[4] = {e4m3x2_f16x2(x), e4m3x2_f16x2(x >> 16), e4m3x2_f16x2(y), e4m3x2_f16x2(y >> 16)};
#pragma unroll
    for (int r = 0; r < NT; ++r) mma(st.o[i][r], a, b[r][0], b[r][1]);
  }
}

// A hidden key has p = 0, but 0 * NaN is NaN: values of a tile that no row sees
// become zero, and a NaN that only some rows see is taken out (take_nan) and
// put into those rows' sums after their P V (put_nan).
template <int D>
__device__ __forceinline__ bool hide_values(uint32_t (&v)[4][D / 32], const Segment &g, int key0, bool dead, int q) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t keep = !dead && g.span.any_sees(key0 + 2 * q + (i & 1) + 8 * (i >> 1)) ? 0xffffffffu : 0u;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      v[i][w] &= keep;
      any |= nan_bytes(v[i][w]);
    }
  }
  return __any_sync(0xffffffffu, any != 0);
}
template <int D>
__device__ __forceinline__ void take_nan(uint32_t (&v)[4][D / 32], uint32_t (&nan_at)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    nan_at[i] = 0;  // bit d: value d of the lane's V row i is NaN
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      const uint32_t bad = nan_bytes(v[i][w]);
      v[i][w] &= ~((bad >> 7) * 0xffu);
#pragma unroll
      for (int j = 0; j < 4; ++j) nan_at[i] |= ((bad >> (8 * j + 7)) & 1u) << (4 * w + j);
    }
  }
}
template <int D, int NT>
__device__ __forceinline__ void put_nan(State<D, NT> &st, const uint32_t (&nan_at)[4], const Segment &g,
                                        const int *row_pos, int key0, int lane) {
  uint32_t rows[NT][2] = {};  // bit d: the row sees a NaN in value d
  for (int from = 0; from < 4; ++from)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bits = __shfl_sync(0xffffffffu, nan_at[i], (lane & ~3) | from);
      const int key = key0 + 2 * from + (i & 1) + 8 * (i >> 1);
#pragma unroll
      for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (g.span.sees(row_pos[8 * r + 2 * (lane & 3) + c], key)) rows[r][c] |= bits;
    }
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (rows[r][c & 1] >> (2 * i + (c >> 1)) & 1u) st.o[i][r][c] = NAN;
}

// One row's share of a lane: Q[q D / 4 .. + D / 4 - 1], scaled into f16; returns the row's exponent (row = f16 row * 2^exponent).
template <int D, typename T>
__device__ __forceinline__ int query_row(uint32_t (&f)[D / 8], const T *row, int q) {
  float x[D / 4];
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (row != nullptr) w = *reinterpret_cast<const uint4 *>(row + D / 4 * q + 16 * j + 8 * h);
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
// RESULT: every part, of a sequence's own keys or of those that a run shares, leaves
// its rows in a slot of its own, for a kernel that joins them all.
template <int D, int NT, bool CLUSTER, bool RESULT, typename T>
__device__ __forceinline__ void attend_part(const AttendParams &p, const CUtensorMap &codes_map) {
  using L = Layout<D, NT>;
  constexpr int ROWS = 8 * NT, LD = L::LD;
  extern __shared__ uint8_t dyn_raw[];
  uint8_t *const dyn = dyn_raw + ((1024 - (smem_addr(dyn_raw) & 1023)) & 1023);
  float *const join = reinterpret_cast<float *>(dyn);
  __shared__ float sm_m[WARPS][ROWS], sm_l[WARPS][ROWS], row_l[ROWS], row_m[ROWS];
  __shared__ int sm_unit[WARPS], row_pos[ROWS];  // position of the row's token, -1: no such row
  __shared__ float row_mult[ROWS];               // scale * log2(e) * the row's power of two
  __shared__ unsigned ticket, stop_word;
  __shared__ uint64_t full[L::STAGES], empty[L::STAGES];
  __shared__ ChunkInfo infos[L::STAGES];
  volatile unsigned *const stop = &stop_word;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gr = lane >> 2, q = lane & 3;
  const Seqs &s = p.s;
  const PlanHead head = *p.plan;
  const PartRec rec = p.parts[blockIdx.x];
  // (the block that waits in the end lets the next kernel start after that only:
  // its CTAs would take SMs in the order that these leave them, 257 for 248 us a
  // batch of prompts)
  if (!p.beside || blockIdx.x != 0) grid_dependency_done();
  // (a run's tokens stand behind its shared keys as if they were one sequence's)
  if (blockIdx.x >= head.parts || !plan_fits(p, head, rec.b, rec.start, rec.n, RESULT ? rec.len - rec.n : rec.len)) return;
  const Segment g = {rec.b, rec.head, rec.start, rec.n, rec.len, rec.row0, rec.rows, rec.part, rec.parts, rec.slot0,
                     Span(p, rec.len - rec.n, rec.len - 1)};
  const int c0 = rec.c0, c1 = rec.c1;
  if (tid == 0) {
    for (int i = 0; i < L::STAGES; ++i) {
      bar_init(&full[i], 1);
      bar_init(&empty[i], WARPS);
    }
    stop_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < ROWS) row_pos[tid] = tid < g.rows ? g.len - g.n + (g.row0 + tid) / p.group : -1;
  __syncthreads();

  State<D, NT> st;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
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
  st.big = false;
  const auto row_at = [&](int r, int64_t ts, int64_t hs) {
    const int i = (g.row0 + r) / p.group, h = g.head * p.group + (g.row0 + r) - i * p.group;
    return (g.start + i) * ts + h * hs;
  };

  if (warp == WARPS) {
    // ---- chunks of codes, 32 chunks' pages and exponents at once ----
    const uint32_t who = elected();
    const int *table = s.table + int64_t(g.b) * s.width;
    Ring ring;
    bool ok = true, stalled = p.stall > 0 && blockIdx.x % p.stall == 0;
    for (int base = c0; ok && base < c1; base += 32) {
      ChunkInfo mine = {0, 0, 0, 0};
      int64_t unit = 0;
      if (base + lane < c1) {
        mine.key0 = g.span.key0(base + lane);
        int page = table[mine.key0 >> s.page_shift];
        mine.dead = page < 0 || page >= s.pages;
        if (mine.dead) {
          report(s.status, STATUS_PAGE);
          page = 0;
        }
        unit = int64_t(page) * 2 * s.kv_heads + g.head;
        mine.ek = p.exps[unit];
        mine.ev = p.exps[unit + s.kv_heads];
      }
      const int k_row = int((unit << s.page_shift) + (mine.key0 & ((1 << s.page_shift) - 1)));
      const auto copy = [&](int i, int slot) {
        const int row = __shfl_sync(0xffffffffu, k_row, i);
        if (who) {
          const uint32_t dst = smem_addr(dyn + slot * L::CHUNK);
          asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(&full[slot])),
                       "r"(L::CHUNK)
                       : "memory");
          tma_rows(dst, &codes_map, row, &full[slot]);
          tma_rows(dst + 64 * D, &codes_map, row + (s.kv_heads << s.page_shift), &full[slot]);
        }
      };
      const int count = min(32, c1 - base);
      // the first chunks' copies start before their exponents are here
      const int early = base == c0 ? min(count, L::STAGES) : 0;
      for (int i = 0; i < early; ++i) copy(i, i);
      for (int i = 0; i < count; ++i, ring.next(L::STAGES)) {
        if (i >= early) {
          ok = warp_wait(&empty[ring.slot], ring.phase ^ 1, stop, s.status, p.wait_ns);
          if (!ok) break;
          copy(i, ring.slot);
        }
        ChunkInfo c;
        c.key0 = __shfl_sync(0xffffffffu, mine.key0, i);
        // (not where they were loaded: their first use would hold up the early copies)
        c.ek = held_exponent(__shfl_sync(0xffffffffu, mine.ek, i));
        c.ev = held_exponent(__shfl_sync(0xffffffffu, mine.ev, i));
        c.dead = __shfl_sync(0xffffffffu, mine.dead, i);
        if (who) {
          infos[ring.slot] = c;
          if (!stalled) bar_arrive(&full[ring.slot]);
        }
        stalled = false;
      }
    }
  } else {
    // ---- queries ----
    uint32_t own[NT == 1 ? D / 8 : 1];
    float mult[2];
    uint32_t *const staged = reinterpret_cast<uint32_t *>(dyn + L::QUERIES);
    if constexpr (NT == 1) {
      const T *row = gr < g.rows ? static_cast<const T *>(p.q) + row_at(gr, p.q_ts, p.q_hs) : nullptr;
      const int e = query_row<D>(own, row, q);
      mult[0] = p.scale_log2 * pow2(__shfl_sync(0xffffffffu, e, 8 * q));
      mult[1] = p.scale_log2 * pow2(__shfl_sync(0xffffffffu, e, 8 * q + 4));
    } else {
      if (warp < NT) {
        const int r = 8 * warp + gr;
        uint32_t f[D / 8];
        const T *row = r < g.rows ? static_cast<const T *>(p.q) + row_at(r, p.q_ts, p.q_hs) : nullptr;
        const int e = query_row<D>(f, row, q);
        if (q == 0) row_mult[r] = p.scale_log2 * pow2(e);
#pragma unroll
        for (int w = 0; w < D / 16; ++w)
          *reinterpret_cast<uint2 *>(&staged[((w * NT + warp) * 32 + lane) * 2]) = make_uint2(f[2 * w], f[2 * w + 1]);
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
    }
    const auto mult_of = [&](int i, int c) {
      if constexpr (NT == 1)
        return mult[c];
      else
        return row_mult[8 * i + 2 * q + c];
    };
    const auto query = [&](int w, int i) {
      if constexpr (NT == 1)
        return make_uint2(own[2 * w], own[2 * w + 1]);
      else
        return *reinterpret_cast<const uint2 *>(&staged[((w * NT + i) * 32 + lane) * 2]);
    };
    // chunks whole_lo .. whole_hi - 1 every row sees whole
    int whole_lo = 0;
    const int whole_hi = g.span.sink_chunks + ((g.span.first + 1) >> 6) - g.span.window_chunk0;
    if (p.window > 0)
      whole_lo = g.span.sink_chunks + max(0, ((max(0, g.span.last - p.window + 1) + 63) >> 6) - g.span.window_chunk0);

    // ---- 16 keys of each chunk a warp ----
    Ring ring;
    for (int chunk = c0; chunk < c1; ++chunk, ring.next(L::STAGES)) {
      if (!warp_wait(&full[ring.slot], ring.phase, stop, s.status, p.wait_ns)) break;
      const uint8_t *rows = dyn + ring.slot * L::CHUNK + 16 * warp * D;
      const ChunkInfo info = infos[ring.slot];
      // S^T = K Q^T, in two chains of sums
      constexpr int CHAINS = 2;
      float sum[CHAINS][NT][4] = {};
      {
        uint32_t k[2][D / 16];
        load_k<D>(k, rows, gr, q);
#pragma unroll
        for (int w = 0; w < D / 16; ++w) {
          const uint32_t a[4] = {e4m3x2_f16x2(k[0][w]), e4m3x2_f16x2(k[1][w]), e4m3x2_f16x2(k[0][w] >> 16),
                                 e4m3x2_f16x2(k[1][w] >> 16)};
#pragma unroll
          for (int r = 0; r < NT; ++r) {
            const uint2 q2 = query(w, r);
            mma(sum[w % CHAINS][r], a, q2.x, q2.y);
          }
        }
      }
      uint32_t v[4][D / 32];
      load_v<D>(v, rows + 64 * D, gr, q);
      warp_arrive(&empty[ring.slot]);
      if (chunk == c0) st.unit = info.ev;
      const float mk = pow2(info.ek);
      float sc[NT][4];
#pragma unroll
      for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          sc[r][c] = (CHAINS == 2 ? sum[0][r][c] + sum[CHAINS - 1][r][c] : sum[0][r][c]) * (mult_of(r, c & 1) * mk);
      uint32_t b[NT][2];
      bool nan = false;
      const int key0 = info.key0 + 16 * warp;
      if (info.dead || chunk < whole_lo || chunk >= whole_hi) {
#pragma unroll
        for (int r = 0; r < NT; ++r)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (info.dead || !g.span.sees(row_pos[8 * r + 2 * q + (c & 1)], key0 + gr + 8 * (c >> 1)))
              sc[r][c] = -INFINITY;
        nan = hide_values<D>(v, g, key0, info.dead, q);
      }
      softmax_step(st, sc, b, info.ev);
      uint32_t nan_at[4];
      if (nan) take_nan<D>(v, nan_at);
      pv_step(st, v, b);
      if (nan) put_nan(st, nan_at, g, row_pos, key0, lane);
    }
  }

  // ---- join the warps ----
  __syncthreads();
  if (*stop != 0) {
    // given up: copies in flight land first (50 ms).  The block then goes on: a
    // cluster's others read its shared memory, and the parts of a segment count
    // each other in the workspace, whose counters go back to zero only if all come.
    const unsigned long long t0 = now_ns();
    while (now_ns() - t0 < 50000000ull) {
    }
  }
  // Value gr D / 8 + 2 j + e of a row lies at 16 j + 2 gr + e: the lanes that
  // store together (gr and 8 q) then meet in no bank.
  if (warp < WARPS) {
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
          *reinterpret_cast<float2 *>(&join[(warp * ROWS + r) * LD + 16 * j + 2 * gr]) =
              make_float2(st.o[j][i][c], st.o[j][i][c + 2]);
      }
    if (lane == 0) sm_unit[warp] = st.unit;
  }
  __syncthreads();
  const bool whole = !CLUSTER && !RESULT && g.parts == 1;
  const int rows = g.rows;
  const auto store = [&](int r, int d, const float (&x)[8], float l) {
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    uint4 w;
    w.x = pack2<T>(x[0] * by, x[1] * by);
    w.y = pack2<T>(x[2] * by, x[3] * by);
    w.z = pack2<T>(x[4] * by, x[5] * by);
    w.w = pack2<T>(x[6] * by, x[7] * by);
    *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + row_at(r, p.o_ts, p.o_hs) + d) = w;
  };
  const auto part_slot = [&](int c) { return p.partial + int64_t(g.slot0 + c) * ROWS * (D + 2); };
  // a cluster's parts stay in shared memory, behind what is joined here
  float *const slot = CLUSTER ? join + WARPS * ROWS * LD : RESULT ? part_slot(0) : part_slot(g.part);
  for (int i = tid; i < rows * (D / 8); i += THREADS) {
    const int r = i / (D / 8), d = i % (D / 8) * 8;
    float m = NONE, l = 0.0f, x[8] = {};
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sm_m[w][r]);
    const float *at = &join[r * LD + d % (D / 8) * 8 + d / (D / 8) * 2];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      float f = exp2_fast(sm_m[w][r] - m);
      l += f * sm_l[w][r];
      f *= pow2(sm_unit[w]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 u = *reinterpret_cast<const float2 *>(at + w * ROWS * LD + 16 * j);
        x[2 * j] += f * u.x, x[2 * j + 1] += f * u.y;
      }
    }
    if (!whole && d == 0) row_m[r] = m, row_l[r] = l;
    if (whole) {
      store(r, d, x, l);
    } else {
      *reinterpret_cast<float4 *>(slot + r * D + d) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4 *>(slot + r * D + d + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
  }
  if (whole) return;
  // results of the segment that go through the workspace, and which is this
  const int results = CLUSTER ? g.parts / p.cluster : g.parts, result = CLUSTER ? g.part / p.cluster : g.part;
  if constexpr (CLUSTER) {
    const int n = p.cluster;
    cluster_sync();
    const int share = (rows * (D / 4) + n - 1) / n, i0 = cluster_rank() * share;
    for (int i = i0 + tid; i < min(i0 + share, rows * (D / 4)); i += THREADS) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float4 u[MOST_CLUSTER];
      float ms[MOST_CLUSTER], ls[MOST_CLUSTER], m = NONE, l = 0.0f;
#pragma unroll
      for (int c = 0; c < MOST_CLUSTER; ++c)
        if (c < n) {
          ms[c] = peer_load(peer_addr(&row_m[r], c));
          ls[c] = peer_load(peer_addr(&row_l[r], c));
          u[c] = peer_load4(peer_addr(slot + r * D + d, c));
          m = fmaxf(m, ms[c]);
        }
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int c = 0; c < MOST_CLUSTER; ++c)
        if (c < n) {
          const float f = exp2_fast(ms[c] - m);
          l += f * ls[c];
          x.x += f * u[c].x, x.y += f * u[c].y, x.z += f * u[c].z, x.w += f * u[c].w;
        }
      if (results > 1) {
        float *const to = part_slot(result);
        __stcg(reinterpret_cast<float4 *>(to + r * D + d), x);
        if (d == 0) {
          __stcg(to + ROWS * D + r, m);
          __stcg(to + ROWS * D + ROWS + r, l);
        }
        continue;
      }
      const float by = l == 0.0f ? 0.0f : 1.0f / l;
      *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + row_at(r, p.o_ts, p.o_hs) + d) =
          make_uint2(pack2<T>(x.x * by, x.y * by), pack2<T>(x.z * by, x.w * by));
    }
    cluster_sync();  // no block ends while another reads it
    if (results == 1 || cluster_rank() != 0) return;
  }
  if constexpr (!CLUSTER) {
    __syncthreads();
    if (tid < rows) {
      __stcg(slot + ROWS * D + tid, row_m[tid]);
      __stcg(slot + ROWS * D + ROWS + tid, row_l[tid]);
    }
  }
  if constexpr (RESULT) return;
  // ---- parts join in groups of GROUP, groups in the segment: the last of
  // each to arrive does it, in the parts' order ----
  const auto last_of = [&](int c, int level, int count) {
    __syncthreads();
    if (tid == 0) {
      // the barrier orders the block's stores before this thread's fence
      unsigned *at = p.counters + (g.slot0 + c) * 2 + level;
      __threadfence();
      ticket = atomicAdd(at, 1u);
      if (ticket == unsigned(count - 1)) *at = 0;
      __threadfence();
    }
    __syncthreads();
    return ticket == unsigned(count - 1);
  };
  // parts a, a + step, .. as one: into `out`, or over part a
  float *const part_m = join, *const part_l = join + 64 * ROWS;  // at most 64 parts at once
  const auto gather = [&](int a, int count, int step, bool last) {
    for (int i = tid; i < count * ROWS; i += THREADS) {
      const float *at = part_slot(a + i / ROWS * step) + ROWS * D + i % ROWS;
      part_m[i] = __ldcg(at);
      part_l[i] = __ldcg(at + ROWS);
    }
    __syncthreads();
    for (int r = warp; r < rows; r += ALL_WARPS) {  // a lane two parts
      const float m0 = lane < count ? part_m[lane * ROWS + r] : NONE;
      const float m1 = lane + 32 < count ? part_m[(lane + 32) * ROWS + r] : NONE;
      float m = fmaxf(m0, m1);
      for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      const float f0 = exp2_fast(m0 - m), f1 = exp2_fast(m1 - m);
      float l = 0.0f;
      if (lane < count) {
        part_m[lane * ROWS + r] = f0;
        l = f0 * part_l[lane * ROWS + r];
      }
      if (lane + 32 < count) {
        part_m[(lane + 32) * ROWS + r] = f1;
        l += f1 * part_l[(lane + 32) * ROWS + r];
      }
      for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      if (lane == 0) row_m[r] = m, row_l[r] = l;
    }
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += THREADS) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const float *at = part_slot(a) + r * D + d;
      const int64_t stride = int64_t(step) * ROWS * (D + 2);
      for (int c0 = 0; c0 < count; c0 += 16) {  // sixteen loads in flight
        float4 u[16];
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (c0 + c < count) u[c] = __ldcg(reinterpret_cast<const float4 *>(at + (c0 + c) * stride));
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (c0 + c < count) {
            const float f = part_m[(c0 + c) * ROWS + r];
            x.x += f * u[c].x, x.y += f * u[c].y, x.z += f * u[c].z, x.w += f * u[c].w;
          }
      }
      if (last) {
        const float by = row_l[r] == 0.0f ? 0.0f : 1.0f / row_l[r];
        *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + row_at(r, p.o_ts, p.o_hs) + d) =
            make_uint2(pack2<T>(x.x * by, x.y * by), pack2<T>(x.z * by, x.w * by));
      } else {  // only this thread reads or writes these values of part a now
        __stcg(reinterpret_cast<float4 *>(part_slot(a) + r * D + d), x);
      }
    }
    if (!last && tid < rows) {
      __stcg(part_slot(a) + ROWS * D + tid, row_m[tid]);
      __stcg(part_slot(a) + ROWS * D + ROWS + tid, row_l[tid]);
    }
  };
  // all at once up to ONE_LEVEL, else groups of GROUP, or more if there were over 64
  const int group = results <= ONE_LEVEL ? results : max(GROUP, (results + 63) / 64);
  const int lead = result / group * group, count = min(group, results - lead);
  const int groups = (results + group - 1) / group;
  if (!last_of(lead, 0, count)) return;
  gather(lead, count, 1, groups == 1);
  if (groups == 1 || !last_of(0, 1, groups)) return;
  gather(0, groups, group, true);
}

// Beside the tile kernel, which was launched before it and whose sequences are
// others, it starts when all of that kernel's CTAs run: SMs without a unit, or
// past their last, take parts (512 tokens behind 3584 keys with 47 single tokens
// of 700-8191 keys: 175 -> 129 us a call).  What came before both is done then;
// that it is also visible here, without this kernel's own wait, follows from
// the word that the tile kernel released after its wait, and a block that does
// not find it there waits.  The last block to have looked takes the word back.
// One block waits for the tile kernel in the end, so that what comes after this
// kernel comes after both.
__device__ __forceinline__ void ready_or_wait(const AttendParams &p) {
  __shared__ unsigned ready;
  if (threadIdx.x == 0)
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(ready) : "l"(p.ready) : "memory");
  __syncthreads();
  if (ready == 0) grid_dependency_wait();
  // and to the copies that the loading warp will start
  asm volatile("fence.proxy.async.global;" ::: "memory");
}
__device__ __forceinline__ void took_ready(const AttendParams &p) {
  if (threadIdx.x == 0 && atomicAdd(p.ready + 1, 1u) == gridDim.x - 1) p.ready[0] = p.ready[1] = 0;
}

template <int D, int NT, bool CLUSTER, bool RESULT, typename T>
__global__ void __launch_bounds__(THREADS, ROWS_PER_SM)
rows_kernel(const AttendParams p, const __grid_constant__ CUtensorMap codes_map) {
  if (p.beside)
    ready_or_wait(p);
  else
    grid_dependency_wait();
  attend_part<D, NT, CLUSTER, RESULT, T>(p, codes_map);
  if (p.beside) {
    took_ready(p);
    if (blockIdx.x == 0) grid_dependency_wait();
  }
}

template <int D, int NT, bool CLUSTER, bool RESULT, typename T>
int launch(const AttendParams &p, const CUtensorMap &map, int device, int grid, cudaStream_t stream) {
  static KernelSetup setup;
  const int rc = setup.ready("emmy_kv8_attend", rows_kernel<D, NT, CLUSTER, RESULT, T>, device, Layout<D, NT>::DYN);
  if (rc != EMMY_OK) return rc;
  return launch_clusters("emmy_kv8_attend", rows_kernel<D, NT, CLUSTER, RESULT, T>, CLUSTER ? p.cluster : 1, dim3(grid),
                         THREADS, Layout<D, NT>::DYN, stream, p, map);
}

template <int D, typename T>
int launch_nt(const AttendParams &p, const CUtensorMap &map, int device, int grid, cudaStream_t stream) {
  if (p.shared != SHARED_NONE)
    return p.nt == 1 ? launch<D, 1, false, true, T>(p, map, device, grid, stream)
                     : launch<D, 2, false, true, T>(p, map, device, grid, stream);
  if (p.cluster > 0)
    return p.nt == 1 ? launch<D, 1, true, false, T>(p, map, device, grid, stream)
                     : launch<D, 2, true, false, T>(p, map, device, grid, stream);
  return p.nt == 1 ? launch<D, 1, false, false, T>(p, map, device, grid, stream)
                   : launch<D, 2, false, false, T>(p, map, device, grid, stream);
}

}  // namespace

int rows_attend(const AttendParams &p, const emmy_kv8 &cache, const PlanShape &shape, bool bf16, cudaStream_t stream) {
  const int64_t grid = shape.most_parts;
  // the pool as rows of head_dim bytes, 64 of them a box
  const int64_t rows = int64_t(cache.pages) * 2 * cache.kv_heads * cache.page_size;
  emmy_tmap_desc d = {};
  d.base = cache.codes;
  d.rank = 2;
  d.dtype = EMMY_TMAP_U8;
  d.dims[0] = d.strides[0] = cache.head_dim;
  d.dims[1] = rows;
  d.box[0] = cache.head_dim;
  d.box[1] = 64;
  d.swizzle = cache.head_dim;
  d.l2_promote = 256;
  alignas(64) CUtensorMap map;
  const int rc = emmy_tmap_encode(&d, &map);
  if (rc != EMMY_OK) return rc;
  if (cache.head_dim == 64)
    return bf16 ? launch_nt<64, __nv_bfloat16>(p, map, cache.device, int(grid), stream)
                : launch_nt<64, __half>(p, map, cache.device, int(grid), stream);
  return bf16 ? launch_nt<128, __nv_bfloat16>(p, map, cache.device, int(grid), stream)
              : launch_nt<128, __half>(p, map, cache.device, int(grid), stream);
}

}  // namespace kv8
