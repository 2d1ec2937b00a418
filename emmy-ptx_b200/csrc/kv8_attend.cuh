// Shared by the attention kernels over the paged 8-bit cache.
#pragma once

#include <cuda_bf16.h>

#include "kv8.cuh"

namespace kv8 {

// A plan (see kv8_plan.cu): head, then records for the parts of the row kernel,
// for those of the tile kernel, and for the tile kernel's units that were cut.
struct alignas(16) PlanHead {
  int parts, units, joins;
  int group, window, sinks, row_limit, seqs, kv_heads, nt, width, page_shift, cluster;  // what it was made for
  int pad[3];
};
struct alignas(16) PartRec {
  int b, head, c0, c1;  // chunks c0 .. c1 - 1 of the segment's line
  int part, parts, slot0, row0;
  int start, n, len, rows;
};
struct alignas(16) UnitRec {
  int b, head, row0, start;
  int n, len, c0, c1;  // chunks c0 .. c1 - 1 of the unit's line
  int slot, pad[3];    // workspace slot of a cut unit's part, -1: the unit is whole
};
struct alignas(16) JoinRec {
  int head, row0, start, rows;  // rows of the sequence's kv head
  int slot0, parts, b, pad;
};

struct AttendParams {
  Seqs s;
  const uint8_t *codes;
  const int8_t *exps;
  const void *q;
  void *out;
  int64_t q_ts, q_hs, o_ts, o_hs;  // token and head strides, elements
  float *partial;       // parts of the row kernel
  float *tile_partial;  // parts of the tile kernel: O [head_dim][256 rows], maxima, sums
  unsigned *counters;
  PlanHead *plan;
  PartRec *parts;
  UnitRec *units;
  JoinRec *joins;
  float scale_log2;  // scale * log2(e)
  int group;         // query heads of a kv head
  int window, sinks;
  int row_limit;     // sequences with more rows of a kv head than this are the tile kernel's
  int nt;            // 8-row blocks of the row kernel
  int cluster;       // CTAs of a cluster of the row kernel, 0: none
  bool beside;       // the row kernel was launched to run beside the tile kernel
  unsigned *ready;   // there: what came before both is done, and the row kernel's blocks that know
  int stall;         // one block in so many withholds its first keys (0: none)
  unsigned long long wait_ns;  // limit of the kernels' waits
};

// How large a plan gets and what it aims at, from what the host knows.
struct PlanShape {
  bool rows, tiles;    // which kernels run
  int nt;              // 8-row blocks of the row kernel
  int target;          // parts that the row kernel's segments are to be cut into
  bool spread;         // in two waves rather than one
  int cluster;         // CTAs of a cluster, which joins its parts in shared memory; 0: no clusters
  bool single;         // and every segment is one cluster
  int slots;           // workspace slots for cut segments' parts
  int tile_target;     // parts that the tile kernel's units may be cut into, 0: none is
  int64_t most_parts, most_units, most_joins;
  uint64_t partial_bytes;  // of the row kernel's parts
  uint64_t workspace_bytes, plan_bytes;
};

// The record is for this call, and what it says is within the arrays.
__device__ __forceinline__ bool plan_fits(const AttendParams &p, const PlanHead &h, int b, int start, int n, int len) {
  const bool ok = h.group == p.group && h.window == p.window && h.sinks == p.sinks && h.row_limit == p.row_limit &&
                  h.seqs == p.s.seqs && h.kv_heads == p.s.kv_heads && h.nt == p.nt && h.width == p.s.width && h.cluster == p.cluster &&
                  h.page_shift == p.s.page_shift && start + n <= p.s.tokens &&
                  len <= (int64_t(p.s.width) << p.s.page_shift);
  if (!ok) report(p.s.status, STATUS_PLAN);
  return ok;
}

// Which keys a block of query rows sees, and the 64-key chunks that hold
// them: those of the sinks, then those of the window.  Chunks never straddle
// a page (page sizes are multiples of 64).
struct Span {
  int first, last;  // positions of the first and last token
  int window, sinks;
  int sink_chunks, window_chunk0, chunks;

  Span() = default;
  // tokens at positions first_ .. last_, first_ <= last_
  __device__ __forceinline__ Span(const AttendParams &p, int first_, int last_)
      : first(first_), last(last_), window(p.window), sinks(p.sinks) {
    const int low = window > 0 ? max(0, first - window + 1) : 0;
    window_chunk0 = low >> 6;
    sink_chunks = min((sinks + 63) >> 6, window_chunk0);
    chunks = sink_chunks + (last >> 6) + 1 - window_chunk0;
  }
  // first key of chunk i of the line
  __device__ __forceinline__ int key0(int i) const {
    return (i < sink_chunks ? i : i - sink_chunks + window_chunk0) << 6;
  }
  __device__ __forceinline__ bool sees(int pos, int key) const {
    return key <= pos && (window == 0 || pos - key < window || key < sinks);
  }
  __device__ __forceinline__ bool any_sees(int key) const {
    return key <= last && (window == 0 || first - key < window || key < sinks);
  }
  // every token sees keys a .. b
  __device__ __forceinline__ bool all_see(int a, int b) const {
    return b <= first && (window == 0 || last - a < window || b < sinks);
  }
  // some token sees some key of a .. b
  __device__ __forceinline__ bool wanted(int a, int b) const {
    return a <= last && (window == 0 || first - b < window || a < sinks);
  }
};

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float &lo, float &hi);
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float &lo, float &hi) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t w, float &lo, float &hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
  lo = f.x;
  hi = f.y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Maxima beyond this (log2 units) leave no room in f32 for the exponents that are
// added to them elsewhere: V's unit is then kept at the page's own exponent.
constexpr float BIG = 65536.0f;
// The maximum of a row that has seen no key: f32's lowest, below every score but
// -inf.  (Not -inf: hidden scores are that, and -inf - -inf is NaN.)
constexpr float NONE = -3.402823466e38f;
__device__ __forceinline__ bool is_big(float m) { return fabsf(m) > BIG && m != NONE; }

// 2^x: subnormal results are zero, 2^-inf = 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Exponent k of a row's largest finite magnitude, 2^k <= amax < 2^(k + 1),
// kept where 2^k and 2^-k are normal f32; 0 for a row of zeros.
__device__ __forceinline__ int row_exponent(float amax) {
  const int e = int(__float_as_uint(amax) >> 23) - 127;
  return amax == 0.0f ? 0 : max(min(e, 126), -126);
}

// Rows of a kv head up to which a sequence is the row kernel's, in blocks of at
// most ROWS_BLOCK rows that each read the keys again, from L2, as neighbours: 16
// rows' sums are what registers hold at three CTAs an SM, but for one register's
// spill where d = 128 and clusters join (blocks of 32 at two CTAs: 28.4 us against
// 29.5 for five drafts of 16 sequences, but spills from 25 rows on).  Row kernel |
// tile kernel, 16 sequences of 500-6000 keys, by rows, us: d = 128, 5 heads: 17:
// 33 | 57, 32: 36 | 58, 40: 51 | 58, 48: 53 | 58, 64: 61 | 58; d = 64, 8 heads: 17:
// 36 | 58, 32: 38 | 60, 40: 65 | 60, 48: 65 | 76, 64: 74 | 76.
constexpr int ROWS_MOST = 32, ROWS_BLOCK = 16;
constexpr int ROWS_PER_SM = 3;  // CTAs of the row kernel, by its launch bounds
constexpr int TILE_ROWS = 256;  // rows of a unit of the tile kernel
constexpr int TILE_CUT = 8;     // chunks of a unit's part at least: a cut has to be worth its join
// 8-row blocks of a CTA of the row kernel, for the rows of the largest sequence.
inline int rows_blocks(int64_t rows) { return rows <= 8 ? 1 : 2; }

int plan_attend(const AttendParams &p, const PlanShape &shape, cudaStream_t stream);
int tiles_attend(const AttendParams &p, const emmy_kv8 &cache, const PlanShape &shape, bool bf16, cudaStream_t stream);
int tiles_join(const AttendParams &p, const emmy_kv8 &cache, const PlanShape &shape, bool bf16, cudaStream_t stream);
int rows_attend(const AttendParams &p, const emmy_kv8 &cache, const PlanShape &shape, bool bf16, cudaStream_t stream);

}  // namespace kv8
