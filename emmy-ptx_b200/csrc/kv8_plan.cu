// emmy_kv8_attend_plan -- how attend cuts its work, from the lengths on the
// device.
//
// Row kernel: a segment is one (sequence, kv head) with its visible 64-key
// chunks.  Where all segments fit on the GPU at once, parts of at most q
// chunks, q the least of a few tries that leaves them one wave: equal parts
// that start together.  Otherwise (spread) two waves of parts of about equal
// length, which the order of arrival evens out.  Measured before the plan was
// a kernel of its own (us, one wave | two): 2 sequences of 131071 keys 37 | 43,
// 48 with a window of 1024 19 | 28, 16 with five drafts 33 | 41; but 64 of
// 700-8191 keys, 512 segments on 444 CTAs, 111 | 97.
// Tile kernel: units of 256 query rows of one (sequence, kv head), those with
// the most chunks first (by 256 steps of the most): the hardware hands units
// out in order, and the short ones fill up the end.
//
// One CTA: a thread takes a few sequences, scans give each its first record,
// and the records are then written a thread each.  A layer's worth of work for
// attend is some microseconds, and every layer of a step shares the plan.
#include "kv8_attend.cuh"

namespace kv8 {
namespace {

constexpr int THREADS = 1024, WARPS = 32, EACH = EMMY_KV8_MAX_SEQS / THREADS;
constexpr int TILE_ROWS = 256;

struct PlanParams {
  AttendParams a;
  int target, min_chunks, most_parts, most_units;
  bool spread;
};

__device__ __forceinline__ int warp_scan(int x, int lane) {  // inclusive
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += u;
  }
  return x;
}
// Exclusive scan over the block, and the total.
__device__ __forceinline__ int block_scan(int x, int &total, int *sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int at = warp_scan(x, lane);
  __syncthreads();
  if (lane == 31) sums[warp] = at;
  __syncthreads();
  const int s = sums[lane], all = warp_scan(s, lane);
  total = __shfl_sync(0xffffffffu, all, 31);
  at += warp == 0 ? 0 : __shfl_sync(0xffffffffu, all, (warp + 31) & 31);
  return at - x;
}

// Parts of a segment of c chunks, at no more than q chunks a part, or (spread)
// as near to q as may be.
__device__ __forceinline__ int parts_of(int c, int q, bool spread) {
  return c == 0 ? 0 : spread ? max(1, min((2 * c + q) / (2 * q), c)) : (c + q - 1) / q;
}

// Last i < n with first[i] <= x.
__device__ __forceinline__ int owner_of(const int *first, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS) plan_kernel(const PlanParams p) {
  __shared__ int part_at[EMMY_KV8_MAX_SEQS], slot_at[EMMY_KV8_MAX_SEQS];  // 32 KB; then unit_at
  __shared__ int sums[WARPS];
  grid_dependency_wait();
  grid_dependency_done();
  const Seqs &s = p.a.s;
  const int tid = threadIdx.x, H = s.kv_heads, b0 = tid * EACH;
  int chunks[EACH], blocks[EACH];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    chunks[i] = blocks[i] = 0;
    if (b0 + i < s.seqs) {
      int start, n, len;
      lengths(s, b0 + i, start, n, len);
      if (n > 0) {
        if (n * p.a.group <= p.a.row_limit)
          chunks[i] = Span(p.a, len - n, len - 1).chunks;
        else
          blocks[i] = (n * p.a.group + TILE_ROWS - 1) / TILE_ROWS;
      }
    }
    mine += chunks[i];
  }
  int all;
  block_scan(mine, all, sums);
  const int64_t work = int64_t(all) * H;
  const int q0 = max(p.min_chunks, int((work + p.target - 1) / p.target));
  int q = q0;
  if (!p.spread)
    for (int t = 1; t < 5; ++t) {
      int parts = 0, total;
#pragma unroll
      for (int i = 0; i < EACH; ++i) parts += parts_of(chunks[i], q, false);
      block_scan(parts, total, sums);
      if (int64_t(total) * H <= p.target) break;
      q = q0 + (q0 * (1 << t) + 15) / 16;  // 1/8, 1/4, 1/2, 1 above q0
    }
  int parts = 0, slots = 0, n_parts, n_slots, n_units, units = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int k = parts_of(chunks[i], q, p.spread);
    parts += k * H;
    slots += k > 1 ? k * H : 0;
    units += blocks[i] * H;
  }
  int at = block_scan(parts, n_parts, sums), slot = block_scan(slots, n_slots, sums);
  int unit = block_scan(units, n_units, sums);
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (b0 + i < s.seqs) {
      const int k = parts_of(chunks[i], q, p.spread);
      part_at[b0 + i] = at;
      slot_at[b0 + i] = slot;
      at += k * H;
      slot += k > 1 ? k * H : 0;
    }
  __syncthreads();
  // the launches have room for so many (see rows_attend and tiles_attend)
  n_parts = min(n_parts, p.most_parts);
  n_units = min(n_units, p.most_units);
  if (tid == 0)
    *p.a.plan = PlanHead{n_parts, n_units, p.a.group, p.a.window, p.a.sinks, p.a.row_limit, s.seqs, H, p.a.nt, s.width, s.page_shift, 0};
  for (int i = tid; i < n_parts; i += THREADS) {
    const int b = owner_of(part_at, s.seqs, i), rel = i - part_at[b];
    PartRec r;
    r.b = b;
    lengths(s, b, r.start, r.n, r.len);
    const int c = Span(p.a, r.len - r.n, r.len - 1).chunks, k = parts_of(c, q, p.spread);
    r.head = rel / k;
    r.part = rel - r.head * k;
    r.parts = k;
    r.slot0 = slot_at[b] + r.head * k;
    r.c0 = int(int64_t(c) * r.part / k);
    r.c1 = int(int64_t(c) * (r.part + 1) / k);
    r.chunks = c;
    r.pad = 0;
    p.a.parts[i] = r;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (b0 + i < s.seqs) {
      part_at[b0 + i] = unit;
      unit += blocks[i] * H;
    }
  __syncthreads();
  // counting sort by chunks, the most first; units alike in any order
  const auto unit_of = [&](int i, int &chunks) {
    const int b = owner_of(part_at, s.seqs, i), rel = i - part_at[b];
    UnitRec r;
    r.b = b;
    lengths(s, b, r.start, r.n, r.len);
    r.head = rel % H;
    r.row0 = ((r.n * p.a.group + TILE_ROWS - 1) / TILE_ROWS - 1 - rel / H) * TILE_ROWS;
    r.pad[0] = r.pad[1] = 0;
    const int last = min(r.row0 + TILE_ROWS, r.n * p.a.group) - 1, first = r.len - r.n;
    chunks = Span(p.a, first + r.row0 / p.a.group, first + last / p.a.group).chunks;
    return r;
  };
  constexpr int STEPS = 256;
  __shared__ int count[STEPS], most;
  if (tid < STEPS) count[tid] = 0;
  if (tid == 0) most = 1;
  __syncthreads();
  int c, top = 1;
  for (int i = tid; i < n_units; i += THREADS) {
    unit_of(i, c);
    top = max(top, c);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) atomicMax(&most, top);
  __syncthreads();
  const auto step_of = [&](int chunks) { return int(int64_t(most - chunks) * STEPS / (most + 1)); };
  for (int i = tid; i < n_units; i += THREADS) {
    unit_of(i, c);
    atomicAdd(&count[step_of(c)], 1);
  }
  __syncthreads();
  const int mine_count = tid < STEPS ? count[tid] : 0;
  const int before = block_scan(mine_count, c, sums);
  if (tid < STEPS) count[tid] = before;
  __syncthreads();
  for (int i = tid; i < n_units; i += THREADS) {
    const UnitRec r = unit_of(i, c);
    p.a.units[atomicAdd(&count[step_of(c)], 1)] = r;
  }
}

}  // namespace

int plan_attend(const AttendParams &a, const PlanShape &shape, cudaStream_t stream) {
  PlanParams p;
  p.a = a;
  p.target = shape.target;
  p.spread = shape.spread;
  p.min_chunks = 2;  // a join costs about what ten chunks do
  p.most_parts = int(shape.most_parts);
  p.most_units = int(shape.most_units);
  return launch_kernel("emmy_kv8_attend_plan", plan_kernel, dim3(1), THREADS, 0, stream, p);
}

}  // namespace kv8
