// emmy_kv8_attend_plan -- how attend cuts its work, from the lengths on the
// device.
//
// Row kernel: a segment is one (sequence, kv head, block of up to 16 rows) with
// its visible 64-key chunks.  Where all segments fit on the GPU at once, parts
// of at most q chunks, q the least of a few tries that leaves them one wave:
// equal parts that start together.  Otherwise (spread) two waves of parts of
// about equal length, which the order of arrival evens out.  Measured, without
// clusters (us, one wave | two): 2 sequences of 131071 keys 34.8 | 40.0, 48 with
// a window of 1024 16.4 | 24.9, 16 with five drafts 33.0 | 39.3; but, with more
// segments than the 444 CTAs that fit, 64 of 700-8191 keys 117.8 | 112.8 and 56
// of 4000 92.4 | 89.3.  Short segments
// (by what the table can hold) are a cluster each, whose CTAs join in shared
// memory, and a few long ones some clusters each: fewer partial results go
// through the workspace.  Some of a cluster's parts may be empty.
// Tile kernel: units of 256 query rows of one (sequence, kv head); where there
// are fewer than SMs they are cut along the keys, too, and joined by a kernel
// of their own.  The longest come first (by 256 steps of the longest): the
// CTAs take them in turn from the front and from the back, so that those with
// the longest of one round get the shortest of the next.
//
// One CTA: a thread takes a few sequences, scans give each its first record,
// and the records are then written a thread each.  Every layer of a step shares
// the plan: 7.6 us for one sequence of 1025 keys, 10.4 for 64 of 700-8191, 21 for
// 4096 of 1-200, 35 for six prompts of 200-1500 tokens.
#include "kv8_attend.cuh"

namespace kv8 {
namespace {

constexpr int THREADS = 1024, WARPS = 32, EACH = EMMY_KV8_MAX_SEQS / THREADS;

struct PlanParams {
  AttendParams a;
  int target, min_chunks, most_parts, most_units, most_joins, tile_target;
  bool spread, single;
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

// Parts of a segment of c chunks, at no more than q chunks a part: whole
// clusters, or (spread) as near to q as may be.
__device__ __forceinline__ int parts_of(const PlanParams &p, int c, int q) {
  const int n = p.a.cluster;
  return c == 0 ? 0 : p.single ? n : n > 0 ? n * ((c + n * q - 1) / (n * q)) : p.spread ? max(1, min((2 * c + q) / (2 * q), c)) : (c + q - 1) / q;
}

// Workspace slots of a segment of k parts: one a part, or one a cluster.
__device__ __forceinline__ int slots_of(const PlanParams &p, int k) {
  const int n = p.a.cluster > 0 ? k / p.a.cluster : k;
  return n > 1 ? n : 0;
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
  int chunks[EACH], blocks[EACH];  // segments' chunks; row blocks of 16, or units of 256
  int mine = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    chunks[i] = blocks[i] = 0;
    if (b0 + i < s.seqs) {
      int start, n, len;
      lengths(s, b0 + i, start, n, len);
      if (n > 0) {
        const bool few = n * p.a.group <= p.a.row_limit;
        if (few) chunks[i] = Span(p.a, len - n, len - 1).chunks;
        const int rows = few ? ROWS_BLOCK : TILE_ROWS;
        blocks[i] = (n * p.a.group + rows - 1) / rows;
      }
    }
    mine += chunks[i] * blocks[i];
  }
  int all;
  block_scan(mine, all, sums);
  const int64_t work = int64_t(all) * H;
  const int64_t share = (work + p.target - 1) / p.target;
  const int q0 = max(p.min_chunks, int(min(share, int64_t(1) << 24)));  // a sequence has no more chunks
  int q = q0;
  if (!p.spread && !p.single)
    for (int t = 1; t <= 16; t += t < 4 ? 1 : t < 8 ? 2 : 4) {
      int parts = 0, total;
#pragma unroll
      for (int i = 0; i < EACH; ++i) parts += parts_of(p, chunks[i], q) * blocks[i];
      block_scan(parts, total, sums);
      if (int64_t(total) * H <= p.target) break;
      q = q0 + (q0 * t + 15) / 16;  // a sixteenth above q0, two, .. and at last all of it
    }
  int parts = 0, slots = 0, n_parts, n_slots, n_units, units = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int k = parts_of(p, chunks[i], q);
    parts += k * blocks[i] * H;
    slots += slots_of(p, k) * blocks[i] * H;
    units += chunks[i] > 0 ? 0 : blocks[i] * H;
  }
  int at = block_scan(parts, n_parts, sums), slot = block_scan(slots, n_slots, sums);
  int unit = block_scan(units, n_units, sums);
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (b0 + i < s.seqs) {
      const int k = parts_of(p, chunks[i], q);
      part_at[b0 + i] = at;
      slot_at[b0 + i] = slot;
      at += k * blocks[i] * H;
      slot += slots_of(p, k) * blocks[i] * H;
    }
  __syncthreads();
  n_parts = min(n_parts, p.most_parts);
  for (int i = tid; i < n_parts; i += THREADS) {
    const int b = owner_of(part_at, s.seqs, i), rel = i - part_at[b];
    PartRec r;
    r.b = b;
    lengths(s, b, r.start, r.n, r.len);
    const int c = Span(p.a, r.len - r.n, r.len - 1).chunks, k = parts_of(p, c, q);
    const int rows = r.n * p.a.group, nb = (rows + ROWS_BLOCK - 1) / ROWS_BLOCK, each = (rows + nb - 1) / nb;
    // row blocks of a part are neighbours: they share its keys in L2
    int block = rel % nb;
    const int cut = rel / nb;
    r.head = cut / k;
    r.part = cut - r.head * k;
    if (const int n = p.a.cluster; n > 0) {  // a cluster's CTAs are the neighbours
      block = rel / n % nb;
      r.part = rel / n / nb % (k / n) * n + rel % n;
      r.head = rel / nb / k;
    }
    r.parts = k;
    r.slot0 = slot_at[b] + (r.head * nb + block) * slots_of(p, k);
    r.c0 = int(int64_t(c) * r.part / k);
    r.c1 = int(int64_t(c) * (r.part + 1) / k);
    r.row0 = block * each;
    r.rows = min(each, rows - r.row0);
    p.a.parts[i] = r;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (b0 + i < s.seqs) {
      part_at[b0 + i] = unit;
      unit += chunks[i] > 0 ? 0 : blocks[i] * H;
    }
  __syncthreads();
  // ---- units: whole or cut, then a counting sort by length, longest first ----
  const auto unit_of = [&](int i) {
    const int b = owner_of(part_at, s.seqs, i), rel = i - part_at[b];
    UnitRec r = {};
    r.b = b;
    lengths(s, b, r.start, r.n, r.len);
    r.head = rel % H;
    r.row0 = rel / H * TILE_ROWS;
    const int last = min(r.row0 + TILE_ROWS, r.n * p.a.group) - 1, first = r.len - r.n;
    r.c1 = Span(p.a, first + r.row0 / p.a.group, first + last / p.a.group).chunks;
    r.slot = -1;
    return r;
  };
  constexpr int STEPS = 256;
  __shared__ int count[STEPS], most, joins, tile_slots;
  __shared__ unsigned long long sum;
  if (tid < STEPS) count[tid] = 0;
  if (tid == 0) most = 1, joins = tile_slots = 0, sum = 0;
  __syncthreads();
  int top = 1;
  unsigned long long all_chunks = 0;
  for (int i = tid; i < n_units; i += THREADS) {
    const int c = unit_of(i).c1;
    top = max(top, c);
    all_chunks += c;
  }
  atomicMax(&most, top);
  atomicAdd(&sum, all_chunks);
  __syncthreads();
  // chunks a part
  const int limit = p.tile_target == 0 || n_units >= p.tile_target
                        ? most
                        : max(TILE_CUT, int((sum + p.tile_target - 1) / p.tile_target));
  const auto step_of = [&](int c) { return int(int64_t(most - c) * STEPS / (most + 1)); };
  const auto longest = [&](int c, int k) { return (c + k - 1) / k; };
  for (int i = tid; i < n_units; i += THREADS) {
    const int c = unit_of(i).c1, k = (c + limit - 1) / limit;
    atomicAdd(&count[step_of(longest(c, k))], k);
  }
  __syncthreads();
  int n_records;
  const int before = block_scan(tid < STEPS ? count[tid] : 0, n_records, sums);
  if (tid < STEPS) count[tid] = before;
  __syncthreads();
  for (int i = tid; i < n_units; i += THREADS) {
    UnitRec r = unit_of(i);
    const int c = r.c1, k = (c + limit - 1) / limit;
    const int at0 = atomicAdd(&count[step_of(longest(c, k))], k);
    const int slot0 = k > 1 ? atomicAdd(&tile_slots, k) : -1;
    for (int part = 0; part < k; ++part) {
      r.c0 = int(int64_t(c) * part / k);
      r.c1 = int(int64_t(c) * (part + 1) / k);
      if (k > 1) r.slot = slot0 + part;
      if (at0 + part < p.most_units) p.a.units[at0 + part] = r;
    }
    if (k > 1) {
      const int j = atomicAdd(&joins, 1);
      if (j < p.most_joins) p.a.joins[j] = JoinRec{r.head, r.row0, r.start, r.n * p.a.group, slot0, k, r.b, 0};
    }
  }
  __syncthreads();
  // the launches have room for so many (see shape_of)
  if (tid == 0)
    *p.a.plan = PlanHead{n_parts, min(n_records, p.most_units), min(joins, p.most_joins), p.a.group, p.a.window,
                         p.a.sinks, p.a.row_limit, s.seqs, H, p.a.nt, s.width, s.page_shift, p.a.cluster, {}};
}

}  // namespace

int plan_attend(const AttendParams &a, const PlanShape &shape, cudaStream_t stream) {
  PlanParams p;
  p.a = a;
  p.target = shape.target;
  p.spread = shape.spread;
  p.single = shape.single;
  // a join through the workspace costs about what ten chunks do
  p.min_chunks = shape.cluster > 0 ? 10 : 2;
  p.most_parts = int(shape.most_parts);
  p.most_units = int(shape.most_units);
  p.most_joins = int(shape.most_joins);
  p.tile_target = shape.tile_target;
  return launch_kernel("emmy_kv8_attend_plan", plan_kernel, dim3(1), THREADS, 0, stream, p);
}

}  // namespace kv8
