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
// 4096 of 1-200, 35 for six prompts of 200-1500 tokens; with shared keys 18 to 19.
#include "kv8_attend.cuh"

namespace kv8 {
namespace {

constexpr int THREADS = 1024, WARPS = 32, EACH = EMMY_KV8_MAX_SEQS / THREADS;

struct PlanParams {
  AttendParams a;
  int target, min_chunks, most_units, most_joins, tile_target;
  bool spread, single;
  int most_pre, pre_target, max_runs, max_tokens;  // of shared keys
  bool wide;                                       // heads of 128
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

__device__ __forceinline__ PlanHead head_of(const AttendParams &a, int parts, int units, int joins) {
  return PlanHead{parts, units, joins, a.group, a.window, a.sinks, a.row_limit, a.s.seqs, a.s.kv_heads,
                  a.nt, a.s.width, a.s.page_shift, a.cluster, a.shared, a.most_parts, a.units_at};
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
  n_parts = min(n_parts, p.a.most_parts);
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
    *p.a.plan = head_of(p.a, n_parts, min(n_records, p.most_units), min(joins, p.most_joins));
}

// What a run that begins at sequence b comes to: its new tokens' rows of a kv
// head and its shared keys; 0 keys where b begins none, or one that cannot be.
struct Run {
  int start, tokens, keys;
  __device__ __forceinline__ Run(const PlanParams &p, int b) : start(0), tokens(0), keys(0) {
    const Seqs &s = p.a.s;
    const int count = p.a.runs[s.seqs + b], held = p.a.runs[2 * s.seqs + b];
    if (p.a.runs[b] != b || count < 2 || held == 0) return;
    if (count > s.seqs - b || held < 0 || held % (1 << s.page_shift) != 0 || held > int64_t(s.width) << s.page_shift) {
      report(s.status, STATUS_LENGTH);
      return;
    }
    start = s.q_starts[b];
    tokens = s.q_starts[b + count] - start;
    if (start < 0 || tokens <= 0 || start > s.tokens - tokens || tokens > p.max_tokens) return;
    keys = held;
  }
};

// The plan of a call with shared keys.  A run's blocks of query rows (the tile
// kernel's units, or the row kernel's) are each cut into the same number of parts:
// their keys are the same, so blocks of a part are neighbours.  Each sequence's own
// keys are segments and parts as above.  Part `part` of row block `block` of a kv
// head leaves its result in slot slot0 + (head * parts + part) * blocks + block, so
// a row finds its results by where it stands.
__global__ void __launch_bounds__(THREADS) plan_shared_kernel(const PlanParams p) {
  __shared__ int at_of[EMMY_KV8_MAX_SEQS];
  __shared__ int sums[WARPS], longest;
  __shared__ unsigned long long run_tokens, run_work;  // of all runs
  grid_dependency_wait();
  grid_dependency_done();
  const Seqs &s = p.a.s;
  const int tid = threadIdx.x, H = s.kv_heads, b0 = tid * EACH, G = p.a.group, RB = p.a.pre_rows;
  const bool tiles = p.a.shared == SHARED_TILES;
  for (int i = tid; i < s.tokens; i += THREADS) p.a.seq_of[i] = -1;
  // ---- runs ----
  int pre_chunks[EACH], pre_blocks[EACH], pre_tokens[EACH], runs = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    pre_chunks[i] = pre_blocks[i] = pre_tokens[i] = 0;
    if (b0 + i < s.seqs) {
      const Run r(p, b0 + i);
      if (r.keys > 0) {
        pre_chunks[i] = r.keys >> 6;
        pre_blocks[i] = (r.tokens * G + RB - 1) / RB;
        pre_tokens[i] = r.tokens;
        ++runs;
      }
    }
  }
  if (tid == 0) longest = 1, run_tokens = run_work = 0;
  int all, nth = block_scan(runs, all, sums), mine;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (pre_chunks[i] > 0 && nth++ >= p.max_runs) pre_chunks[i] = pre_blocks[i] = 0;  // one more than there is room for
    if (pre_chunks[i] == 0) continue;
    atomicMax(&longest, pre_chunks[i]);
    atomicAdd(&run_tokens, static_cast<unsigned long long>(pre_tokens[i]));
    atomicAdd(&run_work, static_cast<unsigned long long>(pre_chunks[i]) * pre_blocks[i]);
  }
  __syncthreads();
  // runs that overlap: there may not be room for so many blocks of rows, so all
  // sequences are left to themselves
  const bool overlap = run_tokens > static_cast<unsigned long long>(s.tokens);
  const int64_t pre_work = overlap ? 0 : static_cast<int64_t>(run_work);
  if (overlap) {
    if (tid == 0) report(s.status, STATUS_LENGTH);
#pragma unroll
    for (int i = 0; i < EACH; ++i) pre_chunks[i] = pre_blocks[i] = 0;
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (b0 + i < s.seqs) p.a.results[b0 + i] = ResultRec{pre_chunks[i], 0, 0, pre_blocks[i], 0, 0, 0, 1, 0, 0, {}};
  __syncthreads();
  // ---- each sequence's own keys ----
  int chunks[EACH], blocks[EACH], first[EACH], tokens[EACH];  // blocks: of rows
  mine = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    chunks[i] = blocks[i] = first[i] = tokens[i] = 0;
    const int b = b0 + i;
    if (b < s.seqs) {
      int start, n, len;
      lengths(s, b, start, n, len);
      const int lead = p.a.runs[b];
      int shared = 0;
      // a run that cannot be, or not here, leaves its sequences to themselves
      if (lead >= 0 && lead <= b && p.a.runs[lead] == lead && b - lead < max(p.a.runs[s.seqs + lead], 1)) {
        const Run r(p, lead);
        shared = p.a.results[lead].chunks;
        // new tokens among the shared keys, or rows that are not the run's
        if (shared > 0 && n > 0 && (shared << 6 > len - n || start < r.start || start + n > r.start + r.tokens)) {
          report(s.status, STATUS_LENGTH);
          n = 0;
        }
      }
      if (n > 0) {
        chunks[i] = Span(p.a, len - n, len - 1).chunks - shared;
        blocks[i] = (n * G + ROWS_BLOCK - 1) / ROWS_BLOCK;
        first[i] = start, tokens[i] = n;
        for (int t = 0; t < n; ++t) p.a.seq_of[start + t] = b;
      }
    }
    mine += chunks[i] * blocks[i];
  }
  int own_work;
  block_scan(mine, own_work, sums);
  // ---- chunks of a part of shared keys ----
  // Row kernel: as many as leave one wave of parts, if any of some tries do.  Tile
  // kernel: those for which this ends first: a block takes FIXED us before its first
  // product and after its last one, and CHUNK a chunk; it runs beside the row kernel,
  // whose chunks of own keys take OWN us of an SM each; and a result costs RESULT us
  // to write and join (all timed inside the kernels).  64 sequences behind 8192 keys:
  // 128 blocks of 8 chunks, the most that fit, 53 us, 64 of 16, as this picks, 41.
  int limit = longest;
  float best = 0.0f;
  if (p.pre_target > 0) {
    const int64_t share = (pre_work * H + p.pre_target - 1) / p.pre_target;
    const int l0 = max(int(min(share, int64_t(1) << 24)), tiles ? TILE_CUT : 2);
    const float FIXED = p.wide ? 10.0f : 7.0f, CHUNK = p.wide ? 1.03f : 0.88f, OWN = 0.46f, RESULT = p.wide ? 0.053f : 0.027f;
    // parts for l0 chunks, and for an eighth more each time
    constexpr int TRIES = 16;
    __shared__ int parts_for[TRIES];
    if (tid < TRIES) parts_for[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (pre_chunks[i] > 0)
        for (int t = 0, tried = l0; t < TRIES; ++t, tried += max(1, tried >> 3))
          atomicAdd(&parts_for[t], pre_blocks[i] * ((pre_chunks[i] + tried - 1) / tried));
    __syncthreads();
    limit = 0;
    for (int t = 0, tried = l0; t < TRIES; ++t, tried += max(1, tried >> 3)) {
      const float n = float(parts_for[t]) * H, tile = FIXED + CHUNK * tried;
      if (n > p.pre_target && t < TRIES - 1) continue;
      const float ends = fmaxf(tile, (n * tile + OWN * own_work * H) / p.pre_target) + RESULT * n;
      if (limit == 0 || (tiles && ends < best)) limit = tried, best = ends;
    }
  }
  int pre = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) pre += pre_blocks[i] * H * ((pre_chunks[i] + limit - 1) / limit);
  int n_pre, pre_at = block_scan(pre, n_pre, sums);
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (b0 + i < s.seqs) {
      const int k = (pre_chunks[i] + limit - 1) / limit;
      at_of[b0 + i] = pre_at;
      p.a.results[b0 + i].slot0 = pre_at;
      p.a.results[b0 + i].parts = k;
      pre_at += pre_blocks[i] * H * k;
    }
  __syncthreads();
  n_pre = min(n_pre, p.most_pre);
  for (int i = tid; i < n_pre; i += THREADS) {
    const int b = owner_of(at_of, s.seqs, i), rel = i - at_of[b];
    const ResultRec f = p.a.results[b];
    const Run r(p, b);
    const int block = rel % f.blocks, part = rel / f.blocks % f.parts, head = rel / (f.blocks * f.parts);
    const int c0 = int(int64_t(f.chunks) * part / f.parts), c1 = int(int64_t(f.chunks) * (part + 1) / f.parts);
    // its tokens as if they came behind the shared keys
    if (tiles)
      p.a.units[i] = UnitRec{b, head, block * RB, r.start, r.tokens, r.keys + r.tokens, c0, c1, i, {}};
    else
      p.a.parts[i] = PartRec{b, head, c0, c1, part, f.parts, i, block * RB,
                             r.start, r.tokens, r.keys + r.tokens, min(RB, r.tokens * G - block * RB)};
  }
  // ---- parts of own keys ----
  const int first_part = tiles ? 0 : n_pre;
  const int64_t share = (int64_t(own_work) * H + p.target - 1) / p.target;
  // chunks of a part at most: their share; more, as the start of a block costs what three
  // chunks do, up to two fifths of the time that the shared keys take by the estimate
  // above (a chunk takes a block 1.4 us beside two others: best / 1.4 * 2 / 5), as the
  // last blocks should not take long.  The estimate is the tile kernel's for runs of the
  // row kernel, too; with their share and min_chunks alone: 8 runs of 4 behind 4096 keys
  // 31.0 -> 29.5 us, 2 of 8 behind 8192 27.8 -> 26.1, but 32 of 2 with 2 tokens 50.3 ->
  // 54.3.  Where shared keys are not cut there is no estimate, and it is 0.
  const int q = max(max(p.min_chunks, int(best / 3.5f)), int(min(share, int64_t(1) << 24)));
  int parts = 0, n_parts;
#pragma unroll
  for (int i = 0; i < EACH; ++i) parts += (chunks[i] + q - 1) / q * blocks[i] * H;
  int at = block_scan(parts, n_parts, sums);
  __syncthreads();  // at_of is read above
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (b0 + i < s.seqs) {
      const int b = b0 + i, k = (chunks[i] + q - 1) / q, lead = p.a.runs[b];
      at_of[b] = at;
      ResultRec f = {0, 0, 0, 1, 0, first_part + at, k, max(blocks[i], 1), first[i], tokens[i], {}};
      if (chunks[i] > 0 && lead >= 0 && lead <= b && p.a.runs[lead] == lead && b - lead < max(p.a.runs[s.seqs + lead], 1)) {
        const ResultRec of = p.a.results[lead];  // (others write only what comes behind `row`)
        f.chunks = of.chunks, f.slot0 = of.slot0, f.parts = of.parts, f.blocks = max(of.blocks, 1);
        f.row = (s.q_starts[b] - s.q_starts[lead]) * G;
      }
      at += k * blocks[i] * H;
      if (lead == b) {
        p.a.results[b].own_slot0 = f.own_slot0;
        p.a.results[b].own_parts = k;
        p.a.results[b].own_blocks = f.own_blocks;
        p.a.results[b].start = f.start;
        p.a.results[b].n = f.n;
      } else {
        p.a.results[b] = f;
      }
    }
  __syncthreads();
  n_parts = min(n_parts, p.a.most_parts - first_part);
  const auto part_of = [&](int i) {
    const int b = owner_of(at_of, s.seqs, i), rel = i - at_of[b];
    const ResultRec f = p.a.results[b];
    PartRec r;
    r.b = b;
    lengths(s, b, r.start, r.n, r.len);
    const int c = Span(p.a, r.len - r.n, r.len - 1).chunks - f.chunks, k = f.own_parts, nb = f.own_blocks;
    const int rows = r.n * G, each = (rows + nb - 1) / nb;
    const int block = rel % nb, cut = rel / nb;
    r.head = cut / k;
    r.part = cut - r.head * k;
    r.parts = k;
    r.slot0 = first_part + i;
    r.c0 = f.chunks + int(int64_t(c) * r.part / k);
    r.c1 = f.chunks + int(int64_t(c) * (r.part + 1) / k);
    r.row0 = block * each;
    r.rows = min(each, rows - r.row0);
    return r;
  };
  // the longest first, so that the last ones to start are short (by 256 steps of q;
  // 33 sequences with four drafts, three of them of 4100-4800 own keys: 28 -> 25 us)
  constexpr int STEPS = 256;
  __shared__ int count[STEPS];
  if (tid < STEPS) count[tid] = 0;
  __syncthreads();
  const auto step_of = [&](const PartRec &r) { return int(int64_t(max(q - (r.c1 - r.c0), 0)) * (STEPS - 1) / q); };
  for (int i = tid; i < n_parts; i += THREADS) atomicAdd(&count[step_of(part_of(i))], 1);
  __syncthreads();
  int n_records;
  const int before = block_scan(tid < STEPS ? count[tid] : 0, n_records, sums);
  if (tid < STEPS) count[tid] = before;
  __syncthreads();
  for (int i = tid; i < n_parts; i += THREADS) {
    const PartRec r = part_of(i);
    p.a.parts[first_part + atomicAdd(&count[step_of(r)], 1)] = r;
  }
  if (tid == 0)
    *p.a.plan = head_of(p.a, first_part + n_parts, tiles ? n_pre : 0, s.tokens);
}

PlanParams params_of(const AttendParams &a, const PlanShape &shape) {
  PlanParams p;
  p.a = a;
  p.target = shape.target;
  p.spread = shape.spread;
  p.single = shape.single;
  // a join through the workspace costs about what ten chunks do
  p.min_chunks = shape.cluster > 0 ? 10 : shape.shared == SHARED_TILES ? 8 : shape.shared == SHARED_ROWS ? 4 : 2;
  p.most_units = int(shape.most_units);
  p.most_joins = int(shape.most_joins);
  p.tile_target = shape.tile_target;
  p.most_pre = int(shape.most_pre);
  p.pre_target = shape.pre_target;
  p.max_runs = shape.max_runs;
  p.max_tokens = shape.max_tokens;
  p.wide = shape.wide;
  return p;
}

}  // namespace

int plan_attend(const AttendParams &a, const PlanShape &shape, cudaStream_t stream) {
  return launch_kernel("emmy_kv8_attend_plan", plan_kernel, dim3(1), THREADS, 0, stream, params_of(a, shape));
}
int plan_shared(const AttendParams &a, const PlanShape &shape, cudaStream_t stream) {
  return launch_kernel("emmy_kv8_attend_shared_plan", plan_shared_kernel, dim3(1), THREADS, 0, stream, params_of(a, shape));
}

}  // namespace kv8
