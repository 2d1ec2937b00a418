// emmy_kv8_attend -- attention of new queries over the paged 8-bit cache:
// checks, workspace and plan, and which kernel takes which sequences.
#include <algorithm>
#include <cmath>

#include "kv8_attend.cuh"

namespace kv8 {
namespace {

// A sequence with up to ROWS_MOST rows of a kv head is the row kernel's, others
// the tile kernel's; a call's only sequence is whichever's its most rows ask
// for.
int shape_of(const char *what, const emmy_kv8 *c, int heads, PlanShape &p) {
  p = PlanShape{};
  if (heads < 1 || heads % c->kv_heads != 0)
    return fail(EMMY_EINVAL, what, "heads must be a positive multiple of kv_heads");
  if (int64_t(heads) * c->tokens > 0x7fffffff) return fail(EMMY_EINVAL, what, "too many query rows");
  if (int64_t(c->pages) * 2 * c->kv_heads * c->page_size > 0x7fffffff)
    return fail(EMMY_EINVAL, what, "a layer holds at most 2^31 - 1 rows of head_dim codes");
  const int sms = sm_count(c->device);
  if (sms == 0) return fail(EMMY_ECUDART, what, "cannot read the device's SM count");
  const int64_t group = heads / c->kv_heads, most = group * c->max_q;
  p.tiles = most > ROWS_MOST;
  p.rows = !p.tiles || c->seqs > 1;
  const int64_t few = most < ROWS_MOST ? most : ROWS_MOST;
  p.nt = rows_blocks(few);
  const int64_t segments = int64_t(c->seqs) * c->kv_heads * ((few + ROWS_BLOCK - 1) / ROWS_BLOCK);
  const int wave = sms * ROWS_PER_SM;
  p.spread = segments > wave;
  // Workspace slots, two counters each, but the last two of the zeros are
  // AttendParams::ready.  Two waves: a cut segment has c >= 1.5 q
  // chunks and at most c / q + 1/2 parts, a third above its share.
  const int fit = EMMY_KV8_WORKSPACE_ZERO / 8 - 1;
  p.slots = 3 * wave < fit ? 3 * wave : fit;
  p.target = p.spread ? p.slots * 2 / 3 : wave < p.slots ? wave : p.slots;
  // The parts wanted, or, where no try fitted, one of each segment more; but
  // no more than chunks that the table could hold.
  p.most_parts = (p.spread ? p.slots : p.target) + segments;
  const int64_t chunks = int64_t(c->table_width) * c->page_size / 64 * segments;
  if (chunks < p.most_parts) p.most_parts = chunks;
  if (!p.rows) p.most_parts = 0;
  // Short segments as clusters of 8, 4 or 2 CTAs that join in shared memory.  In
  // cycles, at about 700 a chunk: parts of a cluster and its join take cap / n
  // chunks and 1500, parts that fill the GPU and their join through L2
  // segments * cap / wave chunks and 8000.
  p.cluster = 0;
  p.single = false;
  const int64_t cap = int64_t(c->table_width) * c->page_size / 64;
  for (int n = 8; n >= 2 && p.cluster == 0 && p.rows; n /= 2)
    if (segments * n <= wave && cap >= n && 7 * cap * (wave - segments * n) < 65 * n * wave) p.cluster = n, p.single = true;
  if (p.single) p.most_parts = segments * p.cluster;
  // A few long ones as some clusters of 4 each, of which nine tenths of a wave
  // fit on the GPU's processing clusters (2 sequences of 131071 keys: 35.5 ->
  // 34.0 us against single CTAs).
  if (!p.single && p.rows && segments * 8 <= wave) {
    p.cluster = 4;
    p.target = wave * 9 / 10 / 4 * 4;
    p.most_parts = p.target + segments * 4;
  }
  // Units: at most one part-filled one of a sequence.  Fewer than SMs may be
  // cut, into at most one more part each than their share of the SMs, where
  // the table can hold more chunks than are worth a join (a prompt of 200
  // tokens without its empty launch: 16.0 -> 14.3 us).
  const int64_t units = p.tiles ? (c->tokens * group / TILE_ROWS + c->seqs) * c->kv_heads : 0;
  p.tile_target = units > 0 && units < sms && cap > TILE_CUT ? sms : 0;
  p.most_units = units + p.tile_target;
  p.most_joins = p.tile_target > 0 ? units : 0;
  // the plan counts chunks in 32 bits
  if (p.most_units > 0x7fffffff || segments > (1 << 24) || chunks / c->kv_heads > (1 << 30))
    return fail(EMMY_EINVAL, what, "too many sequences and heads for one call");
  p.partial_bytes = uint64_t(p.slots) * 8 * p.nt * (c->head_dim + 2) * 4;
  p.workspace_bytes = EMMY_KV8_WORKSPACE_ZERO + p.partial_bytes +
                      (p.tile_target > 0 ? uint64_t(p.most_units) * TILE_ROWS * (c->head_dim + 2) * 4 : 0);
  // kernels read the record of their index before they know how many there are
  p.plan_bytes = sizeof(PlanHead) + uint64_t(p.most_parts) * sizeof(PartRec) +
                 uint64_t(p.most_units) * sizeof(UnitRec) + uint64_t(p.most_joins) * sizeof(JoinRec);
  return EMMY_OK;
}

// A call with shared keys: the runs' rows over those, by the row kernel where no run
// has more than ROWS_MOST of a kv head, else by the tile kernel, and beside it each
// sequence's own keys by the row kernel; every part leaves a result, and a kernel
// joins them.  Longer sequences' rows fill tiles by themselves, and a window leaves
// few shared keys: those calls are as without sharing.  Measured, us: the own keys'
// kernel after the shared keys', its last blocks taking the results in: 64 sequences
// behind 8192 keys 60, 128 behind 32768 78 (d = 128); side by side with a join 40, 62.
// Every segment has a slot for its result, whatever its sequence shares: 4 KB for 8 rows
// of 128, so 1024 sequences of 8 kv heads take 40 MB and 4096 142 MB, unshared calls 5.5.
// Shared keys of as many units as there are SMs, or more, are not cut and not sorted.
int shape_shared(const char *what, const emmy_kv8 *c, const emmy_kv8_shared *sh, int heads, int window, PlanShape &p) {
  const int rc = shape_of(what, c, heads, p);
  if (rc != EMMY_OK) return rc;
  if (p.tiles || window > 0 || sh->max_runs == 0 || sh->max_tokens == 0) return EMMY_OK;
  const int sms = sm_count(c->device);
  const int64_t group = heads / c->kv_heads, few = group * c->max_q, run_rows = group * sh->max_tokens;
  const int64_t segments = int64_t(c->seqs) * c->kv_heads * ((few + ROWS_BLOCK - 1) / ROWS_BLOCK);
  const int64_t cap = int64_t(c->table_width) * c->page_size / 64;
  const int wave = sms * ROWS_PER_SM;
  p.max_runs = sh->max_runs, p.max_tokens = sh->max_tokens;
  p.wide = c->head_dim == 128;
  p.cluster = 0, p.single = false;
  int64_t units;
  if (run_rows <= ROWS_MOST) {
    p.shared = SHARED_ROWS;
    p.nt = std::max(p.nt, rows_blocks(run_rows));
    p.pre_rows = 8 * p.nt;
    units = int64_t(p.max_runs) * ((run_rows + p.pre_rows - 1) / p.pre_rows) * c->kv_heads;
    p.pre_target = units < wave ? wave : 0;
  } else {
    p.shared = SHARED_TILES;
    p.pre_rows = TILE_ROWS;
    units = (c->tokens * group / TILE_ROWS + p.max_runs) * c->kv_heads;
    p.pre_target = units < sms ? sms : 0;
  }
  p.most_pre = units + p.pre_target;
  // (more segments than blocks that fit: thirds of a block's share even out, 4
  // sequences behind 4096 shared keys beside 60 of 4100-4700 keys 132 -> 107 us)
  p.target = p.spread ? 3 * wave : p.shared == SHARED_TILES ? 2 * wave : wave;
  p.most_parts = std::min(p.target + segments, cap * segments) + (p.shared == SHARED_ROWS ? p.most_pre : 0);
  if (p.most_pre > 0x7fffffff || p.most_parts > 0x7fffffff) return fail(EMMY_EINVAL, what, "too many sequences and heads for one call");
  if (p.shared == SHARED_TILES) p.most_units = p.most_pre;
  p.partial_bytes = uint64_t(p.most_parts) * 8 * p.nt * (c->head_dim + 2) * 4;
  p.workspace_bytes = EMMY_KV8_WORKSPACE_ZERO + p.partial_bytes +
                      uint64_t(p.most_units) * p.pre_rows * (c->head_dim + 2) * 4;
  p.plan_bytes = sizeof(PlanHead) + uint64_t(p.most_parts) * sizeof(PartRec) + uint64_t(p.most_units) * sizeof(UnitRec) +
                 uint64_t(c->seqs) * sizeof(ResultRec) + uint64_t(c->tokens) * 4;
  return EMMY_OK;
}

int check_shared(const char *what, const emmy_kv8 *c, const emmy_kv8_shared *sh) {
  if (sh == nullptr) return fail(EMMY_EINVAL, what, "null description of what is shared");
  if (sh->max_runs < 0 || sh->max_runs > c->seqs || sh->max_tokens < 0 || sh->max_tokens > c->tokens)
    return fail(EMMY_EINVAL, what, "bad max_runs or max_tokens");
  return EMMY_OK;
}

// The checks that attend and its plan share.
int check_args(const char *what, const emmy_kv8 *cache, const emmy_kv8_shared *shared, const emmy_kv8_attend_args *a,
               PlanShape &shape, AttendParams &p) {
  int rc = check_cache(what, cache);
  if (rc == EMMY_OK) rc = check_seqs(what, cache);
  if (rc != EMMY_OK) return rc;
  if (a == nullptr) return fail(EMMY_EINVAL, what, "null arguments");
  rc = shared == nullptr ? shape_of(what, cache, a->heads, shape) : shape_shared(what, cache, shared, a->heads, a->window, shape);
  if (rc != EMMY_OK) return rc;
  if (a->window < 0 || a->sinks < 0) return fail(EMMY_EINVAL, what, "window and sinks must not be negative");
  if (a->sinks > 0 && a->window == 0) return fail(EMMY_EINVAL, what, "sinks need a window");
  if (a->plan == 0 || a->plan % 16 || a->plan_bytes < shape.plan_bytes)
    return fail(EMMY_EINVAL, what, "plan is missing, unaligned or too small");
  p = AttendParams{};
  p.s = seqs_of(*cache);
  p.codes = reinterpret_cast<const uint8_t *>(cache->codes);
  p.exps = reinterpret_cast<const int8_t *>(cache->exps);
  p.plan = reinterpret_cast<PlanHead *>(a->plan);
  p.parts = reinterpret_cast<PartRec *>(p.plan + 1);
  p.units = reinterpret_cast<UnitRec *>(p.parts + shape.most_parts);
  p.joins = reinterpret_cast<JoinRec *>(p.units + shape.most_units);
  p.group = a->heads / cache->kv_heads;
  // a sequence holds at most 2^30 keys; sums with more would overflow
  p.window = a->window < 1 << 30 ? a->window : 1 << 30;
  p.sinks = a->sinks < 1 << 30 ? a->sinks : 1 << 30;
  p.row_limit = shape.rows ? ROWS_MOST : 0;
  p.nt = shape.nt;
  p.cluster = shape.cluster;
  p.most_parts = int(shape.most_parts);
  p.units_at = 2 * unsigned(shape.most_units) + (shape.tile_target > 0);  // at most 2^31 - 1 units
  p.shared = shape.shared;
  if (shape.shared != SHARED_NONE) {
    if (shared->runs == 0 || shared->runs % 4) return fail(EMMY_EINVAL, what, "runs is missing or unaligned");
    p.runs = reinterpret_cast<const int *>(shared->runs);
    p.results = reinterpret_cast<ResultRec *>(p.units + shape.most_units);
    p.seq_of = reinterpret_cast<int *>(p.results + cache->seqs);
    p.pre_rows = shape.pre_rows;
  }
  return EMMY_OK;
}

int sizes(const char *what, const emmy_kv8 *cache, const emmy_kv8_shared *shared, int32_t heads, uint64_t *workspace_bytes,
          uint64_t *plan_bytes) {
  int rc = check_cache(what, cache);
  if (rc == EMMY_OK) rc = check_counts(what, cache);
  if (rc == EMMY_OK && (workspace_bytes == nullptr || plan_bytes == nullptr))
    rc = fail(EMMY_EINVAL, what, "null result");
  PlanShape shape;
  if (rc == EMMY_OK) rc = shape_of(what, cache, heads, shape);
  if (rc != EMMY_OK) return rc;
  *workspace_bytes = shape.workspace_bytes;
  *plan_bytes = shape.plan_bytes;
  if (shared == nullptr) return EMMY_OK;
  // with a window the call is as without sharing, so the larger ones
  rc = shape_shared(what, cache, shared, heads, 0, shape);
  if (rc != EMMY_OK) return rc;
  *workspace_bytes = std::max(*workspace_bytes, shape.workspace_bytes);
  *plan_bytes = std::max(*plan_bytes, shape.plan_bytes);
  return EMMY_OK;
}

int plan(const char *what, const emmy_kv8 *cache, const emmy_kv8_shared *shared, const emmy_kv8_attend_args *a, emmy_stream stream) {
  PlanShape shape;
  AttendParams p;
  const int rc = check_args(what, cache, shared, a, shape, p);
  if (rc != EMMY_OK) return rc;
  const OnDevice on(cache->device);
  if (on.err != cudaSuccess) return cuda_fail(what, on.err);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return shape.shared != SHARED_NONE ? plan_shared(p, shape, st) : plan_attend(p, shape, st);
}

int attend(const char *what, const emmy_kv8 *cache, const emmy_kv8_shared *shared, const emmy_kv8_attend_args *a,
           emmy_stream stream) {
  PlanShape shape;
  AttendParams p;
  int rc = check_args(what, cache, shared, a, shape, p);
  if (rc != EMMY_OK) return rc;
  if (a->dtype != EMMY_KV8_BF16 && a->dtype != EMMY_KV8_F16)
    return fail(EMMY_EINVAL, what, "dtype must be bf16 or f16");
  const float scale_log2 = a->scale * 1.4426950408889634f;
  if (!std::isfinite(scale_log2)) return fail(EMMY_EINVAL, what, "scale must be finite, times log2(e) too");
  if (cache->tokens == 0 || cache->max_q == 0) return EMMY_OK;
  if (a->q == 0 || a->out == 0) return fail(EMMY_EINVAL, what, "null q or out");
  if (a->q % 16 || a->out % 16 || a->q_strides[0] % 8 || a->q_strides[1] % 8 || a->out_strides[0] % 8 ||
      a->out_strides[1] % 8)
    return fail(EMMY_EINVAL, what, "q and out: base and strides must be multiples of 16 bytes");
  const int bad = rows_trouble(a->q, a->q_strides, a->heads, 2, a->out, a->out_strides, a->heads, 2, cache->tokens,
                               cache->head_dim, false);
  if (bad != ROWS_FINE)
    return fail(EMMY_EINVAL, what, bad == ROWS_NEGATIVE ? "q and out: strides must not be negative"
                                   : bad == ROWS_SELF   ? "rows of out overlap"
                                                        : "q and out overlap");
  if (a->workspace == 0 || a->workspace % 16 || a->workspace_bytes < shape.workspace_bytes)
    return fail(EMMY_EINVAL, what, "workspace is missing, unaligned or too small");
  p.q = reinterpret_cast<const void *>(a->q);
  p.out = reinterpret_cast<void *>(a->out);
  p.q_ts = a->q_strides[0], p.q_hs = a->q_strides[1];
  p.o_ts = a->out_strides[0], p.o_hs = a->out_strides[1];
  p.counters = reinterpret_cast<unsigned *>(a->workspace);
  p.partial = reinterpret_cast<float *>(a->workspace + EMMY_KV8_WORKSPACE_ZERO);
  p.tile_partial = reinterpret_cast<float *>(a->workspace + EMMY_KV8_WORKSPACE_ZERO + shape.partial_bytes);
  p.scale_log2 = scale_log2;
  wait_limit(p.wait_ns, p.stall);
  const OnDevice on(cache->device);
  if (on.err != cudaSuccess) return cuda_fail(what, on.err);
  const bool bf16 = a->dtype == EMMY_KV8_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  note_capture(st);
  const bool tiles = shape.tiles || shape.shared == SHARED_TILES;
  p.beside = tiles && shape.rows;
  p.ready = p.counters + EMMY_KV8_WORKSPACE_ZERO / 4 - 2;
  if (tiles) rc = tiles_attend(p, *cache, shape, bf16, st);
  if (rc == EMMY_OK && shape.rows) {
    rc = rows_attend(p, *cache, shape, bf16, st);
    if (rc != EMMY_OK && p.beside) cudaMemsetAsync(p.ready, 0, 8, st);  // nobody else will
  }
  if (rc == EMMY_OK && shape.tile_target > 0) rc = tiles_join(p, *cache, shape, bf16, st);
  if (rc == EMMY_OK && shape.shared != SHARED_NONE) rc = shared_join(p, *cache, bf16, st);
  return rc;
}

}  // namespace
}  // namespace kv8

extern "C" int emmy_kv8_attend_sizes(const emmy_kv8 *cache, int32_t heads, uint64_t *workspace_bytes,
                                     uint64_t *plan_bytes) {
  return kv8::sizes("emmy_kv8_attend_sizes", cache, nullptr, heads, workspace_bytes, plan_bytes);
}

extern "C" int emmy_kv8_attend_plan(const emmy_kv8 *cache, const emmy_kv8_attend_args *a, emmy_stream stream) {
  return kv8::plan("emmy_kv8_attend_plan", cache, nullptr, a, stream);
}

extern "C" int emmy_kv8_attend(const emmy_kv8 *cache, const emmy_kv8_attend_args *a, emmy_stream stream) {
  return kv8::attend("emmy_kv8_attend", cache, nullptr, a, stream);
}

extern "C" int emmy_kv8_attend_shared_sizes(const emmy_kv8 *cache, const emmy_kv8_shared *shared, int32_t heads,
                                            uint64_t *workspace_bytes, uint64_t *plan_bytes) {
  static const char *what = "emmy_kv8_attend_shared_sizes";
  int rc = kv8::check_cache(what, cache);
  if (rc == EMMY_OK) rc = kv8::check_shared(what, cache, shared);
  return rc != EMMY_OK ? rc : kv8::sizes(what, cache, shared, heads, workspace_bytes, plan_bytes);
}

extern "C" int emmy_kv8_attend_shared_plan(const emmy_kv8 *cache, const emmy_kv8_shared *shared,
                                           const emmy_kv8_attend_args *a, emmy_stream stream) {
  static const char *what = "emmy_kv8_attend_shared_plan";
  int rc = kv8::check_cache(what, cache);
  if (rc == EMMY_OK) rc = kv8::check_shared(what, cache, shared);
  return rc != EMMY_OK ? rc : kv8::plan(what, cache, shared, a, stream);
}

extern "C" int emmy_kv8_attend_shared(const emmy_kv8 *cache, const emmy_kv8_shared *shared,
                                      const emmy_kv8_attend_args *a, emmy_stream stream) {
  static const char *what = "emmy_kv8_attend_shared";
  int rc = kv8::check_cache(what, cache);
  if (rc == EMMY_OK) rc = kv8::check_shared(what, cache, shared);
  return rc != EMMY_OK ? rc : kv8::attend(what, cache, shared, a, stream);
}
