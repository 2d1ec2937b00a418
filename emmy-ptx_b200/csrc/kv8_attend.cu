// emmy_kv8_attend -- attention of new queries over the paged 8-bit cache:
// checks, workspace and plan, and which kernel takes which sequences.
#include <cmath>
#include <numeric>

#include "kv8_attend.cuh"

namespace kv8 {
namespace {

// A sequence with up to ROWS_MOST rows of a kv head is the row kernel's, others
// the tile kernel's; a call's only sequence is whichever's its most rows ask
// for.
int shape_of(const char *what, const emmy_kv8 *c, int heads, PlanShape &p) {
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

// The checks that attend and its plan share.
int check_args(const char *what, const emmy_kv8 *cache, const emmy_kv8_attend_args *a, PlanShape &shape, AttendParams &p) {
  int rc = check_cache(what, cache);
  if (rc == EMMY_OK) rc = check_seqs(what, cache);
  if (rc != EMMY_OK) return rc;
  if (a == nullptr) return fail(EMMY_EINVAL, what, "null arguments");
  rc = shape_of(what, cache, a->heads, shape);
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
  return EMMY_OK;
}

}  // namespace
}  // namespace kv8

extern "C" int emmy_kv8_attend_sizes(const emmy_kv8 *cache, int32_t heads, uint64_t *workspace_bytes,
                                     uint64_t *plan_bytes) {
  using namespace kv8;
  static const char *what = "emmy_kv8_attend_sizes";
  int rc = check_cache(what, cache);
  if (rc == EMMY_OK) rc = check_counts(what, cache);
  if (rc == EMMY_OK && (workspace_bytes == nullptr || plan_bytes == nullptr))
    rc = fail(EMMY_EINVAL, what, "null result");
  PlanShape shape;
  if (rc == EMMY_OK) rc = shape_of(what, cache, heads, shape);
  if (rc != EMMY_OK) return rc;
  *workspace_bytes = shape.workspace_bytes;
  *plan_bytes = shape.plan_bytes;
  return EMMY_OK;
}

extern "C" int emmy_kv8_attend_plan(const emmy_kv8 *cache, const emmy_kv8_attend_args *a, emmy_stream stream) {
  using namespace kv8;
  static const char *what = "emmy_kv8_attend_plan";
  PlanShape shape;
  AttendParams p;
  const int rc = check_args(what, cache, a, shape, p);
  if (rc != EMMY_OK) return rc;
  const OnDevice on(cache->device);
  if (on.err != cudaSuccess) return cuda_fail(what, on.err);
  return plan_attend(p, shape, static_cast<cudaStream_t>(stream));
}

extern "C" int emmy_kv8_attend(const emmy_kv8 *cache, const emmy_kv8_attend_args *a, emmy_stream stream) {
  using namespace kv8;
  static const char *what = "emmy_kv8_attend";
  PlanShape shape;
  AttendParams p;
  int rc = check_args(what, cache, a, shape, p);
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
  if (a->q_strides[0] < 0 || a->q_strides[1] < 0 || a->out_strides[0] < 0 || a->out_strides[1] < 0)
    return fail(EMMY_EINVAL, what, "q and out: strides must not be negative");
  // rows of out one after another, tokens within heads or heads within tokens
  const int64_t ts = a->out_strides[0], hs = a->out_strides[1], D = cache->head_dim;
  const int64_t T = cache->tokens, Hq = a->heads;
  if ((T > 1 && ts < D) || (Hq > 1 && hs < D) || (T > 1 && Hq > 1 && (ts <= hs ? hs < ts * (T - 1) + D : ts < hs * (Hq - 1) + D)))
    return fail(EMMY_EINVAL, what, "rows of out overlap");
  const auto extent = [&](const int64_t st[2]) {
    return uint64_t((cache->tokens - 1) * st[0] + (a->heads - 1) * st[1] + cache->head_dim) * 2;
  };
  // rows of q and out in turn, as slices of one wider array are: of heads, of
  // tokens where heads come first, or of elements
  const auto in_turn = [&](int64_t step_q, int64_t step_out, int64_t wide_q, int64_t wide_out) {
    if (step_q != step_out || step_q == 0) return false;
    const int64_t by = int64_t(a->out - a->q) / 2 % step_q, off = by < 0 ? by + step_q : by;
    return off >= wide_q && off + wide_out <= step_q;
  };
  if (overlap(a->q, extent(a->q_strides), a->out, extent(a->out_strides))) {
    const int64_t qt = a->q_strides[0], qh = a->q_strides[1], step = std::gcd(std::gcd(qt, qh), std::gcd(ts, hs));
    if (!in_turn(qt, ts, (Hq - 1) * qh + D, (Hq - 1) * hs + D) && !in_turn(qh, hs, (T - 1) * qt + D, (T - 1) * ts + D) &&
        !in_turn(step, step, D, D))
      return fail(EMMY_EINVAL, what, "q and out overlap");
  }
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
  p.beside = shape.tiles && shape.rows;
  p.ready = p.counters + EMMY_KV8_WORKSPACE_ZERO / 4 - 2;
  if (shape.tiles) rc = tiles_attend(p, *cache, shape, bf16, st);
  if (rc == EMMY_OK && shape.rows) {
    rc = rows_attend(p, *cache, shape, bf16, st);
    if (rc != EMMY_OK && p.beside) cudaMemsetAsync(p.ready, 0, 8, st);  // nobody else will
  }
  if (rc == EMMY_OK && shape.tile_target > 0) rc = tiles_join(p, *cache, shape, bf16, st);
  return rc;
}
