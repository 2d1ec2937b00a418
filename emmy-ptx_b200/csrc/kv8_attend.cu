// emmy_kv8_attend -- attention of new queries over the paged 8-bit cache:
// checks, workspace, and which kernel takes which sequences.
#include <cmath>

#include "kv8_attend.cuh"

namespace kv8 {
namespace {

const char *const WHAT = "emmy_kv8_attend";

int check_heads(const char *what, const emmy_kv8 *c, int heads) {
  if (heads < 1 || heads % c->kv_heads != 0)
    return fail(EMMY_EINVAL, what, "heads must be a positive multiple of kv_heads");
  if (int64_t(heads) * c->tokens > 0x7fffffff) return fail(EMMY_EINVAL, what, "too many query rows");
  return EMMY_OK;
}

}  // namespace
}  // namespace kv8

extern "C" int emmy_kv8_attend_workspace(const emmy_kv8 *cache, int32_t heads, uint64_t *bytes) {
  using namespace kv8;
  static const char *what = "emmy_kv8_attend_workspace";
  int rc = check_cache(what, cache);
  if (rc == EMMY_OK && bytes == nullptr) rc = fail(EMMY_EINVAL, what, "null result");
  if (rc == EMMY_OK) rc = check_heads(what, cache, heads);
  if (rc != EMMY_OK) return rc;
  if (sm_count(cache->device) == 0) return fail(EMMY_ECUDART, what, "cannot read the device's SM count");
  const int64_t rows = int64_t(heads / cache->kv_heads) * cache->max_q;
  const int nt = rows_blocks(rows < ROWS_MOST ? rows : ROWS_MOST);
  *bytes = EMMY_KV8_WORKSPACE_ZERO + rows_partial_bytes(nt, cache->head_dim, cache->device);
  return EMMY_OK;
}

extern "C" int emmy_kv8_attend(const emmy_kv8 *cache, const emmy_kv8_attend_args *a, emmy_stream stream) {
  using namespace kv8;
  int rc = check_cache(WHAT, cache);
  if (rc == EMMY_OK) rc = check_seqs(WHAT, cache);
  if (rc != EMMY_OK) return rc;
  if (a == nullptr) return fail(EMMY_EINVAL, WHAT, "null arguments");
  rc = check_heads(WHAT, cache, a->heads);
  if (rc != EMMY_OK) return rc;
  if (a->dtype != EMMY_KV8_BF16 && a->dtype != EMMY_KV8_F16)
    return fail(EMMY_EINVAL, WHAT, "dtype must be bf16 or f16");
  if (a->window < 0 || a->sinks < 0) return fail(EMMY_EINVAL, WHAT, "window and sinks must not be negative");
  if (a->sinks > 0 && a->window == 0) return fail(EMMY_EINVAL, WHAT, "sinks need a window");
  if (!std::isfinite(a->scale)) return fail(EMMY_EINVAL, WHAT, "scale must be finite");
  if (cache->tokens == 0 || cache->max_q == 0) return EMMY_OK;
  if (a->q == 0 || a->out == 0) return fail(EMMY_EINVAL, WHAT, "null q or out");
  if (a->q % 16 || a->out % 16 || a->q_strides[0] % 8 || a->q_strides[1] % 8 || a->out_strides[0] % 8 ||
      a->out_strides[1] % 8)
    return fail(EMMY_EINVAL, WHAT, "q and out: base and strides must be multiples of 16 bytes");
  if (a->q_strides[0] < 0 || a->q_strides[1] < 0 || a->out_strides[0] < 0 || a->out_strides[1] < 0)
    return fail(EMMY_EINVAL, WHAT, "q and out: strides must not be negative");
  const auto extent = [&](const int64_t st[2]) {
    return uint64_t((cache->tokens - 1) * st[0] + (a->heads - 1) * st[1] + cache->head_dim) * 2;
  };
  if (overlap(a->q, extent(a->q_strides), a->out, extent(a->out_strides)))
    return fail(EMMY_EINVAL, WHAT, "q and out overlap");
  uint64_t need = 0;
  rc = emmy_kv8_attend_workspace(cache, a->heads, &need);
  if (rc != EMMY_OK) return rc;
  if (a->workspace == 0 || a->workspace % 16 || a->workspace_bytes < need)
    return fail(EMMY_EINVAL, WHAT, "workspace is missing, unaligned or too small");

  AttendParams p;
  p.s = seqs_of(*cache);
  p.codes = reinterpret_cast<const uint8_t *>(cache->codes);
  p.exps = reinterpret_cast<const int8_t *>(cache->exps);
  p.q = reinterpret_cast<const void *>(a->q);
  p.out = reinterpret_cast<void *>(a->out);
  p.q_ts = a->q_strides[0], p.q_hs = a->q_strides[1];
  p.o_ts = a->out_strides[0], p.o_hs = a->out_strides[1];
  p.counters = reinterpret_cast<unsigned *>(a->workspace);
  p.partial = reinterpret_cast<float *>(a->workspace + EMMY_KV8_WORKSPACE_ZERO);
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.group = a->heads / cache->kv_heads;
  p.window = a->window;
  p.sinks = a->sinks;
  p.target = 0;
  p.spread = false;
  // A sequence with up to ROWS_MOST rows of a kv head is the row kernel's,
  // others the tile kernel's, which takes the one sequence of a call that may
  // be either.
  const int64_t most = int64_t(p.group) * cache->max_q;
  const bool tiles = most > ROWS_MOST, rows = !tiles || cache->seqs > 1;
  p.row_limit = rows ? ROWS_MOST : 0;
  const int nt = rows_blocks(most < ROWS_MOST ? most : ROWS_MOST);
  if (int64_t(cache->pages) * 2 * cache->kv_heads * cache->page_size > 0x7fffffff)
    return fail(EMMY_EINVAL, WHAT, "a layer holds at most 2^31 - 1 rows of head_dim codes");
  if (int64_t(cache->seqs) * cache->kv_heads > (1 << 24))
    return fail(EMMY_EINVAL, WHAT, "too many sequences and heads for one call");
  const OnDevice on(cache->device);
  if (on.err != cudaSuccess) return cuda_fail(WHAT, on.err);
  const bool bf16 = a->dtype == EMMY_KV8_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (tiles) {
    rc = tiles_attend(p, *cache, bf16, st);
    if (rc != EMMY_OK) return rc;
  }
  return rows ? rows_attend(p, *cache, nt, bf16, st) : EMMY_OK;
}
