// Host-side checks shared by the entry points of the paged 8-bit cache.
#include <cmath>
#include <cstdio>
#include <numeric>

#include "kv8.cuh"

void emmyrt_set_last_error(const char *msg);  // emmyrt.cpp; not exported

namespace kv8 {

int fail(int code, const char *what, const char *msg) {
  char buf[256];
  snprintf(buf, sizeof buf, "%s: %s", what, msg);
  emmyrt_set_last_error(buf);
  return code;
}

int cuda_fail(const char *what, cudaError_t e) {
  return fail(EMMY_ECUDART, what, cudaGetErrorString(e));
}

int check_cache(const char *what, const emmy_kv8 *c) {
  if (c == nullptr) return fail(EMMY_EINVAL, what, "null cache description");
  if (c->codes == 0 || c->exps == 0) return fail(EMMY_EINVAL, what, "null cache storage");
  if (c->codes % 16 != 0) return fail(EMMY_EINVAL, what, "codes must be 16-byte aligned");
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(EMMY_EINVAL, what, "head_dim must be 64 or 128");
  if (c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
    return fail(EMMY_EINVAL, what, "page_size must be 64, 128 or 256");
  if (c->kv_heads < 1 || c->kv_heads > 1024)
    return fail(EMMY_EINVAL, what, "kv_heads must be between 1 and 1024");
  if (c->pages < 1) return fail(EMMY_EINVAL, what, "the cache has no pages");
  if (c->device < 0) return fail(EMMY_EINVAL, what, "negative device");
  return EMMY_OK;
}

Seqs seqs_of(const emmy_kv8 &c) {
  Seqs s;
  s.table = reinterpret_cast<const int *>(c.page_table);
  s.kv_lens = reinterpret_cast<const int *>(c.kv_lens);
  s.q_starts = reinterpret_cast<const int *>(c.q_starts);
  s.status = reinterpret_cast<unsigned *>(c.status);
  s.seqs = c.seqs;
  s.width = c.table_width;
  s.pages = c.pages;
  s.tokens = c.tokens;
  s.max_q = c.max_q;
  s.kv_heads = c.kv_heads;
  s.page_shift = c.page_size == 64 ? 6 : c.page_size == 128 ? 7 : 8;
  return s;
}

int check_seqs(const char *what, const emmy_kv8 *c) {
  if (c->page_table == 0 || c->kv_lens == 0 || c->q_starts == 0)
    return fail(EMMY_EINVAL, what, "null page table, kv_lens or q_starts");
  if (c->page_table % 4 || c->kv_lens % 4 || c->q_starts % 4 || c->status % 4)
    return fail(EMMY_EINVAL, what, "page table, lengths and status must be 4-byte aligned");
  return check_counts(what, c);
}

int check_counts(const char *what, const emmy_kv8 *c) {
  if (c->seqs < 1 || c->seqs > EMMY_KV8_MAX_SEQS)
    return fail(EMMY_EINVAL, what, "seqs must be between 1 and 4096");
  if (c->table_width < 1 || c->tokens < 0 || c->max_q < 0 || c->max_q > c->tokens)
    return fail(EMMY_EINVAL, what, "bad table_width, tokens or max_q");
  if (int64_t(c->table_width) * c->page_size > (int64_t(1) << 30))
    return fail(EMMY_EINVAL, what, "a sequence holds at most 2^30 keys");
  return EMMY_OK;
}

int rows_trouble(emmy_dptr q, const int64_t q_strides[2], int64_t q_heads, int q_size, emmy_dptr out,
                 const int64_t out_strides[2], int64_t H, int size, int64_t T, int64_t D, bool in_place) {
  const int64_t qt = q_strides[0], qh = q_strides[1], ts = out_strides[0], hs = out_strides[1];
  if (qt < 0 || qh < 0 || ts < 0 || hs < 0) return ROWS_NEGATIVE;
  // rows of out one after another, tokens within heads or heads within tokens
  if ((T > 1 && ts < D) || (H > 1 && hs < D) || (T > 1 && H > 1 && (ts <= hs ? hs < ts * (T - 1) + D : ts < hs * (H - 1) + D)))
    return ROWS_SELF;
  if (in_place) return ROWS_FINE;
  if (!overlap(q, uint64_t((T - 1) * qt + (q_heads - 1) * qh + D) * q_size, out,
               uint64_t((T - 1) * ts + (H - 1) * hs + D) * size))
    return ROWS_FINE;
  if (q_size != size) return ROWS_BOTH;
  // rows of both in turn, as slices of one wider array are: of heads, of
  // tokens where heads come first, or of elements
  const auto in_turn = [&](int64_t step_q, int64_t step_out, int64_t wide_q, int64_t wide_out) {
    if (step_q != step_out || step_q == 0) return false;
    const int64_t by = int64_t(out - q) / size % step_q, off = by < 0 ? by + step_q : by;
    return off >= wide_q && off + wide_out <= step_q;
  };
  const int64_t step = std::gcd(std::gcd(qt, qh), std::gcd(ts, hs));
  if (in_turn(qt, ts, (q_heads - 1) * qh + D, (H - 1) * hs + D) || in_turn(qh, hs, (T - 1) * qt + D, (T - 1) * ts + D) ||
      in_turn(step, step, D, D))
    return ROWS_FINE;
  return ROWS_BOTH;
}

const char *rotary_trouble(const emmy_rotary *r) {
  if (r == nullptr) return "null rotary description";
  if (r->head_dim < 2 || r->head_dim > 2 * EMMY_ROTARY_PAIRS) return "head_dim must be between 2 and 512";
  if (r->dims < 2 || r->dims % 2 != 0 || r->dims > r->head_dim) return "dims must be even, between 2 and head_dim";
  if (!std::isfinite(r->gain)) return "gain must be finite";
  return nullptr;
}

int sm_count(int device) {
  static int known[64] = {};
  if (device >= 0 && device < 64 && known[device] > 0) return known[device];
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
  if (device >= 0 && device < 64) known[device] = n;
  return n;
}

static std::atomic<uint64_t> g_wait_limit{EMMY_KV8_WAIT_NS};
static std::atomic<int32_t> g_stall{0};
void wait_limit(unsigned long long &ns, int &stall) {
  ns = g_wait_limit.load(std::memory_order_relaxed);
  stall = g_stall.load(std::memory_order_relaxed);
}

static std::atomic<uint64_t> g_captured{0};
void note_capture(cudaStream_t stream) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  // what is wrong with the stream the launch will say
  if (cudaStreamIsCapturing(stream, &st) != cudaSuccess)
    cudaGetLastError();
  else if (st != cudaStreamCaptureStatusNone)
    g_captured.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace kv8

extern "C" int emmy_kv8_captured(uint64_t *calls) {
  if (calls == nullptr) return kv8::fail(EMMY_EINVAL, "emmy_kv8_captured", "null result");
  *calls = kv8::g_captured.load(std::memory_order_relaxed);
  return EMMY_OK;
}

extern "C" int emmy_kv8_wait_limit(uint64_t ns, int32_t stall) {
  if (stall < 0) return kv8::fail(EMMY_EINVAL, "emmy_kv8_wait_limit", "stall must not be negative");
  kv8::g_stall.store(stall, std::memory_order_relaxed);
  kv8::g_wait_limit.store(ns, std::memory_order_relaxed);
  return EMMY_OK;
}

extern "C" int emmy_stream_capturing(emmy_stream stream, int *capturing) {
  if (capturing == nullptr) return kv8::fail(EMMY_EINVAL, "emmy_stream_capturing", "null result");
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  const cudaError_t e = cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &st);
  if (e != cudaSuccess) return kv8::cuda_fail("emmy_stream_capturing", e);
  *capturing = st != cudaStreamCaptureStatusNone;
  return EMMY_OK;
}

extern "C" int emmy_stream_id(emmy_stream stream, uint64_t *id) {
  if (id == nullptr) return kv8::fail(EMMY_EINVAL, "emmy_stream_id", "null result");
  unsigned long long word = 0;
  const cudaError_t e = cudaStreamGetId(static_cast<cudaStream_t>(stream), &word);
  if (e != cudaSuccess) return kv8::cuda_fail("emmy_stream_id", e);
  *id = word;
  return EMMY_OK;
}

extern "C" int emmy_device_enter(int device, int *before) {
  if (before == nullptr) return kv8::fail(EMMY_EINVAL, "emmy_device_enter", "null result");
  cudaError_t e = cudaGetDevice(before);
  if (e == cudaSuccess) e = cudaSetDevice(device);
  return e == cudaSuccess ? EMMY_OK : kv8::cuda_fail("emmy_device_enter", e);
}

extern "C" int emmy_device_leave(int before) {
  int now = before;
  cudaError_t e = cudaGetDevice(&now);
  if (e == cudaSuccess && now != before) e = cudaSetDevice(before);
  return e == cudaSuccess ? EMMY_OK : kv8::cuda_fail("emmy_device_leave", e);
}
