// emmy_kv8_copy_pages -- copies of whole pages, in every layer at once.
//
// Bound by memory: every byte of a page is read once and written once.  One
// CTA copies 16 KB of one page with four 16-byte loads of each thread in
// flight before the first store; the pairs travel in the kernel's parameters,
// so a call needs no device-side list, is one launch for all layers, and can
// be captured.
#include "kv8.cuh"

namespace kv8 {
namespace {

constexpr int COPY_THREADS = 256, COPY_VEC = 4;  // 16 KB a CTA

template <int N>
struct Pairs {
  int src[N], dst[N];
};

template <int N>
__global__ void __launch_bounds__(COPY_THREADS)
copy_kernel(uint4 *codes, int8_t *exps, int pages, int page_vecs, int page_exps, int chunks,
            const __grid_constant__ Pairs<N> pairs) {
  grid_dependency_wait();
  grid_dependency_done();
  const int pair = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int64_t layer = int64_t(blockIdx.y) * pages;
  const int64_t src = layer + pairs.src[pair], dst = layer + pairs.dst[pair];
  const uint4 *from = codes + src * page_vecs;
  uint4 *to = codes + dst * page_vecs;
  const int at = chunk * COPY_THREADS * COPY_VEC + threadIdx.x;
  uint4 v[COPY_VEC];
#pragma unroll
  for (int i = 0; i < COPY_VEC; ++i)
    if (at + i * COPY_THREADS < page_vecs) v[i] = __ldcs(from + at + i * COPY_THREADS);
#pragma unroll
  for (int i = 0; i < COPY_VEC; ++i)
    if (at + i * COPY_THREADS < page_vecs) __stcs(to + at + i * COPY_THREADS, v[i]);
  if (chunk == 0)
    for (int i = threadIdx.x; i < page_exps; i += COPY_THREADS)
      exps[dst * page_exps + i] = exps[src * page_exps + i];
}

template <int N>
int launch(const emmy_kv8 &c, int layers, const int32_t *src, const int32_t *dst, int n,
                   cudaStream_t stream) {
  Pairs<N> pairs = {};
  for (int i = 0; i < n; ++i) pairs.src[i] = src[i], pairs.dst[i] = dst[i];
  const int page_exps = 2 * c.kv_heads;
  const int page_vecs = page_exps * c.page_size * (c.head_dim / 16);
  const int per = COPY_THREADS * COPY_VEC, chunks = (page_vecs + per - 1) / per;
  return launch_kernel("emmy_kv8_copy_pages", copy_kernel<N>, dim3(n * chunks, layers), COPY_THREADS, 0, stream,
                       reinterpret_cast<uint4 *>(c.codes), reinterpret_cast<int8_t *>(c.exps), int(c.pages), page_vecs,
                       page_exps, chunks, pairs);
}

}  // namespace
}  // namespace kv8

extern "C" int emmy_kv8_copy_pages(const emmy_kv8 *cache, int32_t layers, const int32_t *src,
                                   const int32_t *dst, int32_t n, emmy_stream stream) {
  using namespace kv8;
  static const char *what = "emmy_kv8_copy_pages";
  const int rc = check_cache(what, cache);
  if (rc != EMMY_OK) return rc;
  if (layers < 1 || layers > 65535) return fail(EMMY_EINVAL, what, "layers must be between 1 and 65535");
  if (n < 0 || n > EMMY_KV8_MAX_PAIRS) return fail(EMMY_EINVAL, what, "at most 480 pairs in a call");
  if (n == 0) return EMMY_OK;
  if (src == nullptr || dst == nullptr) return fail(EMMY_EINVAL, what, "null page lists");
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= cache->pages || dst[i] < 0 || dst[i] >= cache->pages)
      return fail(EMMY_EINVAL, what, "a page number is outside the pool");
  const OnDevice on(cache->device);
  if (on.err != cudaSuccess) return cuda_fail(what, on.err);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // short lists travel in 512 bytes of parameters, long ones in 3840
  return n <= 64 ? launch<64>(*cache, layers, src, dst, n, st)
                 : launch<EMMY_KV8_MAX_PAIRS>(*cache, layers, src, dst, n, st);
}
