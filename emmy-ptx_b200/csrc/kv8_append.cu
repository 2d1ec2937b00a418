// emmy_kv8_append -- new keys and values into pages of 8-bit codes.
//
// For each page, side (K or V) and kv head that gets new tokens:
//   a = max |x| over the new finite values, e(a) = least e: a <= 448 * 2^e
//   e = max(e of the page, e(a)) where the page held tokens, else e(a)
//   code = RN_e4m3(x * 2^-e);  older codes, when e grew: RN(code * 2^(e_old - e))
// One rounding of each value (two for one whose page grew later; a change of
// scale by a power of two is exact above e4m3's subnormals).
//
// Bound by memory: each new value is read once (2 or 4 bytes) and written
// once (1 byte).  One CTA does one (page, side, head), its rows spread over
// the warps and held in registers, as they came, between the maximum and the
// rounding, so nothing is read twice; a page's rows are contiguous in the pool.
// Where no sequence has more than one new token, a warp does one (sequence,
// side, head).
#include <cuda_bf16.h>

#include "kv8.cuh"

namespace kv8 {
namespace {

struct AppendParams {
  Seqs s;
  uint8_t *codes;
  int8_t *exps;
  const void *x[2];
  int64_t ts[2], hs[2];  // token and head strides, elements
};

// Sixteen bytes of values: as they are held, and as f32.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ void load(const T *p) { w = __ldg(reinterpret_cast<const uint4 *>(p)); }
  __device__ __forceinline__ float at(int i) const;
};
template <>
__device__ __forceinline__ float Vec<float>::at(int i) const {
  return __uint_as_float((&w.x)[i]);
}
template <>
__device__ __forceinline__ float Vec<__nv_bfloat16>::at(int i) const {
  const uint32_t x = (&w.x)[i / 2];
  return __uint_as_float(i & 1 ? x & 0xffff0000u : x << 16);
}
template <>
__device__ __forceinline__ float Vec<__half>::at(int i) const {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&(&w.x)[i / 2]));
  return i & 1 ? f.y : f.x;
}
// The largest finite magnitude, and amax.
template <typename T>
__device__ __forceinline__ float max_finite(const Vec<T> &v, float amax) {
#pragma unroll
  for (int i = 0; i < Vec<T>::N; ++i) {
    const float a = fabsf(v.at(i));
    amax = a < INFINITY ? fmaxf(amax, a) : amax;  // neither infinities nor NaN
  }
  return amax;
}
__device__ __forceinline__ float warp_max(float x) {  // x >= 0
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x)));
}
// Least e in [least, E_MAX] with amax <= 448 * 2^e.
__device__ __forceinline__ int fit_exponent(float amax, int least) {
  // amax = m * 2^k, m in [1, 2): fits under 448 = 1.75 * 2^8 with e = k - 8
  // or, where m > 1.75, k - 7 (f32 subnormals clamp to E_MIN all the same)
  const uint32_t bits = __float_as_uint(amax);
  const int e = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(min(e, E_MAX), max(E_MIN, least));
}

__device__ __forceinline__ float scaled(float x, int e) {
  // 2^-e in one step is representable (e in [-32, 63])
  return x * pow2(-e);
}

// Two e4m3 codes, times 2^shift (shift <= 0), rounded again.
__device__ __forceinline__ uint32_t recode2(uint32_t w, float f) {
  const uint32_t h = e4m3x2_f16x2(w);
  const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&h));
  return f32x2_e4m3x2(v.y * f, v.x * f);
}

// The codes of `rows` rows from the page's first on, rounded from 2^old to 2^e.
template <int D>
__device__ __forceinline__ void recode_rows(uint8_t *codes, int rows, int old, int e, int t, int threads) {
  const float f = pow2(old - e);
  uint4 *q = reinterpret_cast<uint4 *>(codes);
  for (int i = t; i < rows * (D / 16); i += threads) {
    uint4 c = q[i];
    uint32_t *w = &c.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = recode2(w[j], f) | recode2(w[j] >> 16, f) << 16;
    q[i] = c;
  }
}

template <typename T>
__device__ __forceinline__ void store_codes(uint8_t *at, const Vec<T> &v, int e) {
  uint32_t w[2] = {};
#pragma unroll
  for (int j = 0; j < Vec<T>::N; j += 2)
    w[j / 4] |= f32x2_e4m3x2(scaled(v.at(j + 1), e), scaled(v.at(j), e)) << (8 * (j & 2));
  if constexpr (Vec<T>::N == 8)
    *reinterpret_cast<uint2 *>(at) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t *>(at) = w[0];
}

// Exponent of a page's side and head that was `held` before, as it may be.
__device__ __forceinline__ int held_exponent(int8_t held) { return max(min(int(held), E_MAX), E_MIN); }

// Slot of this grid's page list -> (sequence, page of the sequence).  The
// pages that n tokens touch are at most n / P + 2, and floor((s + n) / P) -
// floor(s / P) >= floor(n / P), so sequence b may own the slots from
// q_starts[b] / P + 2 b on; the last b at or below the slot is the owner.
__device__ __forceinline__ int owner(const Seqs &s, int slot) {
  const int lane = threadIdx.x & 31;
  int count = 0;
  for (int b0 = 0; b0 < s.seqs; b0 += 32) {
    const int b = b0 + lane;
    const bool at = b < s.seqs && (s.q_starts[b] >> s.page_shift) + 2 * b <= slot;
    const int here = __popc(__ballot_sync(0xffffffffu, at));
    count += here;
    if (here < 32) break;
  }
  return count - 1;
}

template <int D, typename T>
__global__ void append_kernel(const AppendParams p) {
  using V = Vec<T>;
  constexpr int LPR = D / V::N;             // lanes per row, 16 bytes each
  constexpr int RPW = 32 / LPR;             // rows per warp and pass
  constexpr int PASSES = 64 / (4 * RPW);    // 64 rows to 128 threads
  const Seqs &s = p.s;
  grid_dependency_wait();
  grid_dependency_done();
  const int b = owner(s, blockIdx.x);
  if (b < 0) return;
  int start, n, len;
  lengths(s, b, start, n, len);
  if (n == 0) return;
  const int P = 1 << s.page_shift, first = len - n;
  const int page_of_seq = (first >> s.page_shift) + blockIdx.x - ((start >> s.page_shift) + 2 * b);
  if (page_of_seq < first >> s.page_shift || page_of_seq > (len - 1) >> s.page_shift) return;
  const int page = s.table[int64_t(b) * s.width + page_of_seq];
  const int head = blockIdx.y, side = blockIdx.z;
  const int pos0 = page_of_seq << s.page_shift;
  const int lo = max(first - pos0, 0), hi = min(len - pos0, P);  // new rows of the page
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int col = lane % LPR * V::N, row0 = warp * RPW + lane / LPR, step = warps * RPW;
  const T *x = static_cast<const T *>(side ? p.x[1] : p.x[0]) + head * (side ? p.hs[1] : p.hs[0]) + col;
  const int64_t ts = side ? p.ts[1] : p.ts[0];
  V v[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = row0 + i * step;
    v[i].w = make_uint4(0, 0, 0, 0);
    if (r >= lo && r < hi) v[i].load(x + (int64_t(start) + pos0 + r - first) * ts);
  }
  if (page < 0 || page >= s.pages) {
    report(s.status, STATUS_PAGE);
    return;
  }
  const int64_t unit = (int64_t(page) * 2 + side) * s.kv_heads + head;
  uint8_t *codes = p.codes + (unit << s.page_shift) * D;
  const int old = lo > 0 ? held_exponent(p.exps[unit]) : E_MIN;
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) amax = max_finite(v[i], amax);
  __shared__ float part[16];
  amax = warp_max(amax);
  if (lane == 0) part[warp] = amax;
  __syncthreads();
  for (int w = 0; w < warps; ++w) amax = fmaxf(amax, part[w]);
  const int e = fit_exponent(amax, old);
  if (threadIdx.x == 0) p.exps[unit] = int8_t(e);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = row0 + i * step;
    if (r >= lo && r < hi) store_codes(codes + int64_t(r) * D + col, v[i], e);
  }
  if (lo > 0 && e > old) recode_rows<D>(codes, lo, old, e, threadIdx.x, blockDim.x);
}

// One new token of a sequence, or none: a warp a (sequence, side, head).
template <int D, typename T>
__global__ void __launch_bounds__(128) append_one_kernel(const AppendParams p) {
  using V = Vec<T>;
  constexpr int LPR = D / V::N;
  const Seqs &s = p.s;
  grid_dependency_wait();
  grid_dependency_done();
  const int b = blockIdx.x, unit_of_seq = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (unit_of_seq >= 2 * s.kv_heads) return;
  int start, n, len;
  lengths(s, b, start, n, len);
  if (n == 0) return;
  if (n > 1) {  // more than the call's max_q
    report(s.status, STATUS_LENGTH);
    return;
  }
  const int page = s.table[int64_t(b) * s.width + ((len - 1) >> s.page_shift)];
  const int side = unit_of_seq >= s.kv_heads, head = unit_of_seq - side * s.kv_heads;
  V v;
  v.w = make_uint4(0, 0, 0, 0);
  if (lane < LPR)
    v.load(static_cast<const T *>(side ? p.x[1] : p.x[0]) + start * (side ? p.ts[1] : p.ts[0]) +
           head * (side ? p.hs[1] : p.hs[0]) + lane * V::N);
  if (page < 0 || page >= s.pages) {
    report(s.status, STATUS_PAGE);
    return;
  }
  const int64_t unit = (int64_t(page) * 2 + side) * s.kv_heads + head;
  uint8_t *codes = p.codes + (unit << s.page_shift) * D;
  const int lo = (len - 1) & ((1 << s.page_shift) - 1);
  const int old = lo > 0 ? held_exponent(p.exps[unit]) : E_MIN;
  const int e = fit_exponent(warp_max(max_finite(v, 0.0f)), old);
  if (lane == 0) p.exps[unit] = int8_t(e);
  if (lane < LPR) store_codes(codes + int64_t(lo) * D + lane * V::N, v, e);
  if (lo > 0 && e > old) recode_rows<D>(codes, lo, old, e, lane, 32);
}

template <int D, typename T>
int launch(const AppendParams &p, bool one, int64_t slots, cudaStream_t stream) {
  if (one)
    return launch_kernel("emmy_kv8_append", append_one_kernel<D, T>, dim3(p.s.seqs, (2 * p.s.kv_heads + 3) / 4), 128, 0,
                         stream, p);
  return launch_kernel("emmy_kv8_append", append_kernel<D, T>, dim3(unsigned(slots), p.s.kv_heads, 2),
                       2 << p.s.page_shift, 0, stream, p);
}

template <int D>
int launch_type(const AppendParams &p, int dtype, bool one, int64_t slots, cudaStream_t stream) {
  if (dtype == EMMY_KV8_F32) return launch<D, float>(p, one, slots, stream);
  if (dtype == EMMY_KV8_BF16) return launch<D, __nv_bfloat16>(p, one, slots, stream);
  return launch<D, __half>(p, one, slots, stream);
}

}  // namespace
}  // namespace kv8

extern "C" int emmy_kv8_append(const emmy_kv8 *cache, emmy_dptr k, emmy_dptr v, int32_t dtype,
                               const int64_t k_strides[2], const int64_t v_strides[2],
                               emmy_stream stream) {
  using namespace kv8;
  static const char *what = "emmy_kv8_append";
  int rc = check_cache(what, cache);
  if (rc == EMMY_OK) rc = check_seqs(what, cache);
  if (rc != EMMY_OK) return rc;
  if (k_strides == nullptr || v_strides == nullptr) return fail(EMMY_EINVAL, what, "null strides");
  if (dtype != EMMY_KV8_F32 && dtype != EMMY_KV8_BF16 && dtype != EMMY_KV8_F16)
    return fail(EMMY_EINVAL, what, "dtype must be f32, bf16 or f16");
  if (cache->tokens == 0 || cache->max_q == 0) return EMMY_OK;
  if (k == 0 || v == 0) return fail(EMMY_EINVAL, what, "null k or v");
  const int unit = dtype == EMMY_KV8_F32 ? 4 : 8;  // elements in 16 bytes
  if (k % 16 || v % 16 || k_strides[0] % unit || k_strides[1] % unit || v_strides[0] % unit ||
      v_strides[1] % unit)
    return fail(EMMY_EINVAL, what, "k and v: base and strides must be multiples of 16 bytes");
  AppendParams p;
  p.s = seqs_of(*cache);
  p.codes = reinterpret_cast<uint8_t *>(cache->codes);
  p.exps = reinterpret_cast<int8_t *>(cache->exps);
  p.x[0] = reinterpret_cast<const void *>(k);
  p.x[1] = reinterpret_cast<const void *>(v);
  p.ts[0] = k_strides[0], p.hs[0] = k_strides[1];
  p.ts[1] = v_strides[0], p.hs[1] = v_strides[1];
  const OnDevice on(cache->device);
  if (on.err != cudaSuccess) return cuda_fail(what, on.err);
  // the slots that owner() gives out
  const int64_t slots = (int64_t(cache->tokens) >> p.s.page_shift) + 2 * int64_t(cache->seqs);
  if (slots > 0x7fffffff) return fail(EMMY_EINVAL, what, "too many tokens");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->head_dim == 64 ? launch_type<64>(p, dtype, cache->max_q == 1, slots, st)
                               : launch_type<128>(p, dtype, cache->max_q == 1, slots, st);
}
