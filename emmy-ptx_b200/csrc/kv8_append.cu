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
// once (1 byte).  One CTA does one page, a few of its (side, head)s one after
// another: a thread copies its own 16-byte pieces of the next one's rows into
// shared memory (cp.async) while it takes the maximum of this one's and rounds
// them, so loads stay in flight through the reductions.  Where no sequence has
// more than one new token, a warp does one (sequence, side, head).
#include <cuda_bf16.h>

#include <algorithm>

#include "kv8.cuh"

namespace kv8 {
namespace {

struct AppendParams {
  Seqs s;
  uint8_t *codes;
  int8_t *exps;
  const void *x[2];
  int64_t ts[2], hs[2];  // token and head strides, elements
  int units;             // (side, head)s of a page that a CTA does
};

// Sixteen bytes of values: as they are held, and as f32.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ void load(const void *p) { w = *static_cast<const uint4 *>(p); }
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

// Slot of this grid's page list -> its sequence's lengths and the page of the
// sequence; false: none.  The pages that n tokens touch are at most n / P + 2,
// and floor((s + n) / P) - floor(s / P) >= floor(n / P), so sequence b may own
// the slots from q_starts[b] / P + 2 b on; the last b at or below the slot is
// the owner.  A warp reads 32 sequences' lengths at once.
__device__ __forceinline__ bool owner(const Seqs &s, int slot, int &b, int &start, int &n, int &len, int &page_of_seq) {
  const int lane = threadIdx.x & 31;
  int from = -1, qs = 0, qe = 0, kv = 0;  // the last group that has a sequence at or below the slot
  for (int b0 = 0; b0 < s.seqs; b0 += 32) {
    const bool in = b0 + lane < s.seqs;
    const int q0 = in ? s.q_starts[b0 + lane] : 0, q1 = in ? s.q_starts[b0 + lane + 1] : 0;
    const int k = in ? s.kv_lens[b0 + lane] : 0;
    const int here = __popc(__ballot_sync(0xffffffffu, in && (q0 >> s.page_shift) + 2 * (b0 + lane) <= slot));
    if (here > 0) from = b0 + here - 1, qs = q0, qe = q1, kv = k;
    if (here < 32) break;
  }
  if (from < 0) return false;
  b = from;
  start = __shfl_sync(0xffffffffu, qs, from & 31);
  len = __shfl_sync(0xffffffffu, kv, from & 31);
  n = checked_n(s, start, __shfl_sync(0xffffffffu, qe, from & 31) - start, len);
  const int first = (len - n) >> s.page_shift;
  page_of_seq = first + slot - ((start >> s.page_shift) + 2 * b);
  return n > 0 && page_of_seq >= first && page_of_seq <= (len - 1) >> s.page_shift;
}

// Threads for a page of P rows: eight 16-byte pieces each.
template <int D, typename T>
constexpr int page_threads(int page) {
  return page * D * int(sizeof(T)) / 128;
}
template <int D, typename T>
constexpr int MOST_THREADS = page_threads<D, T>(256);

// 16 bytes, or zeros where there is nothing to copy.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

template <int D, typename T>
__global__ void __launch_bounds__(MOST_THREADS<D, T>) append_kernel(const AppendParams p) {
  using V = Vec<T>;
  constexpr int LPR = D / V::N;  // lanes per row, 16 bytes each
  constexpr int RPW = 32 / LPR;  // rows per warp and pass
  constexpr int PASSES = 8;
  extern __shared__ uint4 pieces[];  // [2][PASSES][threads]
  __shared__ float part[2][32];
  const Seqs &s = p.s;
  grid_dependency_wait();
  grid_dependency_done();
  int b, start, n, len, page_of_seq;
  if (!owner(s, blockIdx.x, b, start, n, len, page_of_seq)) return;
  const int P = 1 << s.page_shift, first = len - n, H = s.kv_heads;
  const int page = s.table[int64_t(b) * s.width + page_of_seq];
  const int pos0 = page_of_seq << s.page_shift;
  const int lo = max(first - pos0, 0), hi = min(len - pos0, P);  // new rows of the page
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  const int col = lane % LPR * V::N, row0 = warp * RPW + lane / LPR, step = warps * RPW;
  const int64_t token0 = int64_t(start) + pos0 - first;  // row 0 of the page, were it new
  const auto fetch = [&](int u, int buf) {
    const int side = u >= H, head = u - side * H;
    const int64_t ts = side ? p.ts[1] : p.ts[0];
    const T *x = static_cast<const T *>(side ? p.x[1] : p.x[0]) + head * (side ? p.hs[1] : p.hs[0]) + col;
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(pieces + buf * PASSES * threads + tid));
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = row0 + i * step;
      const bool real = r >= lo && r < hi;
      copy16(to + i * threads * 16, x + (token0 + (real ? r : lo)) * ts, real);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int u0 = blockIdx.y * p.units, u1 = min(u0 + p.units, 2 * H);
  fetch(u0, 0);
  const bool bad = page < 0 || page >= s.pages;
  if (bad && tid == 0) report(s.status, STATUS_PAGE);
  const int64_t unit0 = int64_t(bad ? 0 : page) * 2 * H;
  int held = lo > 0 ? p.exps[unit0 + u0] : 0;
  for (int u = u0; u < u1; ++u) {
    const int buf = (u - u0) & 1, old = lo > 0 ? held_exponent(held) : E_MIN;
    if (u + 1 < u1) {
      fetch(u + 1, buf ^ 1);
      held = lo > 0 ? p.exps[unit0 + u + 1] : 0;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // every thread reads only the pieces it copied
    const uint4 *mine = pieces + buf * PASSES * threads + tid;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      V v;
      v.load(mine + i * threads);
      amax = max_finite(v, amax);
    }
    amax = warp_max(amax);
    if (lane == 0) part[buf][warp] = amax;
    __syncthreads();
    amax = warp_max(lane < warps ? part[buf][lane] : 0.0f);
    if (bad) continue;
    const int e = fit_exponent(amax, old);
    uint8_t *codes = p.codes + ((unit0 + u) << s.page_shift) * D;
    if (tid == 0) p.exps[unit0 + u] = int8_t(e);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = row0 + i * step;
      if (r >= lo && r < hi) {
        V v;
        v.load(mine + i * threads);
        store_codes(codes + r * D + col, v, e);
      }
    }
    if (lo > 0 && e > old) recode_rows<D>(codes, lo, old, e, tid, threads);
  }
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
int launch(AppendParams p, bool one, int64_t slots, int device, cudaStream_t stream) {
  const int units = 2 * p.s.kv_heads;
  if (one)
    return launch_kernel("emmy_kv8_append", append_one_kernel<D, T>, dim3(p.s.seqs, (units + 3) / 4), 128, 0, stream, p);
  // several (side, head)s a CTA once there are more than fill the GPU twice
  const int threads = page_threads<D, T>(1 << p.s.page_shift);
  const int64_t fill = int64_t(sm_count(device)) * 2 * (2048 / threads < 7 ? 2048 / threads : 7);
  p.units = int(std::min<int64_t>(units, std::max<int64_t>(1, slots * units / std::max<int64_t>(fill, 1))));
  int smem = 2 * 8 * 16 * threads;
  constexpr int ROOM = 200 * 1024;
  if (smem > ROOM) smem /= 2, p.units = 1;  // no second buffer, so no second unit (f32 pages of 128 KB)
  static KernelSetup setup;
  const int rc = setup.ready("emmy_kv8_append", append_kernel<D, T>, device,
                             std::min(ROOM, 2 * 8 * 16 * MOST_THREADS<D, T>));
  if (rc != EMMY_OK) return rc;
  return launch_kernel("emmy_kv8_append", append_kernel<D, T>, dim3(unsigned(slots), (units + p.units - 1) / p.units),
                       threads, smem, stream, p);
}

template <int D>
int launch_type(const AppendParams &p, int dtype, bool one, int64_t slots, int device, cudaStream_t stream) {
  if (dtype == EMMY_KV8_F32) return launch<D, float>(p, one, slots, device, stream);
  if (dtype == EMMY_KV8_BF16) return launch<D, __nv_bfloat16>(p, one, slots, device, stream);
  return launch<D, __half>(p, one, slots, device, stream);
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
  note_capture(st);
  return cache->head_dim == 64 ? launch_type<64>(p, dtype, cache->max_q == 1, slots, cache->device, st)
                               : launch_type<128>(p, dtype, cache->max_q == 1, slots, cache->device, st);
}
