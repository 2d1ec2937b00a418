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
// the warps and held in registers between the maximum and the rounding, so
// nothing is read twice; a page's rows are contiguous in the pool.
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

// Eight consecutive values as f32.
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
  x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const __half *p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
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

template <int D, int PASSES, typename T>
__global__ void append_kernel(const AppendParams p) {
  constexpr int LPR = D / 8;     // lanes per row, eight values each
  constexpr int RPW = 32 / LPR;  // rows per warp and pass
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
  if (page < 0 || page >= s.pages) {
    report(s.status, STATUS_PAGE);
    return;
  }
  const int head = blockIdx.y, side = blockIdx.z;
  const int64_t unit = (int64_t(page) * 2 + side) * s.kv_heads + head;
  uint8_t *codes = p.codes + (unit << s.page_shift) * D;
  const int pos0 = page_of_seq << s.page_shift;
  const int lo = max(first - pos0, 0), hi = min(len - pos0, P);  // new rows of the page
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int col = (lane % LPR) * 8, row0 = warp * RPW + lane / LPR, step = warps * RPW;
  const T *x = static_cast<const T *>(side ? p.x[1] : p.x[0]) + head * (side ? p.hs[1] : p.hs[0]) + col;
  const int64_t ts = side ? p.ts[1] : p.ts[0];
  float v[PASSES][8];
  float amax = 0.0f;
  const int old = lo > 0 ? max(min(int(p.exps[unit]), E_MAX), E_MIN) : E_MIN;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = row0 + i * step;
    if (r >= lo && r < hi) load8(x + (int64_t(start) + pos0 + r - first) * ts, v[i]);
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = row0 + i * step;
    if (r >= lo && r < hi) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = fabsf(v[i][j]);
        if (a < INFINITY) amax = fmaxf(amax, a);  // neither infinities nor NaN
      }
    }
  }
  __shared__ float part[16];
  amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
  if (lane == 0) part[warp] = amax;
  __syncthreads();
  for (int w = 0; w < warps; ++w) amax = fmaxf(amax, part[w]);
  // amax = m * 2^k, m in [1, 2): fits under 448 = 1.75 * 2^8 with e = k - 8
  // or, where m > 1.75, k - 7 (f32 subnormals clamp to E_MIN all the same)
  const uint32_t bits = __float_as_uint(amax);
  int e = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(min(e, E_MAX), max(E_MIN, old));
  if (threadIdx.x == 0) p.exps[unit] = int8_t(e);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = row0 + i * step;
    if (r >= lo && r < hi) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = f32x2_e4m3x2(scaled(v[i][2 * j + 1], e), scaled(v[i][2 * j], e));
      *reinterpret_cast<uint2 *>(codes + int64_t(r) * D + col) =
          make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    }
  }
  if (lo > 0 && e > old) {
    const float f = pow2(old - e);
    uint4 *q = reinterpret_cast<uint4 *>(codes);
    for (int i = threadIdx.x; i < lo * (D / 16); i += blockDim.x) {
      uint4 c = q[i];
      uint32_t *w = &c.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = recode2(w[j], f) | recode2(w[j] >> 16, f) << 16;
      q[i] = c;
    }
  }
}

template <int D, typename T>
int launch(const AppendParams &p, int slots, cudaStream_t stream) {
  // 64 rows to 128 threads: D / 16 passes over the page
  return launch_kernel("emmy_kv8_append", append_kernel<D, D / 16, T>, dim3(slots, p.s.kv_heads, 2),
                       2 << p.s.page_shift, 0, stream, p);
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
  const bool d64 = cache->head_dim == 64;
  if (dtype == EMMY_KV8_F32)
    return d64 ? launch<64, float>(p, int(slots), st) : launch<128, float>(p, int(slots), st);
  if (dtype == EMMY_KV8_BF16)
    return d64 ? launch<64, __nv_bfloat16>(p, int(slots), st) : launch<128, __nv_bfloat16>(p, int(slots), st);
  return d64 ? launch<64, __half>(p, int(slots), st) : launch<128, __half>(p, int(slots), st);
}
