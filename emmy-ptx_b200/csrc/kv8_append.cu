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
//
// emmy_kv8_append_rotated -- the same of keys turned to their positions on the
// way, in f32 and unrounded, and queries turned into an array of their own: more
// (query head)s behind the (side, head)s, with the same copies, maxima and page
// left out.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "kv8.cuh"
#include "rotary.cuh"

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

struct RotatedParams : AppendParams {
  uint64_t frequency[64];
  const void *positions;  // null: the places in the sequences
  int64_t position_stride;
  const void *q;
  void *out;
  int64_t q_ts, q_hs, o_ts, o_hs;
  int dims, heads, out_type;  // heads: 0 where there is no q
  bool wide, interleaved;
  float gain;
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

// Where a token stands: its place in the sequence, or what the caller says.
__device__ __forceinline__ int64_t position_of(const RotatedParams &p, int64_t token, int place) {
  if (p.positions == nullptr) return place;
  return p.wide ? static_cast<const int64_t *>(p.positions)[token * p.position_stride]
                : static_cast<const int *>(p.positions)[token * p.position_stride];
}

// Values col .. col + N - 1 of a row in shared memory, turned to a position.
template <typename T, int N>
__device__ __forceinline__ void turn_piece(const RotatedParams &p, const T *row, int col, int64_t pos, float (&y)[N]) {
  using rotary::to_float;
  if (p.interleaved) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float a = to_float(row[col + i]), b = to_float(row[col + i + 1]);
      y[i] = a, y[i + 1] = b;
      if (col + i < p.dims) {
        float c, s;
        rotary::turn_of(pos, p.frequency[(col + i) / 2], c, s);
        c *= p.gain, s *= p.gain;
        y[i] = a * c - b * s;
        y[i + 1] = a * s + b * c;
      }
    }
  } else {
    const int half = p.dims / 2;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = col + i;
      y[i] = to_float(row[at]);
      if (at < p.dims) {
        const bool low = at < half;
        const float other = to_float(row[low ? at + half : at - half]);
        float c, s;
        rotary::turn_of(pos, p.frequency[low ? at : at - half], c, s);
        c *= p.gain, s *= p.gain;
        y[i] = low ? y[i] * c - other * s : other * s + y[i] * c;
      }
    }
  }
}

template <int N>
__device__ __forceinline__ float max_finite(const float (&y)[N], float amax) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float a = fabsf(y[i]);
    amax = a < INFINITY ? fmaxf(amax, a) : amax;
  }
  return amax;
}
template <int N>
__device__ __forceinline__ void store_codes(uint8_t *at, const float (&y)[N], int e) {
  uint32_t w[2] = {};
#pragma unroll
  for (int j = 0; j < N; j += 2)
    w[j / 4] |= f32x2_e4m3x2(scaled(y[j + 1], e), scaled(y[j], e)) << (8 * (j & 2));
  if constexpr (N == 8)
    *reinterpret_cast<uint2 *>(at) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t *>(at) = w[0];
}
// Turned queries, rounded once to the type they are wanted in.
template <typename U, int N>
__device__ __forceinline__ void store_as(void *out, int64_t at, const float (&y)[N]) {
  rotary::Piece<U, sizeof(U) * N <= 16 ? N : N / 2> w[sizeof(U) * N <= 16 ? 1 : 2];
  constexpr int EACH = sizeof(U) * N <= 16 ? N : N / 2;
#pragma unroll
  for (int i = 0; i < N; ++i) w[i / EACH].v[i % EACH] = rotary::rounded<U>(y[i]);
#pragma unroll
  for (int i = 0; i < N / EACH; ++i) *reinterpret_cast<rotary::Piece<U, EACH> *>(static_cast<U *>(out) + at + i * EACH) = w[i];
}
template <int N>
__device__ __forceinline__ void store_query(const RotatedParams &p, int64_t token, int head, int col, const float (&y)[N]) {
  const int64_t at = token * p.o_ts + head * p.o_hs + col;
  if (p.out_type == EMMY_KV8_F32)
    store_as<float>(p.out, at, y);
  else if (p.out_type == EMMY_KV8_BF16)
    store_as<__nv_bfloat16>(p.out, at, y);
  else
    store_as<__half>(p.out, at, y);
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

template <int D, typename T, typename Params>
__global__ void __launch_bounds__(MOST_THREADS<D, T>) append_kernel(const __grid_constant__ Params p) {
  constexpr bool ROTATED = std::is_same<Params, RotatedParams>::value;
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
    int64_t ts = side ? p.ts[1] : p.ts[0];
    const T *x = static_cast<const T *>(side ? p.x[1] : p.x[0]) + head * (side ? p.hs[1] : p.hs[0]) + col;
    if constexpr (ROTATED)
      if (u >= 2 * H) x = static_cast<const T *>(p.q) + (u - 2 * H) * p.q_hs + col, ts = p.q_ts;
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(pieces + buf * PASSES * threads + tid));
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = row0 + i * step;
      const bool real = r >= lo && r < hi;
      copy16(to + i * threads * 16, x + (token0 + (real ? r : lo)) * ts, real);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int all = 2 * H;
  if constexpr (ROTATED) all += p.heads;
  const int u0 = blockIdx.y * p.units, u1 = min(u0 + p.units, all);
  fetch(u0, 0);
  const bool bad = page < 0 || page >= s.pages;
  if (bad && tid == 0) report(s.status, STATUS_PAGE);
  const int64_t unit0 = int64_t(bad ? 0 : page) * 2 * H;
  const auto held_at = [&](int u) { return lo > 0 && (!ROTATED || u < 2 * H) ? p.exps[unit0 + u] : 0; };
  int held = held_at(u0);
  for (int u = u0; u < u1; ++u) {
    const int buf = (u - u0) & 1, old = lo > 0 ? held_exponent(held) : E_MIN;
    if (u + 1 < u1) {
      fetch(u + 1, buf ^ 1);
      held = held_at(u + 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // every thread reads only the pieces it copied
    const uint4 *mine = pieces + buf * PASSES * threads + tid;
    float amax = 0.0f;
    float turned[ROTATED ? PASSES : 1][V::N];
    bool turn = false;  // keys, which are turned, or queries
    if constexpr (ROTATED) {
      turn = u < H || u >= 2 * H;
      __syncwarp();  // but turned ones are paired with others of the row, which its warp copied
      if (turn) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int r = row0 + i * step;
          if (r < lo || r >= hi) continue;
          const T *row = reinterpret_cast<const T *>(pieces + buf * PASSES * threads + i * threads + (tid & ~(LPR - 1)));
          turn_piece<T>(p, row, col, position_of(p, token0 + r, pos0 + r), turned[i]);
          if (u >= 2 * H)
            store_query(p, token0 + r, u - 2 * H, col, turned[i]);
          else
            amax = max_finite(turned[i], amax);
        }
        __syncwarp();  // before this buffer's next copies
        if (u >= 2 * H) continue;
      }
    }
    if (!turn) {
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        V v;
        v.load(mine + i * threads);
        amax = max_finite(v, amax);
      }
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
        if constexpr (ROTATED)
          if (turn) {
            store_codes(codes + r * D + col, turned[i], e);
            continue;
          }
        V v;
        v.load(mine + i * threads);
        store_codes(codes + r * D + col, v, e);
      }
    }
    if (lo > 0 && e > old) recode_rows<D>(codes, lo, old, e, tid, threads);
  }
}

// One new token of a sequence, or none: a warp a (sequence, side, head).
template <int D, typename T, typename Params>
__global__ void __launch_bounds__(128) append_one_kernel(const __grid_constant__ Params p) {
  constexpr bool ROTATED = std::is_same<Params, RotatedParams>::value;
  using V = Vec<T>;
  constexpr int LPR = D / V::N;
  const Seqs &s = p.s;
  grid_dependency_wait();
  grid_dependency_done();
  const int b = blockIdx.x, unit_of_seq = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  int all = 2 * s.kv_heads;
  if constexpr (ROTATED) all += p.heads;
  if (unit_of_seq >= all) return;
  int start, n, len;
  lengths(s, b, start, n, len);
  if (n == 0) return;
  const int page = s.table[int64_t(b) * s.width + ((len - 1) >> s.page_shift)];
  const int side = unit_of_seq >= s.kv_heads, head = unit_of_seq - side * s.kv_heads;
  V v;
  v.w = make_uint4(0, 0, 0, 0);
  bool query = false;
  if constexpr (ROTATED) query = unit_of_seq >= 2 * s.kv_heads;
  if (query) {
    if constexpr (ROTATED)
      if (lane < LPR)
        v.load(static_cast<const T *>(p.q) + start * p.q_ts + (unit_of_seq - 2 * s.kv_heads) * p.q_hs + lane * V::N);
  } else if (lane < LPR)
    v.load(static_cast<const T *>(side ? p.x[1] : p.x[0]) + start * (side ? p.ts[1] : p.ts[0]) +
           head * (side ? p.hs[1] : p.hs[0]) + lane * V::N);
  float turned[V::N];
  bool turn = false;
  if constexpr (ROTATED) {
    turn = unit_of_seq < s.kv_heads || query;
    if (turn) {
      __shared__ uint4 rows[4][LPR];
      uint4 *row = rows[threadIdx.x >> 5];
      if (lane < LPR) row[lane] = v.w;
      __syncwarp();
      if (lane < LPR) turn_piece<T>(p, reinterpret_cast<const T *>(row), lane * V::N, position_of(p, start, len - 1), turned);
      if (query) {
        if (lane < LPR) store_query(p, start, unit_of_seq - 2 * s.kv_heads, lane * V::N, turned);
        return;
      }
    }
  }
  if (page < 0 || page >= s.pages) {
    report(s.status, STATUS_PAGE);
    return;
  }
  const int64_t unit = (int64_t(page) * 2 + side) * s.kv_heads + head;
  uint8_t *codes = p.codes + (unit << s.page_shift) * D;
  const int lo = (len - 1) & ((1 << s.page_shift) - 1);
  const int old = lo > 0 ? held_exponent(p.exps[unit]) : E_MIN;
  const float amax = turn && lane < LPR ? max_finite(turned, 0.0f) : max_finite(v, 0.0f);
  const int e = fit_exponent(warp_max(amax), old);
  if (lane == 0) p.exps[unit] = int8_t(e);
  if (lane < LPR) {
    uint8_t *at = codes + int64_t(lo) * D + lane * V::N;
    if (turn)
      store_codes(at, turned, e);
    else
      store_codes(at, v, e);
  }
  if (lo > 0 && e > old) recode_rows<D>(codes, lo, old, e, lane, 32);
}

template <int D, typename T, typename Params>
int launch(Params p, bool one, int64_t slots, int device, cudaStream_t stream) {
  int units = 2 * p.s.kv_heads;
  if constexpr (std::is_same<Params, RotatedParams>::value) units += p.heads;
  if (one)
    return launch_kernel("emmy_kv8_append", append_one_kernel<D, T, Params>, dim3(p.s.seqs, (units + 3) / 4), 128, 0, stream, p);
  // several (side, head)s a CTA once there are more than fill the GPU twice
  const int threads = page_threads<D, T>(1 << p.s.page_shift);
  const int64_t fill = int64_t(sm_count(device)) * 2 * (2048 / threads < 7 ? 2048 / threads : 7);
  p.units = int(std::min<int64_t>(units, std::max<int64_t>(1, slots * units / std::max<int64_t>(fill, 1))));
  int smem = 2 * 8 * 16 * threads;
  constexpr int ROOM = 200 * 1024;
  if (smem > ROOM) smem /= 2, p.units = 1;  // no second buffer, so no second unit (f32 pages of 128 KB)
  static KernelSetup setup;
  const int rc = setup.ready("emmy_kv8_append", append_kernel<D, T, Params>, device,
                             std::min(ROOM, 2 * 8 * 16 * MOST_THREADS<D, T>));
  if (rc != EMMY_OK) return rc;
  return launch_kernel("emmy_kv8_append", append_kernel<D, T, Params>, dim3(unsigned(slots), (units + p.units - 1) / p.units),
                       threads, smem, stream, p);
}

template <int D, typename Params>
int launch_type(const Params &p, int dtype, bool one, int64_t slots, int device, cudaStream_t stream) {
  if (dtype == EMMY_KV8_F32) return launch<D, float>(p, one, slots, device, stream);
  if (dtype == EMMY_KV8_BF16) return launch<D, __nv_bfloat16>(p, one, slots, device, stream);
  return launch<D, __half>(p, one, slots, device, stream);
}

// What both calls check, and the parameters that they share.
int append_params(const char *what, const emmy_kv8 *cache, emmy_dptr k, emmy_dptr v, int32_t dtype, const int64_t k_strides[2],
                  const int64_t v_strides[2], AppendParams &p) {
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
  p.s = seqs_of(*cache);
  p.codes = reinterpret_cast<uint8_t *>(cache->codes);
  p.exps = reinterpret_cast<int8_t *>(cache->exps);
  p.x[0] = reinterpret_cast<const void *>(k);
  p.x[1] = reinterpret_cast<const void *>(v);
  p.ts[0] = k_strides[0], p.hs[0] = k_strides[1];
  p.ts[1] = v_strides[0], p.hs[1] = v_strides[1];
  return EMMY_OK;
}

template <typename Params>
int append(const char *what, const Params &p, const emmy_kv8 *cache, int32_t dtype, emmy_stream stream) {
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

}  // namespace
}  // namespace kv8

extern "C" int emmy_kv8_append(const emmy_kv8 *cache, emmy_dptr k, emmy_dptr v, int32_t dtype,
                               const int64_t k_strides[2], const int64_t v_strides[2],
                               emmy_stream stream) {
  using namespace kv8;
  static const char *what = "emmy_kv8_append";
  AppendParams p;
  const int rc = append_params(what, cache, k, v, dtype, k_strides, v_strides, p);
  if (rc != EMMY_OK || cache->tokens == 0 || cache->max_q == 0) return rc;
  return append(what, p, cache, dtype, stream);
}

extern "C" int emmy_kv8_append_rotated(const emmy_kv8 *cache, emmy_dptr k, emmy_dptr v, int32_t dtype,
                                       const int64_t k_strides[2], const int64_t v_strides[2],
                                       const emmy_rotary *rotary, const emmy_kv8_rotated_args *a,
                                       emmy_stream stream) {
  using namespace kv8;
  static const char *what = "emmy_kv8_append_rotated";
  RotatedParams p;
  const int rc = append_params(what, cache, k, v, dtype, k_strides, v_strides, p);
  if (rc != EMMY_OK) return rc;
  if (const char *msg = rotary_trouble(rotary)) return fail(EMMY_EINVAL, what, msg);
  if (rotary->head_dim != cache->head_dim) return fail(EMMY_EINVAL, what, "the rotary's head_dim is not the cache's");
  if (a == nullptr) return fail(EMMY_EINVAL, what, "null arguments");
  if (a->positions % (a->wide ? 8 : 4)) return fail(EMMY_EINVAL, what, "positions must be aligned to their type");
  if (a->heads < 0 || a->heads > 1 << 20) return fail(EMMY_EINVAL, what, "heads must be between 0 and 2^20");
  if (cache->tokens == 0 || cache->max_q == 0) return EMMY_OK;
  for (int i = 0; i < 64; ++i) p.frequency[i] = rotary->turns[i];
  p.positions = reinterpret_cast<const void *>(a->positions);
  p.position_stride = a->position_stride;
  p.wide = a->wide != 0;
  p.dims = rotary->dims, p.interleaved = rotary->interleaved != 0, p.gain = rotary->gain;
  p.heads = a->heads;
  if (a->heads > 0) {
    if (a->q == 0 || a->q_out == 0) return fail(EMMY_EINVAL, what, "null q or q_out");
    if (a->out_dtype != EMMY_KV8_F32 && a->out_dtype != EMMY_KV8_BF16 && a->out_dtype != EMMY_KV8_F16)
      return fail(EMMY_EINVAL, what, "q_out must be f32, bf16 or f16");
    const int size = dtype == EMMY_KV8_F32 ? 4 : 2, out_size = a->out_dtype == EMMY_KV8_F32 ? 4 : 2;
    const int64_t *qs = a->q_strides, *os = a->out_strides;
    if (a->q % 16 || a->q_out % 16 || qs[0] * size % 16 || qs[1] * size % 16 || os[0] * out_size % 16 || os[1] * out_size % 16)
      return fail(EMMY_EINVAL, what, "q and q_out: base and strides must be multiples of 16 bytes");
    const int64_t T = cache->tokens, H = a->heads, Hk = cache->kv_heads, D = cache->head_dim;
    const bool in_place = a->q == a->q_out && dtype == a->out_dtype && (T == 1 || qs[0] == os[0]) && (H == 1 || qs[1] == os[1]);
    const struct {
      emmy_dptr at;
      const int64_t *strides;
      int64_t heads;
      bool same;
    } inputs[3] = {{a->q, qs, H, in_place}, {k, k_strides, Hk, false}, {v, v_strides, Hk, false}};
    for (const auto &x : inputs) {
      const int bad = rows_trouble(x.at, x.strides, x.heads, size, a->q_out, os, H, out_size, T, D, x.same);
      if (bad != ROWS_FINE)
        return fail(EMMY_EINVAL, what, bad == ROWS_NEGATIVE ? "k, v, q and q_out: strides must not be negative"
                                       : bad == ROWS_SELF   ? "rows of q_out overlap"
                                                            : "q_out overlaps q, k or v");
    }
    p.q = reinterpret_cast<const void *>(a->q);
    p.out = reinterpret_cast<void *>(a->q_out);
    p.q_ts = qs[0], p.q_hs = qs[1], p.o_ts = os[0], p.o_hs = os[1];
    p.out_type = a->out_dtype;
  }
  return append(what, p, cache, dtype, stream);
}
