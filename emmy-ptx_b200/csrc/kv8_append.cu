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
// way, in f32 and unrounded, and queries turned into an array of their own: where
// no sequence has more than one new token they are more (query head)s behind the
// (side, head)s, else blocks behind the pages' that do what emmy_rotate does.  In a
// page's rows a key's angle is that of a thread's first row and a multiple of the rows
// between: cos(a + b) = cos a cos b - sin a sin b, with the first angle in registers
// and the multiples' in shared memory, 4 products a pair (an angle's function each
// value: 854 us, so 173, for the case below).  Sines and cosines are good to 2^-18 of
// the values, whose codes are rounded by 2^-4.  41536 tokens in 6 sequences, 8 heads
// and 32 query heads of 128, bf16: 141 us, 6.5 TB/s; the queries' blocks mixed with
// the pages' 164, before them 160, in a launch of their own 157.  One token 2.3 us, 64
// of as many sequences 3.3.
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
  int head_dim;
  bool wide, interleaved, copy;  // copy: q_out is not q
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
template <typename T>
constexpr int type_of = sizeof(T) == 4 ? EMMY_KV8_F32 : std::is_same<T, __half>::value ? EMMY_KV8_F16 : EMMY_KV8_BF16;

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

// Values col .. col + 15 bytes of a row in shared memory, as the frequencies are,
// turned one by one.
template <bool EXACT, typename T>
__device__ __forceinline__ void turn_apart(const RotatedParams &p, const uint64_t *frequency, const T *row, int col, int64_t pos,
                                           float *y) {
  const int half = p.dims / 2;
#pragma unroll
  for (int i = 0; i < Vec<T>::N; ++i) {
    const int at = col + i;
    y[i] = rotary::to_float(row[at]);
    if (at >= p.dims) continue;
    const bool low = p.interleaved ? at % 2 == 0 : at < half;
    const int away = p.interleaved ? 1 : half, other = low ? at + away : at - away;
    float c, s;
    rotary::turn<EXACT>(pos, frequency[p.interleaved ? at / 2 : low ? at : other], p.gain, c, s);
    y[i] = y[i] * c + rotary::to_float(row[other]) * (low ? -s : s);
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

// How a page's keys are turned: the pairs of a piece in another whole piece, or
// within it, at their places in the sequence; or in any other way.
enum { HALVES, NEIGHBOURS, ANY };

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Keys and values by pages, and behind their blocks those of the queries' rows: blocks
// that compute go first, and those that copy fill the end.
struct MixedParams {
  RotatedParams kv;
  rotary::Params q;
  int page_blocks, kv_blocks, blocks;  // blocks of a page; of all pages, and with the queries'
};

// append_kernel with keys turned on the way.  A thread's pieces of a row are two
// that pair up (or, at the end of a row with fewer dims, two of those behind), of
// half as many rows; it holds their values as f32 through the maximum.  Bound by
// instructions as much as by memory: two values an instruction where there is one
// for that, angles by steps, (side, head)s in turn so that blocks are alike.
template <int D, typename T, int MODE, int ROWS, int MOST>
__global__ void __launch_bounds__(MOST, ROWS == 2 && MOST == 256 ? 3 : 1) append_turned_kernel(const __grid_constant__ MixedParams all) {
  const RotatedParams &p = all.kv;
  using V = Vec<T>;
  using P = rotary::Piece<T, V::N>;
  using rotary::mul2, rotary::fma2, rotary::two, rotary::apart;
  constexpr int N = V::N, HALF = N / 2, LPR = D / N, LANES = LPR / 2;
  extern __shared__ uint4 pieces[];  // [2] pages' rows
  __shared__ float part[2][32];
  __shared__ __align__(16) float steps_c[MODE == ANY ? 1 : ROWS][D / 2], steps_s[MODE == ANY ? 1 : ROWS][D / 2];
  const Seqs &s = p.s;
  // (lanes read other frequencies each, which kernel parameters serve one by one)
  __shared__ uint64_t frequency[D / 2];
  if (threadIdx.x < D / 2) frequency[threadIdx.x] = p.frequency[threadIdx.x];
  __syncthreads();
  grid_dependency_wait();
  grid_dependency_done();
  const int kv_block = blockIdx.x;
  if (kv_block >= all.kv_blocks) {
    if constexpr (MODE != ANY) rotary::rotate_block<T, T, N, MODE == NEIGHBOURS>(
          all.q, [&](int i) { return frequency[i]; }, kv_block - all.kv_blocks, blockDim.x);
    return;
  }
  const int nth_page = kv_block / all.page_blocks, nth = kv_block - nth_page * all.page_blocks;
  int b, start, n, len, page_of_seq;
  if (!owner(s, nth_page, b, start, n, len, page_of_seq)) return;
  const int size = 1 << s.page_shift, first = len - n, H = s.kv_heads;
  const int page = s.table[int64_t(b) * s.width + page_of_seq];
  const int pos0 = page_of_seq << s.page_shift;
  const int lo = max(first - pos0, 0), hi = min(len - pos0, size);  // new rows of the page
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  int col = lane % LANES * N, col2 = col + D / 2;
  bool pairs = true;  // the pieces are turned
  if constexpr (MODE == HALVES) {
    const int half = p.dims / 2, behind = lane % LANES - half / N;
    pairs = behind < 0;
    if (!pairs) col = p.dims + behind * N;
    col2 = pairs ? col + half : col + (D - p.dims) / 2;
  }
  // of the new rows
  const int row0 = warp * (32 / LANES) + lane / LANES, step = warps * (32 / LANES), away = col2 - col;
  const int64_t token0 = int64_t(start) + pos0 - first;  // row 0 of the page, were it new
  const int mine = row0 * LPR + col / N, buffer = ROWS * step * LPR;
  const auto fetch = [&](int u, int buf) {
    const int side = u & 1, head = u >> 1;
    const int64_t ts = side ? p.ts[1] : p.ts[0];
    const T *x = static_cast<const T *>(side ? p.x[1] : p.x[0]) + head * (side ? p.hs[1] : p.hs[0]) + col;
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(pieces + buf * buffer + mine));
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = lo + row0 + i * step;
      const bool real = r < hi;
      const T *from = x + (token0 + (real ? r : lo)) * ts;
      copy16(to + i * step * (D * int(sizeof(T))), from, real);
      copy16(to + (i * step * D + away) * int(sizeof(T)), from + away, real);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int u0 = nth * p.units, u1 = min(u0 + p.units, 2 * H);
  fetch(u0, 0);
  const bool bad = page < 0 || page >= s.pages;
  if (bad && tid == 0) report(s.status, STATUS_PAGE);
  const int64_t unit0 = int64_t(bad ? 0 : page) * 2 * H;
  const auto unit_of = [&](int u) { return unit0 + (u & 1 ? H : 0) + (u >> 1); };
  int held = lo > 0 ? p.exps[unit_of(u0)] : 0;
  // angles of keys: of row lo + row0, and of i * step rows
  uint64_t first_c[HALF], first_s[HALF];
  const auto pair_at = [&](int j) { return MODE == HALVES ? col + j : (j < HALF ? col : col2 - N) / 2 + j; };
  if (MODE != ANY && (u1 - u0 > 1 || u0 % 2 == 0)) {  // there are keys
    for (int i = tid; i < ROWS * (D / 2); i += threads) {
      const int row = i / (D / 2), pair = i % (D / 2);
      rotary::turn_of(int64_t(row) * step, frequency[pair], steps_c[row][pair], steps_s[row][pair]);
    }
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      float c[2], s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) rotary::turn<false>(pos0 + lo + row0, frequency[min(pair_at(j + i), D / 2 - 1)], p.gain, c[i], s[i]);
      first_c[j / 2] = two(c[0], c[1]);
      first_s[j / 2] = two(s[0], s[1]);
    }
    __syncthreads();
  }
  for (int u = u0; u < u1; ++u) {
    const int buf = (u - u0) & 1, old = lo > 0 ? held_exponent(held) : E_MIN;
    if (u + 1 < u1) {
      fetch(u + 1, buf ^ 1);
      held = lo > 0 ? p.exps[unit_of(u + 1)] : 0;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // every thread reads only the pieces it copied
    const uint4 *rows = pieces + buf * buffer + mine;
    const bool turn = (u & 1) == 0;
    uint64_t x[ROWS][HALF], y[ROWS][HALF];
    float amax = 0.0f;
    if (MODE == ANY && turn) __syncwarp();  // but for these, paired with any value of a row that their warp copied
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = lo + row0 + i * step;
      if (r >= hi) continue;
      const uint4 *at = rows + i * step * LPR;
      if (MODE == ANY && turn) {
        float v[2 * N];
        const T *row = reinterpret_cast<const T *>(at - col / N);
        const int64_t pos = position_of(p, token0 + r, pos0 + r);
        turn_apart<false>(p, frequency, row, col, pos, &v[0]);
        turn_apart<false>(p, frequency, row, col2, pos, &v[N]);
#pragma unroll
        for (int j = 0; j < HALF; ++j) x[i][j] = two(v[2 * j], v[2 * j + 1]), y[i][j] = two(v[N + 2 * j], v[N + 2 * j + 1]);
      } else {
        rotary::spread<T, N>(*reinterpret_cast<const P *>(at), x[i]);
        rotary::spread<T, N>(*reinterpret_cast<const P *>(at + away / N), y[i]);
      }
      if (MODE == HALVES && turn && pairs) {
#pragma unroll
        for (int j = 0; j < HALF; ++j) {
          const float2 bc = *reinterpret_cast<const float2 *>(&steps_c[i][col + 2 * j]);
          const float2 bs = *reinterpret_cast<const float2 *>(&steps_s[i][col + 2 * j]);
          const uint64_t c2 = two(bc.x, bc.y), s2 = two(bs.x, bs.y);
          const uint64_t c = fma2(first_c[j], c2, mul2(first_s[j], s2 ^ rotary::SIGNS));
          const uint64_t s = fma2(first_s[j], c2, mul2(first_c[j], s2));
          rotary::turn2(x[i][j], y[i][j], c, s, s ^ rotary::SIGNS);
        }
      }
      if (MODE == NEIGHBOURS && turn) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int pair = pair_at(j);
          if (2 * pair >= p.dims) continue;
          const float2 fc = apart(first_c[j / 2]), fs = apart(first_s[j / 2]);
          const float c0 = j & 1 ? fc.y : fc.x, s0 = j & 1 ? fs.y : fs.x, bc = steps_c[i][pair], bs = steps_s[i][pair];
          const float c = c0 * bc - s0 * bs, s = s0 * bc + c0 * bs;
          uint64_t &w = j < HALF ? x[i][j] : y[i][j - HALF];
          const float2 f = apart(w);
          w = two(f.x * c - f.y * s, f.x * s + f.y * c);
        }
      }
#pragma unroll
      for (int j = 0; j < HALF; ++j) {
        const float2 f = apart(x[i][j]), g = apart(y[i][j]);
        amax = max3(amax, fabsf(f.x), fabsf(f.y));
        amax = max3(amax, fabsf(g.x), fabsf(g.y));
      }
    }
    if (MODE == ANY && turn) __syncwarp();  // before this buffer's next copies
    if (amax == INFINITY) {  // (rare) the largest finite one
      amax = 0.0f;
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (lo + row0 + i * step < hi)
#pragma unroll
          for (int j = 0; j < HALF; ++j) {
            const float2 f = apart(x[i][j]), g = apart(y[i][j]);
            const float v[4] = {f.x, f.y, g.x, g.y};
            amax = max_finite(v, amax);
          }
    }
    amax = warp_max(amax);
    if (lane == 0) part[buf][warp] = amax;
    __syncthreads();
    amax = warp_max(lane < warps ? part[buf][lane] : 0.0f);
    if (bad) continue;
    const int e = fit_exponent(amax, old);
    const int64_t unit = unit_of(u);
    uint8_t *codes = p.codes + (unit << s.page_shift) * D;
    if (tid == 0) p.exps[unit] = int8_t(e);
    const uint64_t by = two(pow2(-e), pow2(-e));
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = lo + row0 + i * step;
      if (r >= hi) continue;
      uint32_t w[2][2] = {};
#pragma unroll
      for (int j = 0; j < HALF; ++j) {
        const float2 f = apart(mul2(x[i][j], by)), g = apart(mul2(y[i][j], by));
        w[0][j / 2] |= f32x2_e4m3x2(f.y, f.x) << (16 * (j & 1));
        w[1][j / 2] |= f32x2_e4m3x2(g.y, g.x) << (16 * (j & 1));
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint8_t *at = codes + r * D + (k == 0 ? col : col2);
        if constexpr (N == 8)
          *reinterpret_cast<uint2 *>(at) = make_uint2(w[k][0], w[k][1]);
        else
          *reinterpret_cast<uint32_t *>(at) = w[k][0];
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
  // (lanes read other frequencies each, which kernel parameters serve one by one:
  // once a block, while the kernel before this one ends)
  __shared__ uint64_t frequency[ROTATED ? D / 2 : 1];
  if constexpr (ROTATED) {
    if (threadIdx.x < D / 2) frequency[threadIdx.x] = p.frequency[threadIdx.x];
    __syncthreads();
  }
  grid_dependency_wait();
  grid_dependency_done();
  const int b = blockIdx.x, unit_of_seq = (blockIdx.z * gridDim.y + blockIdx.y) * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
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
  const bool bad = page < 0 || page >= s.pages;
  const int64_t unit = (int64_t(bad ? 0 : page) * 2 + side) * s.kv_heads + head;
  const int lo = (len - 1) & ((1 << s.page_shift) - 1);
  const int held = lo > 0 && !query ? p.exps[unit] : 0;
  float turned[V::N];
  bool turn = false;
  if constexpr (ROTATED) {
    turn = unit_of_seq < s.kv_heads || query;
    if (turn) {
      constexpr int N = V::N;
      const int col = lane * N, half = p.dims / 2;
      // pieces whose values pair up with each other's or within: angles while the
      // values are on their way
      const bool whole = (p.interleaved || half % N == 0) && !(query && p.out_type == EMMY_KV8_F32), low = col < half;
      const int64_t pos = position_of(p, start, len - 1);
      float c[N], sn[N];
      if (whole && lane < LPR && col < p.dims) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (p.interleaved && j % 2 == 1) continue;
          const int pair = p.interleaved ? (col + j) / 2 : (low ? col : col - half) + j;
          rotary::turn<false>(pos, frequency[pair], p.gain, c[j], sn[j]);
        }
      }
      __shared__ uint4 rows[4][LPR];
      uint4 *row = rows[threadIdx.x >> 5];
      if (lane < LPR) row[lane] = v.w;
      __syncwarp();
      if (lane < LPR) {
        if (!whole) {
          if (query && p.out_type == EMMY_KV8_F32)
            turn_apart<true>(p, frequency, reinterpret_cast<const T *>(row), col, pos, turned);
          else
            turn_apart<false>(p, frequency, reinterpret_cast<const T *>(row), col, pos, turned);
        } else {
          V other;
          other.w = p.interleaved || col >= p.dims ? v.w : row[(low ? col + half : col - half) / N];
#pragma unroll
          for (int j = 0; j < N; ++j) {
            turned[j] = v.at(j);
            if (p.interleaved) {
              if (j % 2 == 1 && col + j < p.dims) {
                const float x = v.at(j - 1), y = v.at(j);
                turned[j - 1] = x * c[j - 1] - y * sn[j - 1];
                turned[j] = x * sn[j - 1] + y * c[j - 1];
              }
            } else if (col < p.dims) {
              turned[j] = turned[j] * c[j] + other.at(j) * (low ? -sn[j] : sn[j]);
            }
          }
        }
      }
      if (query) {
        if (lane < LPR) store_query(p, start, unit_of_seq - 2 * s.kv_heads, col, turned);
        return;
      }
    }
  }
  if (bad) {
    report(s.status, STATUS_PAGE);
    return;
  }
  uint8_t *codes = p.codes + (unit << s.page_shift) * D;
  const int old = lo > 0 ? held_exponent(held) : E_MIN;
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

// Whether the queries of pages go with their keys and values: at their places, of
// the same type, in whole pieces.  (Others are a launch of the row kernel's.)
template <typename T>
bool mixes(const RotatedParams &p) {
  constexpr int N = Vec<T>::N;
  return p.heads > 0 && p.positions == nullptr && p.out_type == type_of<T> && (p.interleaved || p.dims / 2 % N == 0);
}

// The queries as rows to turn.
rotary::Params query_rows(const RotatedParams &p) {
  rotary::Params r = {};
  for (int i = 0; i < 64; ++i) r.frequency[i] = p.frequency[i];
  r.x = p.q, r.out = p.out;
  r.positions = p.positions, r.position_stride = p.position_stride, r.wide = p.wide;
  r.tokens = p.s.tokens;
  r.x_ts = p.q_ts, r.x_hs = p.q_hs, r.o_ts = p.o_ts, r.o_hs = p.o_hs;
  r.heads = p.heads, r.dims = p.dims, r.head_dim = p.head_dim;
  r.interleaved = p.interleaved, r.copy = p.copy;
  r.gain = p.gain, r.sign = 1.0f;
  r.s = p.s;
  r.s.status = nullptr;  // the keys' blocks report what is wrong with the lengths
  return r;
}

template <int D, typename T, typename Params>
int launch(Params p, bool one, int64_t slots, int device, cudaStream_t stream) {
  int units = 2 * p.s.kv_heads;
  if constexpr (std::is_same<Params, RotatedParams>::value)
    if (one) units += p.heads;
  if (one) {
    // (2^20 query heads are more than a grid's second dimension takes)
    const int blocks = (units + 3) / 4, y = std::min(blocks, 65535);
    return launch_kernel("emmy_kv8_append", append_one_kernel<D, T, Params>, dim3(p.s.seqs, y, (blocks + y - 1) / y), 128, 0, stream, p);
  }
  // several (side, head)s a CTA once there are more than fill the GPU twice
  int threads = page_threads<D, T>(1 << p.s.page_shift);
  // no more rows than a sequence has new ones
  if constexpr (std::is_same<Params, RotatedParams>::value)
    while (threads > 64 && int64_t(p.s.max_q) * D * int(sizeof(T)) / 128 <= threads / 2) threads /= 2;
  int64_t fill = int64_t(sm_count(device)) * 2 * (2048 / threads < 7 ? 2048 / threads : 7);
  if constexpr (std::is_same<Params, RotatedParams>::value) fill = int64_t(sm_count(device)) * 2 * std::max(768 / (2 * threads), 1);
  p.units = int(std::min<int64_t>(units, std::max<int64_t>(1, slots * units / std::max<int64_t>(fill, 1))));
  int smem = 2 * 8 * 16 * threads;
  constexpr int ROOM = 200 * 1024;
  if (smem > ROOM) smem /= 2, p.units = 1;  // no second buffer, so no second unit (f32 pages of 128 KB)
  constexpr int MOST = MOST_THREADS<D, T>;
  const int page_blocks = (units + p.units - 1) / p.units;
  if constexpr (std::is_same<Params, RotatedParams>::value) {
    MixedParams m;
    m.kv = p;
    m.page_blocks = page_blocks;
    if (slots * page_blocks > 0x7fffffff) return fail(EMMY_EINVAL, "emmy_kv8_append_rotated", "too many tokens and heads");
    m.kv_blocks = m.blocks = int(slots * page_blocks);
    const auto run = [&](auto kernel, KernelSetup &setup, int by) {
      const int rc = setup.ready("emmy_kv8_append_rotated", kernel, device, std::min(ROOM, 2 * 8 * 16 * MOST));
      if (rc != EMMY_OK) return rc;
      return launch_kernel("emmy_kv8_append_rotated", kernel, dim3(m.blocks), by * threads, smem, stream, m);
    };
    static KernelSetup setup[9];
    const auto pick = [&](auto mode, KernelSetup *of) {
      constexpr int M = decltype(mode)::value;
      const int by = 2 * threads <= 512 ? 2 : 1;
      if constexpr (M != ANY)
        if (mixes<T>(p)) {
          m.q = query_rows(p);
          const int64_t rows = rotary::shape_blocks<Vec<T>::N, M == NEIGHBOURS>(m.q, by * threads);
          if (m.kv_blocks + rows > 0x7fffffff) return fail(EMMY_EINVAL, "emmy_kv8_append_rotated", "too many tokens and heads");
          m.blocks = int(m.kv_blocks + rows);
        }
      if (2 * threads <= 256) return run(append_turned_kernel<D, T, M, 2, 256>, of[0], 2);
      if constexpr (2 * MOST > 512)
        if (2 * threads > 512) return run(append_turned_kernel<D, T, M, 4, MOST>, of[2], 1);
      return run(append_turned_kernel<D, T, M, 2, 512>, of[1], 2);
    };
    if (p.positions == nullptr && p.interleaved) return pick(std::integral_constant<int, NEIGHBOURS>(), setup);
    if (p.positions == nullptr && p.dims / 2 % Vec<T>::N == 0) return pick(std::integral_constant<int, HALVES>(), setup + 3);
    return pick(std::integral_constant<int, ANY>(), setup + 6);
  } else {
    static KernelSetup setup;
    const int rc = setup.ready("emmy_kv8_append", append_kernel<D, T>, device, std::min(ROOM, 2 * 8 * 16 * MOST));
    if (rc != EMMY_OK) return rc;
    return launch_kernel("emmy_kv8_append", append_kernel<D, T>, dim3(unsigned(slots), page_blocks), threads, smem, stream, p);
  }
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
  p.head_dim = cache->head_dim;
  p.copy = a->q != a->q_out;
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
  const int rc2 = append(what, p, cache, dtype, stream);
  if (rc2 != EMMY_OK || a->heads == 0 || cache->max_q == 1 || (dtype == EMMY_KV8_F32    ? mixes<float>(p)
                                                               : dtype == EMMY_KV8_BF16 ? mixes<__nv_bfloat16>(p)
                                                                                        : mixes<__half>(p)))
    return rc2;
  rotary::Params r = query_rows(p);
  const OnDevice on(cache->device);
  if (on.err != cudaSuccess) return cuda_fail(what, on.err);
  return rotary::rotate_rows(what, r, dtype, a->out_dtype, static_cast<cudaStream_t>(stream));
}
