// Rotary positions on the device: angles and what turns a pair of values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "kv8.cuh"

namespace rotary {

// sin and cos of position * frequency, the frequency in 2^-64 turns a position.
// A multiple of 2^64 is a whole number of turns, so the product's low 64 bits are
// the angle: exact, but for the frequency's own rounding, at any position, where an
// f32 angle at position 131071 is off by 0.004.  What is left of the nearest
// quarter turn, at most an eighth of one, is rounded to f32 as a whole, so that small
// angles keep its precision (of the upper 32 bits alone, a frequency of 1e-9 does not
// turn position 1 at all), and goes through the Taylor series to x^9 and x^10, which
// are off by less than 2^-29 there.
__device__ __forceinline__ void turn_of(int64_t position, uint64_t frequency, float &c, float &s) {
  const uint64_t t = static_cast<uint64_t>(position) * frequency, quarter = (t + (uint64_t(1) << 61)) >> 62;
  // 2 pi 2^-64
  const float x = static_cast<float>(static_cast<int64_t>(t - (quarter << 62))) * 3.4061215800304705e-19f, y = x * x;
  const float sine = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
  const float cosine =
      fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
  c = quarter & 1 ? sine : cosine;
  s = quarter & 1 ? cosine : sine;
  if (quarter + 1 & 2) c = -c;
  if (quarter & 2) s = -s;
}

// The same to 2^-20, whatever the angle: it is at most pi, rounded three times on its
// way to f32 (3 * 2^-24 of it, 2^-20.8; its lowest bits, below 2^-32 turns, do not
// count), and the special function unit is off by at most 2^-21.2, as CUDA documents
// __cosf and __sinf there.  10 instructions for 45.  For results of 16 bits, which
// round by 2^-12 or more of the larger of a pair, and of 8: the smaller one, and what
// a small angle makes of it, is good to 2^-20 of the larger, not to its own last bit.
__device__ __forceinline__ void turn_near(int64_t position, uint64_t frequency, float &c, float &s) {
  const uint32_t t = static_cast<uint32_t>((static_cast<uint64_t>(position) * frequency) >> 32);
  const float x = static_cast<float>(static_cast<int32_t>(t)) * 1.4629180792671596e-9f;
  c = __cosf(x);
  s = __sinf(x);
}
template <bool EXACT>
__device__ __forceinline__ void turn(int64_t position, uint64_t frequency, float gain, float &c, float &s) {
  if constexpr (EXACT)
    turn_of(position, frequency, c, s);
  else
    turn_near(position, frequency, c, s);
  c *= gain, s *= gain;
}

// Two f32 in one register pair, and products of those: one instruction for two.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 apart(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
constexpr uint64_t SIGNS = 0x8000000080000000ull;
// (x, y) -> (x c - y s, x s + y c), two pairs at once; ns = -s.
__device__ __forceinline__ void turn2(uint64_t &x, uint64_t &y, uint64_t c, uint64_t s, uint64_t ns) {
  const uint64_t a = fma2(x, c, mul2(y, ns));
  y = fma2(x, s, mul2(y, c));
  x = a;
}

// Rows to turn: those of a call by themselves, or a cache's new tokens.
struct Params {
  uint64_t frequency[EMMY_ROTARY_PAIRS];
  const void *x;
  void *out;
  const void *positions;  // null: first, first + 1, .., or the places in the sequences
  int64_t first, position_stride, tokens;
  int64_t x_ts, x_hs, o_ts, o_hs;  // token and head strides, elements
  int heads, dims, head_dim;
  int pieces, turned;     // pieces of a head that threads hold (with those paired with them), those turned
  int slices;             // of a token's heads: thread slice i has heads i, i + slices, ..
  int width;              // threads of a token
  int block_rows;         // rows of a block that takes whole ones
  bool wide, interleaved, copy;
  float gain, sign;
  kv8::Seqs s;            // s.seqs = 0: no sequences
};
// Launches on the current device; types are EMMY_KV8_F32 and so on.
int rotate_rows(const char *what, Params &p, int type, int out_type, cudaStream_t stream);

// N neighbouring values as one access of at most 16 bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) Piece {
  T v[N];
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T rounded(float x);
template <>
__device__ __forceinline__ float rounded<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half rounded<__half>(float x) { return __float2half_rn(x); }

// The same value, or rounded where the types differ.
template <typename U, typename T>
__device__ __forceinline__ U as_type(T x) {
  if constexpr (std::is_same<T, U>::value)
    return x;
  else
    return rounded<U>(to_float(x));
}

// Two neighbouring values of a 32-bit word, and back with one rounding each.
template <typename T>
__device__ __forceinline__ float2 unpacked(uint32_t w) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(0.0f, 0.0f);  // a word is one value
  } else if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  } else {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}
template <typename T>
__device__ __forceinline__ uint32_t packed(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}

// Piece a's values, two to a register pair, and back with one rounding each.
template <typename T, int N>
__device__ __forceinline__ void spread(const Piece<T, N> &a, uint64_t (&x)[N / 2]) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if constexpr (sizeof(T) == 2) {
      const float2 f = unpacked<T>(reinterpret_cast<const uint32_t *>(&a)[i]);
      x[i] = two(f.x, f.y);
    } else {
      x[i] = two(a.v[2 * i], a.v[2 * i + 1]);
    }
  }
}
template <typename U, int N>
__device__ __forceinline__ void gathered(const uint64_t (&x)[N / 2], Piece<U, N> &u) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 f = apart(x[i]);
    if constexpr (sizeof(U) == 2)
      reinterpret_cast<uint32_t *>(&u)[i] = packed<U>(f.x, f.y);
    else
      u.v[2 * i] = f.x, u.v[2 * i + 1] = f.y;
  }
}

// (a, b) turned into (u, v), of pieces a and b whose values pair up (half layout),
// or of one piece a of neighbours; c, s of each pair.
template <typename T, typename U, int N>
__device__ __forceinline__ void turn_pieces(const Piece<T, N> &a, const Piece<T, N> &b, const float (&c)[N], const float (&s)[N],
                                            Piece<U, N> &u, Piece<U, N> &v) {
  if constexpr (N >= 2) {
    uint64_t x[N / 2], y[N / 2];
    spread<T, N>(a, x);
    spread<T, N>(b, y);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint64_t s2 = two(s[2 * i], s[2 * i + 1]);
      turn2(x[i], y[i], two(c[2 * i], c[2 * i + 1]), s2, s2 ^ SIGNS);
    }
    gathered<U, N>(x, u);
    gathered<U, N>(y, v);
  } else {
    const float x = to_float(a.v[0]), y = to_float(b.v[0]);
    u.v[0] = rounded<U>(x * c[0] - y * s[0]);
    v.v[0] = rounded<U>(x * s[0] + y * c[0]);
  }
}
template <typename T, typename U, int N>
__device__ __forceinline__ void turn_neighbours(const Piece<T, N> &a, const float (&c)[N / 2], const float (&s)[N / 2], Piece<U, N> &u) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, U>::value) {
    const uint32_t *x = reinterpret_cast<const uint32_t *>(&a);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 p = unpacked<T>(x[i]);
      reinterpret_cast<uint32_t *>(&u)[i] = packed<T>(p.x * c[i] - p.y * s[i], p.x * s[i] + p.y * c[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float x = to_float(a.v[2 * i]), y = to_float(a.v[2 * i + 1]);
      u.v[2 * i] = rounded<U>(x * c[i] - y * s[i]);
      u.v[2 * i + 1] = rounded<U>(x * s[i] + y * c[i]);
    }
  }
}

// Heads of a thread: as many as are eight loads.
template <bool INTERLEAVED>
constexpr int heads_of = INTERLEAVED ? 8 : 4;

// Place of a new token in its sequence; false: it is in none that can be.
__device__ __forceinline__ bool place_of(const kv8::Seqs &s, int64_t token, int64_t &place) {
  int lo = 0, hi = s.seqs - 1;  // the last sequence that begins at or before it
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.q_starts[mid] <= token) lo = mid; else hi = mid - 1;
  }
  int start, n, len;
  kv8::lengths(s, lo, start, n, len);
  place = len - n + token - start;
  return token >= start && token < int64_t(start) + n;
}

// The work of one block of `threads` threads; frequency(i) is pair i's.
template <typename T, typename U, int N, bool INTERLEAVED, typename F>
__device__ __forceinline__ void rotate_block(const Params &p, const F &frequency, int64_t block, int threads) {
  using P = Piece<T, N>;
  using O = Piece<U, N>;
  constexpr int HEADS = heads_of<INTERLEAVED>;
  constexpr int PAIRS = INTERLEAVED ? N / 2 : N;  // that a thread holds
  // a thread a (token, heads slice, piece)
  const int64_t at_all = block * threads + threadIdx.x, all = p.tokens * p.width;
  if (at_all >= all) return;
  const int64_t token = all <= 0x7fffffff ? int64_t(unsigned(at_all) / unsigned(p.width)) : at_all / p.width;
  const int of_token = int(at_all - token * p.width), slice = of_token / p.pieces, piece = of_token - slice * p.pieces;
  // single values of an interleaved row: pairs are neighbours all the same
  const bool near = N == 1 && p.interleaved, turned = piece < p.turned;
  const int at = near && turned ? 2 * piece : INTERLEAVED || turned ? piece * N : p.dims + (piece - p.turned) * N;
  const int other = at + (near ? 1 : p.dims / 2);
  const T *x = static_cast<const T *>(p.x) + token * p.x_ts;
  U *out = static_cast<U *>(p.out) + token * p.o_ts;
  // on their way while the position is looked up and the angles are computed
  P a[HEADS], b[INTERLEAVED ? 1 : HEADS];
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const int h = slice + j * p.slices;
    if (h >= p.heads) continue;
    a[j] = *reinterpret_cast<const P *>(x + h * p.x_hs + at);
    if constexpr (!INTERLEAVED)
      if (turned) b[j] = *reinterpret_cast<const P *>(x + h * p.x_hs + other);
  }
  int64_t pos = p.first + token;
  if (p.s.seqs > 0 && !place_of(p.s, token, pos)) return;
  if (p.positions != nullptr)
    pos = p.wide ? static_cast<const int64_t *>(p.positions)[token * p.position_stride]
                 : static_cast<const int *>(p.positions)[token * p.position_stride];
  float c[PAIRS], s[PAIRS];
  if (turned) {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      turn<sizeof(U) == 4>(pos, frequency(piece * PAIRS + i), p.gain, c[i], s[i]);
      s[i] *= p.sign;
    }
  }
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const int h = slice + j * p.slices;
    if (h >= p.heads) continue;
    O u, v;
    if (turned) {
      if constexpr (INTERLEAVED) {
        turn_neighbours<T, U, N>(a[j], c, s, u);
        if (at + N > p.dims)  // the last turned ones share a piece with those behind
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (at + i >= p.dims) u.v[i] = as_type<U>(a[j].v[i]);
      } else
        turn_pieces<T, U, N>(a[j], b[j], c, s, u, v);
      if constexpr (!INTERLEAVED) *reinterpret_cast<O *>(out + h * p.o_hs + other) = v;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) u.v[i] = as_type<U>(a[j].v[i]);
    }
    *reinterpret_cast<O *>(out + h * p.o_hs + at) = u;
  }
}

// How a call's rows go to blocks of `threads` threads; returns how many.
template <int N, bool INTERLEAVED>
int64_t shape_blocks(Params &p, int threads) {
  constexpr int HEADS = heads_of<INTERLEAVED>;
  p.turned = INTERLEAVED ? (p.dims + N - 1) / N : p.dims / 2 / N;
  p.pieces = !p.copy ? p.turned : INTERLEAVED ? p.head_dim / N : p.turned + (p.head_dim - p.dims) / N;
  p.slices = (p.heads + HEADS - 1) / HEADS;
  p.width = p.slices * p.pieces;  // at most 2^18 * 512
  return (p.tokens * p.width + threads - 1) / threads;
}

}  // namespace rotary
