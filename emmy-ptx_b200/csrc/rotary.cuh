// Rotary positions on the device: angles and what turns a pair of values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace rotary {

// sin and cos of position * frequency, the frequency in 2^-64 turns a position.
// A multiple of 2^64 is a whole number of turns, so the product's low 64 bits are
// the angle: exact, but for the frequency's own rounding, at any position, where an
// f32 angle at position 131071 is off by 0.004.  What is left of the nearest
// quarter turn, at most an eighth of one, goes through the Taylor series to x^9
// and x^10, which are off by less than 2^-29 there.
__device__ __forceinline__ void turn_of(int64_t position, uint64_t frequency, float &c, float &s) {
  const uint32_t t = static_cast<uint32_t>((static_cast<uint64_t>(position) * frequency) >> 32);
  const uint32_t quarter = (t + 0x20000000u) >> 30;
  // 2 pi 2^-32
  const float x = static_cast<float>(static_cast<int32_t>(t - (quarter << 30))) * 1.4629180792671596e-9f, y = x * x;
  const float sine = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
  const float cosine =
      fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
  c = quarter & 1 ? sine : cosine;
  s = quarter & 1 ? cosine : sine;
  if (quarter + 1 & 2) c = -c;
  if (quarter & 2) s = -s;
}

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

}  // namespace rotary
