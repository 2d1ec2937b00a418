// emmy_rotate -- rotary positions of queries or keys, and their gradients.
//
// The first `dims` values of each head are pairs (a, b), neighbours or half of
// `dims` apart; pair i of a token at position p becomes
//   gain * (a cos(p f_i) - b sin(p f_i), a sin(p f_i) + b cos(p f_i)),
// backward with -sin: the map is linear, and that is its transpose.  Values are
// turned in f32 and rounded once, at the end.
//
// Bound by memory: each value is read and written once.  A thread holds one piece
// (16 bytes, or less where sizes or addresses ask for it) of a token's row, with
// the piece that it is paired with, and does the same of HEADS heads: their angles
// are computed once, while the values are on their way (8191 tokens of 32 heads of
// 128, bf16: 34 us with the loads behind the angles, 24 before them, 22 with sines and
// cosines of 16-bit results from the special function unit; a copy takes 20.5).
// 32768 tokens of 16 heads: 40.6 us, 6.6 TB/s; 4093 of 20 heads of 80, f32, which stay
// in L2: 9.2 us; one token: 2.3.
#include "rotary.cuh"

namespace rotary {
namespace {

constexpr int THREADS = 256;

template <typename T, typename U, int N, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) rotate_kernel(const __grid_constant__ Params p) {
  kv8::grid_dependency_wait();
  kv8::grid_dependency_done();
  // (through shared memory the frequencies would hold up the values: 25.6 us a prompt
  // of 8191 tokens and 32 heads for 21.8)
  rotate_block<T, U, N, INTERLEAVED>(p, [&](int i) { return p.frequency[i]; }, blockIdx.x, THREADS);
}

template <typename T, typename U, int N, bool INTERLEAVED>
int launch(const char *what, Params &p, cudaStream_t stream) {
  const int64_t blocks = shape_blocks<N, INTERLEAVED>(p, THREADS);
  if (blocks > 0x7fffffff) return kv8::fail(EMMY_EINVAL, what, "too many tokens and heads");
  return kv8::launch_kernel(what, rotate_kernel<T, U, N, INTERLEAVED>, dim3(unsigned(blocks)), THREADS, 0, stream, p);
}

// Halves whose values pair up across pieces: rows go through shared memory, piece by
// piece as they lie, and a thread turns its own values with those that it finds
// there.  A block takes whole rows: so many (token, heads slice, slice + slices, ..)
// of `pieces` threads each; a row's threads compute the angle of each of its pairs
// once, and those whose pieces are not turned copy them as they come.  (Pairs of single
// values instead: 6333 tokens of 4 heads of 80 with 6 turned, bf16, 10 us, so 3.8; a
// thread its own values' angles, most of which idle threads wait for: 8191 tokens of
// 32 heads of 128 with 20 or 116 turned 50, so 32 and 35, a few tokens 4.2, so 2.7.
// Words of pieces apart, with no bank conflicts but 34 KB a block: 41 and 44.)
template <typename T, typename U, int N>
__global__ void __launch_bounds__(THREADS) rotate_apart_kernel(const __grid_constant__ Params p) {
  using P = Piece<T, N>;
  constexpr int HEADS = 4;
  __shared__ P rows[HEADS][THREADS];
  __shared__ float2 turns[THREADS * N / 2];  // (c, s) of each pair of each row
  __shared__ uint64_t frequency[EMMY_ROTARY_PAIRS];
  const int tid = threadIdx.x, r = tid / p.pieces, piece = tid - r * p.pieces, half = p.dims / 2;
  if (tid < half) frequency[tid] = p.frequency[tid];
  kv8::grid_dependency_wait();
  kv8::grid_dependency_done();
  const int64_t unit = int64_t(blockIdx.x) * p.block_rows + r, token = unit / p.slices;
  const int slice = int(unit - token * p.slices);
  const bool real = r < p.block_rows && token < p.tokens;
  const T *x = static_cast<const T *>(p.x) + token * p.x_ts + piece * N;
  U *out = static_cast<U *>(p.out) + token * p.o_ts + piece * N;
  P a[HEADS];
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const int h = slice + j * p.slices;
    if (real && h < p.heads) a[j] = *reinterpret_cast<const P *>(x + h * p.x_hs);
  }
  int64_t pos = p.first + token;
  bool placed = real;
  if (real && p.s.seqs > 0) placed = place_of(p.s, token, pos);
  if (real && p.positions != nullptr)
    pos = p.wide ? static_cast<const int64_t *>(p.positions)[token * p.position_stride]
                 : static_cast<const int *>(p.positions)[token * p.position_stride];
  __syncthreads();
  float2 *const mine = turns + r * half;
  if (real)
#pragma unroll 1
    for (int i = piece; i < half; i += p.pieces) {
      float c, s;
      turn<sizeof(U) == 4>(pos, frequency[i], p.gain, c, s);
      mine[i] = make_float2(c, p.sign * s);
    }
#pragma unroll
  for (int j = 0; j < HEADS; ++j)
    if (real && slice + j * p.slices < p.heads) rows[j][tid] = a[j];
  if (placed && p.copy && piece * N >= p.dims) {
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
      const int h = slice + j * p.slices;
      if (h >= p.heads) break;
      Piece<U, N> u;
#pragma unroll
      for (int i = 0; i < N; ++i) u.v[i] = as_type<U>(a[j].v[i]);
      *reinterpret_cast<Piece<U, N> *>(out + h * p.o_hs) = u;
    }
  }
  __syncthreads();
  if (!placed || piece * N >= p.dims) return;
  float c[N], s[N];
  int other[N];  // where the value that each pairs up with is
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = piece * N + i;
    const bool low = at < half;
    const float2 t = at < p.dims ? mine[low ? at : at - half] : make_float2(1.0f, 0.0f);
    c[i] = t.x, s[i] = low ? -t.y : t.y;
    other[i] = at >= p.dims ? at : low ? at + half : at - half;
  }
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const int h = slice + j * p.slices;
    if (h >= p.heads) break;
    const T *row = reinterpret_cast<const T *>(&rows[j][r * p.pieces]);
    const P own = rows[j][tid];
    Piece<U, N> u;
#pragma unroll
    for (int i = 0; i < N; ++i)
      u.v[i] = piece * N + i < p.dims ? rounded<U>(to_float(own.v[i]) * c[i] + to_float(row[other[i]]) * s[i]) : as_type<U>(own.v[i]);
    *reinterpret_cast<Piece<U, N> *>(out + h * p.o_hs) = u;
  }
}

template <typename T, typename U, int N>
int launch_apart(const char *what, Params &p, cudaStream_t stream) {
  p.pieces = p.head_dim / N;
  p.slices = (p.heads + 3) / 4;
  p.block_rows = THREADS / p.pieces;
  const int64_t blocks = (p.tokens * p.slices + p.block_rows - 1) / p.block_rows;
  if (blocks > 0x7fffffff) return kv8::fail(EMMY_EINVAL, what, "too many tokens and heads");
  return kv8::launch_kernel(what, rotate_apart_kernel<T, U, N>, dim3(unsigned(blocks)), THREADS, 0, stream, p);
}

template <typename T, typename U, int N>
int launch_layout(const char *what, Params &p, cudaStream_t stream) {
  if constexpr (N > 1) {
    if (p.interleaved) return launch<T, U, N, true>(what, p, stream);
    if (p.dims / 2 % N != 0) return launch_apart<T, U, N>(what, p, stream);  // (at most 512 / N threads a row)
  }
  return launch<T, U, N, false>(what, p, stream);
}

// The widest pieces that start everywhere on a multiple of their size.  Results of
// another type are an append's queries, which start on multiples of 16 bytes.
template <typename T, typename U>
int launch_type(const char *what, Params &p, cudaStream_t stream) {
  const auto fits = [&](int n) {
    return reinterpret_cast<uintptr_t>(p.x) % (n * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(p.out) % (n * sizeof(U)) == 0 &&
           p.x_ts % n == 0 && p.x_hs % n == 0 && p.o_ts % n == 0 && p.o_hs % n == 0 && p.head_dim % n == 0;
  };
  constexpr int WIDEST = sizeof(T) == 2 && sizeof(U) == 2 ? 8 : 4;
  if (fits(WIDEST)) return launch_layout<T, U, WIDEST>(what, p, stream);
  if constexpr (std::is_same<T, U>::value) {
    if constexpr (WIDEST > 4)
      if (fits(4)) return launch_layout<T, U, 4>(what, p, stream);
    if (fits(2)) return launch_layout<T, U, 2>(what, p, stream);
    return launch_layout<T, U, 1>(what, p, stream);
  }
  return kv8::fail(EMMY_EINVAL, what, "q and q_out: base and strides must be multiples of 16 bytes");
}

template <typename T>
int launch_out(const char *what, Params &p, int out_type, cudaStream_t stream) {
  if (out_type == EMMY_KV8_F32) return launch_type<T, float>(what, p, stream);
  return out_type == EMMY_KV8_BF16 ? launch_type<T, __nv_bfloat16>(what, p, stream) : launch_type<T, __half>(what, p, stream);
}

}  // namespace

int rotate_rows(const char *what, Params &p, int type, int out_type, cudaStream_t stream) {
  if (type == EMMY_KV8_F32) return launch_out<float>(what, p, out_type, stream);
  return type == EMMY_KV8_BF16 ? launch_out<__nv_bfloat16>(what, p, out_type, stream) : launch_out<__half>(what, p, out_type, stream);
}

}  // namespace rotary

extern "C" int emmy_rotate(const emmy_rotary *r, const emmy_rotate_args *a, emmy_stream stream) {
  using namespace rotary;
  using kv8::fail;
  static const char *what = "emmy_rotate";
  if (const char *msg = kv8::rotary_trouble(r)) return fail(EMMY_EINVAL, what, msg);
  if (a == nullptr) return fail(EMMY_EINVAL, what, "null arguments");
  if (a->dtype != EMMY_KV8_F32 && a->dtype != EMMY_KV8_BF16 && a->dtype != EMMY_KV8_F16)
    return fail(EMMY_EINVAL, what, "dtype must be f32, bf16 or f16");
  if (a->device < 0) return fail(EMMY_EINVAL, what, "negative device");
  const int64_t T = a->tokens, H = a->heads, D = r->head_dim;
  if (T < 0 || T > 0x7fffffff) return fail(EMMY_EINVAL, what, "tokens must be between 0 and 2^31 - 1");
  if (H < 0 || H > 1 << 20) return fail(EMMY_EINVAL, what, "heads must be between 0 and 2^20");
  if (T == 0 || H == 0) return EMMY_OK;
  if (a->x == 0 || a->out == 0) return fail(EMMY_EINVAL, what, "null x or out");
  const int size = a->dtype == EMMY_KV8_F32 ? 4 : 2;
  if (a->x % size || a->out % size) return fail(EMMY_EINVAL, what, "x and out must be aligned to their type");
  if (a->positions % (a->wide ? 8 : 4)) return fail(EMMY_EINVAL, what, "positions must be aligned to their type");
  const bool in_place = a->x == a->out && (T == 1 || a->x_strides[0] == a->out_strides[0]) &&
                        (H == 1 || a->x_strides[1] == a->out_strides[1]);
  const int bad = kv8::rows_trouble(a->x, a->x_strides, H, size, a->out, a->out_strides, H, size, T, D, in_place);
  if (bad != kv8::ROWS_FINE)
    return fail(EMMY_EINVAL, what, bad == kv8::ROWS_NEGATIVE ? "x and out: strides must not be negative"
                                   : bad == kv8::ROWS_SELF   ? "rows of out overlap"
                                                             : "x and out overlap");
  Params p;
  for (int i = 0; i < EMMY_ROTARY_PAIRS; ++i) p.frequency[i] = r->turns[i];
  p.x = reinterpret_cast<const void *>(a->x);
  p.out = reinterpret_cast<void *>(a->out);
  p.positions = reinterpret_cast<const void *>(a->positions);
  p.first = a->first;
  p.position_stride = a->position_stride;
  p.tokens = T;
  p.x_ts = a->x_strides[0], p.x_hs = a->x_strides[1];
  p.o_ts = a->out_strides[0], p.o_hs = a->out_strides[1];
  p.heads = int(H), p.dims = r->dims, p.head_dim = r->head_dim;
  p.wide = a->wide != 0;
  p.interleaved = r->interleaved != 0;
  p.copy = !in_place;
  p.s.seqs = 0;
  p.gain = r->gain;
  p.sign = a->backward ? -1.0f : 1.0f;
  const kv8::OnDevice on(a->device);
  if (on.err != cudaSuccess) return kv8::cuda_fail(what, on.err);
  return rotate_rows(what, p, a->dtype, a->dtype, static_cast<cudaStream_t>(stream));
}
