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
// the piece that it is paired with, and does the same of HEADS heads: the angles
// cost about 40 instructions each and are computed once for all of them.
#include "kv8.cuh"
#include "rotary.cuh"

namespace rotary {
namespace {

constexpr int THREADS = 256, HEADS = 4;

struct Params {
  uint64_t frequency[EMMY_ROTARY_PAIRS];
  const void *x;
  void *out;
  const void *positions;  // null: first, first + 1, ..
  int64_t first, position_stride, tokens;
  int64_t x_ts, x_hs, o_ts, o_hs;  // token and head strides, elements
  int heads, dims, head_dim;
  int pieces, turned;     // pieces of a head that threads hold (with those paired with them), those turned
  int slices;             // of a token's heads: thread slice i has heads i, i + slices, ..
  int width, block_tokens;  // threads of a token, tokens of a block
  bool wide, interleaved, copy;
  float gain, sign;
};

template <typename T, int N, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) rotate_kernel(const __grid_constant__ Params p) {
  using P = Piece<T, N>;
  constexpr int PAIRS = INTERLEAVED ? N / 2 : N;  // that a thread holds
  kv8::grid_dependency_wait();
  kv8::grid_dependency_done();
  const int sub = threadIdx.x / p.width;
  const int64_t token = int64_t(blockIdx.x) * p.block_tokens + sub;
  if (sub >= p.block_tokens || token >= p.tokens) return;
  int64_t pos = p.first + token;
  if (p.positions != nullptr)
    pos = p.wide ? static_cast<const int64_t *>(p.positions)[token * p.position_stride]
                 : static_cast<const int *>(p.positions)[token * p.position_stride];
  for (int t = threadIdx.x - sub * p.width; t < p.width; t += p.block_tokens == 1 ? THREADS : p.width) {
    const int slice = t / p.pieces, piece = t - slice * p.pieces;
    const T *x = static_cast<const T *>(p.x) + token * p.x_ts;
    T *out = static_cast<T *>(p.out) + token * p.o_ts;
    if (piece >= p.turned) {
      // behind the turned ones
      const int at = p.dims + (piece - p.turned) * N;
      for (int h = slice; h < p.heads; h += p.slices)
        *reinterpret_cast<P *>(out + h * p.o_hs + at) = *reinterpret_cast<const P *>(x + h * p.x_hs + at);
      continue;
    }
    // single values of an interleaved row: pairs are neighbours all the same
    const bool near = N == 1 && p.interleaved;
    const int at = near ? 2 * piece : piece * N, other = near ? 1 : p.dims / 2;
    float c[PAIRS], s[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      turn_of(pos, p.frequency[piece * PAIRS + i], c[i], s[i]);
      c[i] *= p.gain;
      s[i] *= p.gain * p.sign;
    }
    for (int h0 = slice; h0 < p.heads; h0 += HEADS * p.slices) {
      P a[HEADS], b[INTERLEAVED ? 1 : HEADS];
#pragma unroll
      for (int j = 0; j < HEADS; ++j) {
        const int h = h0 + j * p.slices;
        if (h >= p.heads) continue;
        a[j] = *reinterpret_cast<const P *>(x + h * p.x_hs + at);
        if constexpr (!INTERLEAVED) b[j] = *reinterpret_cast<const P *>(x + h * p.x_hs + at + other);
      }
#pragma unroll
      for (int j = 0; j < HEADS; ++j) {
        const int h = h0 + j * p.slices;
        if (h >= p.heads) continue;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          T &u = INTERLEAVED ? a[j].v[2 * i] : a[j].v[i], &v = INTERLEAVED ? a[j].v[2 * i + 1] : b[INTERLEAVED ? 0 : j].v[i];
          const float fu = to_float(u), fv = to_float(v);
          u = rounded<T>(fu * c[i] - fv * s[i]);
          v = rounded<T>(fu * s[i] + fv * c[i]);
        }
        *reinterpret_cast<P *>(out + h * p.o_hs + at) = a[j];
        if constexpr (!INTERLEAVED) *reinterpret_cast<P *>(out + h * p.o_hs + at + other) = b[j];
      }
    }
  }
}

template <typename T, int N, bool INTERLEAVED>
int launch(Params p, cudaStream_t stream) {
  p.turned = INTERLEAVED ? p.dims / N : p.dims / 2 / N;
  p.pieces = p.turned + (p.copy ? (p.head_dim - p.dims) / N : 0);
  p.slices = (p.heads + HEADS - 1) / HEADS;
  const int64_t width = int64_t(p.slices) * p.pieces;
  p.width = int(width);
  p.block_tokens = width >= THREADS ? 1 : THREADS / int(width);
  const int64_t blocks = (p.tokens + p.block_tokens - 1) / p.block_tokens;
  return kv8::launch_kernel("emmy_rotate", rotate_kernel<T, N, INTERLEAVED>, dim3(unsigned(blocks)),
                            THREADS, 0, stream, p);
}

template <typename T, int N>
int launch_layout(const Params &p, cudaStream_t stream) {
  if constexpr (N > 1)
    if (p.interleaved) return launch<T, N, true>(p, stream);
  return launch<T, N, false>(p, stream);
}

// The widest pieces that start everywhere on a multiple of their size.
template <typename T>
int launch_type(const Params &p, cudaStream_t stream) {
  const auto fits = [&](int n) {
    const int64_t size = int64_t(n) * sizeof(T);
    const int64_t half = p.interleaved ? p.dims : p.dims / 2;
    return reinterpret_cast<uintptr_t>(p.x) % size == 0 && reinterpret_cast<uintptr_t>(p.out) % size == 0 &&
           p.x_ts % n == 0 && p.x_hs % n == 0 && p.o_ts % n == 0 && p.o_hs % n == 0 && half % n == 0 &&
           (!p.copy || (p.head_dim - p.dims) % n == 0);
  };
  if constexpr (sizeof(T) == 2)
    if (fits(8)) return launch_layout<T, 8>(p, stream);
  if (fits(4)) return launch_layout<T, 4>(p, stream);
  if (fits(2)) return launch_layout<T, 2>(p, stream);
  return launch_layout<T, 1>(p, stream);
}

}  // namespace
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
  p.gain = r->gain;
  p.sign = a->backward ? -1.0f : 1.0f;
  const kv8::OnDevice on(a->device);
  if (on.err != cudaSuccess) return kv8::cuda_fail(what, on.err);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dtype == EMMY_KV8_F32) return launch_type<float>(p, st);
  return a->dtype == EMMY_KV8_BF16 ? launch_type<__nv_bfloat16>(p, st) : launch_type<__half>(p, st);
}
