// The results of a call with shared keys as one: for each query row those of its
// run's shared keys and those of its sequence's own, in the parts' order,
//   m = max m_i,  l = sum l_i 2^(m_i - m),  O = sum O_i 2^(m_i - m) / l.
// A warp a row: a lane first has a part's maximum and sum, then D / 32 values of
// O.  Bound by the results, 4 (D + 2) bytes a part and row, from L2, eight loads in
// flight a lane, and by the three dependent loads before them: 4.3 us for 2048 rows
// of 8 + 1 or 2 results (9.5 MB), 4.0 for 128 rows.
#include "kv8_attend.cuh"

namespace kv8 {
namespace {

constexpr int WARPS = 8;

template <int D, typename T>
__global__ void __launch_bounds__(32 * WARPS) shared_join_kernel(const AttendParams p) {
  constexpr int N = D / 32;  // values of a lane
  const int lane = threadIdx.x & 31, heads = p.group * p.s.kv_heads;
  const int row = blockIdx.x * WARPS + (threadIdx.x >> 5), token = row / heads, h = row - token * heads;
  grid_dependency_wait();
  const PlanHead head = *p.plan;
  const int b = token < p.s.tokens ? p.seq_of[token] : -1;
  grid_dependency_done();
  if (!plan_fits(p, head, 0, 0, 0, 0)) return;
  if (head.joins != p.s.tokens) {
    report(p.s.status, STATUS_PLAN);
    return;
  }
  if (b < 0 || b >= p.s.seqs) return;
  const ResultRec f = p.results[b];
  const int n = f.n;
  const int kv_head = h / p.group, r = (token - f.start) * p.group + h - kv_head * p.group;
  float m = NONE, l = 0.0f, x[N] = {};
  // `parts` results, so many floats apart, of slots of so many rows
  const auto take = [&](const float *first, int64_t apart, int slot_rows, int slot_row, int parts) {
    const float *sums = first + slot_rows * D + slot_row, *values = first + slot_row * D + lane * N;
    for (; parts > 0; parts -= 32, sums += 32 * apart) {
      const int count = min(32, parts);
      const float *mine = sums + min(lane, count - 1) * apart;
      const float mi = __ldcg(mine), li = __ldcg(mine + slot_rows);
      float top = fmaxf(mi, m);
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float before = exp2_fast(m - top), w = lane < count ? exp2_fast(mi - top) : 0.0f;
      float sum = lane < count ? w * li : 0.0f;
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      l = l * before + sum;
      m = top;
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= before;
      for (int c0 = 0; c0 < count; c0 += 8) {
        float u[8][N];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const bool real = c0 + c < count;
          if constexpr (N == 4) {
            const float4 v = real ? __ldcg(reinterpret_cast<const float4 *>(values)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            u[c][0] = v.x, u[c][1] = v.y, u[c][2] = v.z, u[c][3] = v.w;
          } else {
            const float2 v = real ? __ldcg(reinterpret_cast<const float2 *>(values)) : make_float2(0.0f, 0.0f);
            u[c][0] = v.x, u[c][1] = v.y;
          }
          values += apart;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float by = __shfl_sync(0xffffffffu, w, (c0 + c) & 31);  // 0 where there is none
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] += by * u[c][j];
        }
      }
    }
  };
  // its results for shared keys, then for its own (one loop's code, not two)
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const bool of_run = i == 0;
    const int slot_rows = of_run ? p.pre_rows : 8 * p.nt, size = slot_rows * (D + 2);
    const int parts = of_run ? f.parts : f.own_parts, blocks = of_run ? f.blocks : f.own_blocks;
    const int at = of_run ? f.row + r : r, each = of_run ? slot_rows : (n * p.group + blocks - 1) / blocks;
    if (parts == 0) continue;
    const int block = at / each;
    take((of_run && p.shared == SHARED_TILES ? p.tile_partial : p.partial) +
             ((of_run ? f.slot0 : f.own_slot0) + int64_t(kv_head) * parts * blocks + block) * size,
         int64_t(blocks) * size, slot_rows, at - block * each, parts);
  }
  const float by = l == 0.0f ? 0.0f : 1.0f / l;
  T *to = static_cast<T *>(p.out) + token * p.o_ts + h * p.o_hs + lane * N;
  if constexpr (N == 4)
    *reinterpret_cast<uint2 *>(to) = make_uint2(pack2<T>(x[0] * by, x[1] * by), pack2<T>(x[2] * by, x[3] * by));
  else
    *reinterpret_cast<uint32_t *>(to) = pack2<T>(x[0] * by, x[1] * by);
}

template <int D, typename T>
int launch(const AttendParams &p, cudaStream_t stream) {
  const int64_t rows = int64_t(p.s.tokens) * p.group * p.s.kv_heads;  // at most 2^31 - 1
  return launch_kernel("emmy_kv8_attend_shared", shared_join_kernel<D, T>, dim3(unsigned((rows + WARPS - 1) / WARPS)),
                       32 * WARPS, 0, stream, p);
}

}  // namespace

int shared_join(const AttendParams &p, const emmy_kv8 &cache, bool bf16, cudaStream_t stream) {
  if (cache.head_dim == 64) return bf16 ? launch<64, __nv_bfloat16>(p, stream) : launch<64, __half>(p, stream);
  return bf16 ? launch<128, __nv_bfloat16>(p, stream) : launch<128, __half>(p, stream);
}

}  // namespace kv8
