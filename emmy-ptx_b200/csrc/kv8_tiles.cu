// Attention of many query rows over the paged 8-bit cache (prompts, chunks of
// prompts behind a history), on tcgen05.
//
// A unit is 256 query rows of one (sequence, kv head) -- tokens x the query
// heads that share the kv head, so these share one pass over its keys -- as
// two tiles A and B of 128 rows, which walk the 64-key chunks that some row
// sees.  One CTA an SM takes unit after unit, and every role runs on into the
// next one as soon as its own work allows: codes and query rows of the next
// unit are on their way, and its first scores are computed, while the softmax
// warps still write this one's rows (a CTA a unit: 228 us a prompt of 8191
// tokens with a window of 512 and d = 64, ten chunks a unit; so: 193).
// Warps:
//   0       tcgen05 O += P V of both tiles (one thread); owns the TMEM
//   1       bulk copies of codes into shared memory, chunks ahead (in a loading
//           warp, which they held up: 266 us a batch of prompts instead of 257)
//   2, 3    tcgen05 S = Q K^T of tile A, B: an issuing warp slows the softmax
//           warps of its sub-partition, and the slowest of a tile sets its pace
//   4-7     softmax and output of tile A, a thread a row; 8-11 of tile B
//   12-15   codes -> f16, stored as the 128-byte-swizzled tiles the MMAs
//           read (K as [keys][d], V as stored: an MN-major operand)
// 128 registers a thread at launch; the softmax warps take 168 (a row's 64
// scores and its packed weights are live together) from the others.
// TMEM: per tile two 64-column S buffers (chunk n of the tile in buffer n % 2,
// P over its first half as packed f16), O and, with d = 64, the query rows.
// With two buffers S of chunk n + 1 is computed while the softmax works on
// chunk n.
//
// The numerics are those of kv8_rows.cu: e4m3 exact in f16, a query row scaled
// by a power of two, scores and sums in f32, p rounded to f16, K's page
// exponent in the factor that takes scores to log2 units and V's in the
// exponent of p; O moves (a pass over its columns) only when a row's maximum
// grew by more than 2^8 or V's exponent strayed by more than 2^6.
#include <algorithm>

#include "kv8_async.cuh"
#include "kv8_attend.cuh"

namespace kv8 {
namespace {

constexpr int TILE = 128, CHUNK = 64, THREADS = 512;
constexpr int STAGES = 3, RAW = 3;  // f16 chunks, and chunks of codes, in shared memory
constexpr int W_PV = 0, W_FETCH = 1, W_QK = 2, W_SOFTMAX = 4, W_LOAD = 12;  // warps
// Registers of the four warpgroups after the split.  The sum is what the
// block was launched with: a split above it would wait for ever.
constexpr int REGS_LAUNCH = 128, REGS_ISSUE = 80, REGS_SOFTMAX = 168, REGS_LOAD = 96;
static_assert(REGS_ISSUE + 2 * REGS_SOFTMAX + REGS_LOAD == 4 * REGS_LAUNCH, "register split");
constexpr float LAZY = 8.0f, LEAST = 1e-37f;
// Weights are 2^(s rm - m) with one rounding of the difference, m = round(max s
// rm): the two differ by up to 2^-24 |m|, a factor common to the row, which
// stays in f16's range up to this |m|.  Beyond it f32 scores are whole multiples
// of 16 and more, and s rm is rounded first, as m was, so that the largest
// weight is 1: the chunk's scores are replaced by the products in TMEM.
constexpr float HUGE_SCORE = 134217728.0f;
constexpr int UNIT_LAZY = 6;
constexpr int Q_COL = 4 * CHUNK + 2 * 64;  // TMEM column of the query rows, d = 64 only

template <int D>
struct Layout {
  // With d = 64 TMEM has room for the query rows, too: products that read them
  // there leave shared memory's bandwidth to the keys (193 -> 189 us a prompt of
  // 8191 tokens with a window of 512).
  static constexpr bool Q_TMEM = D == 64;
  // Rows that lanes hold each one of, read or written 64 bytes at a time by four
  // lanes.  d = 128: read so 242 us a batch of prompts (250 each lane its own),
  // written so, too, 243 and 0.6 us more for a short prompt; d = 64, 8191 tokens
  // with a window: written so 186 us (190), read so 197.
  static constexpr bool READ4 = D == 128, WRITE4 = D == 64;
  static constexpr int Q_TILE = Q_TMEM ? 0 : TILE * D * 2, KV = CHUNK * D * 2;  // bytes
  static constexpr int STAGE0 = 2 * Q_TILE;
  static constexpr int RAW0 = STAGE0 + STAGES * 2 * KV;    // K codes, then V codes
  static constexpr int NAN_ROWS = RAW0 + RAW * KV;         // D bits a row
  static constexpr int END = NAN_ROWS + 2 * TILE * (D / 8);
  // 1 KB to align the tiles; above half an SM's shared memory, so that two
  // CTAs of one SM never wait for each other's TMEM
  static constexpr int DYN = END + 1024 > 120 * 1024 ? END + 1024 : 120 * 1024;
  static constexpr int O_COL = 4 * CHUNK;
};

struct Bars {
  uint64_t q_full[2], kv_full[STAGES], kv_empty[STAGES], raw_full[RAW], raw_empty[RAW];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], drain;
};

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The issuing warps stay converged, so that descriptors live in uniform
// registers; `who` is 1 in the one lane that issues.
__device__ __forceinline__ void tc_commit(uint64_t *b, uint32_t who) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.u32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(b)),
      "r"(who)
      : "memory");
}
// D (+)= A B with A and B in shared memory, or A (TS) in TMEM.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                                       uint32_t who) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(who)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                                       uint32_t who) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(who)
      : "memory");
}
__device__ __forceinline__ void tm_ld32(uint32_t (&r)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tm_st32(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// Half a chunk's time: tile B starts so much later, so that its exponentials
// fall between tile A's on the MUFU that they share (196 -> 190 us a prompt of
// 8191 tokens with a window of 512 and d = 64, 560 -> 557 without one).
__device__ __forceinline__ void stagger() {
  const long long t0 = clock64();
  while (clock64() - t0 < 900) {
  }
}
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// Four lanes' 16-byte pieces, transposed: piece i of lane j <-> piece j of lane i.
// Threads that hold a row each then read and write 64 bytes of a row together.
__device__ __forceinline__ void transpose4(uint4 (&w)[4], int lane) {
#pragma unroll
  for (int bit = 1; bit <= 2; bit <<= 1) {
    const bool up = (lane & bit) != 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int a = bit == 1 ? 2 * i : i, b = a + bit;
      uint32_t *x = &w[a].x, *y = &w[b].x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? x[j] : y[j], bit);
        (up ? x[j] : y[j]) = got;
      }
    }
  }
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two f32 in one register pair.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void tm_ld8(uint32_t (&r)[8], uint32_t at) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(at));
}
__device__ __forceinline__ void tm_st8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle: start address, leading
// and stride byte offsets in 16-byte units, version 1 (bit 46), layout 2.
__device__ __forceinline__ uint64_t smem_desc(uint32_t at, uint32_t lbo, uint32_t sbo) {
  return uint64_t((at >> 4) & 0x3fff) | uint64_t(lbo >> 4) << 16 | uint64_t(sbo >> 4) << 32 | 1ull << 46 |
         2ull << 61;
}
// kind::f16, f16 operands, f32 sums; bit 16: B is MN-major.
template <int M, int N, bool B_MN>
constexpr uint32_t IDESC = 1u << 4 | uint32_t(B_MN) << 16 | uint32_t(N >> 3) << 17 | uint32_t(M >> 4) << 24;

// 16-byte piece j (0-7) of 128-byte row r of a swizzled tile.
__device__ __forceinline__ uint32_t swizzled(int r, int j) { return r * 128 + ((j ^ (r & 7)) << 4); }

// The record's rows and keys are within the arrays.
__device__ __forceinline__ bool plan_holds(const AttendParams &p, int start, int n, int len) {
  const bool ok = start + n <= p.s.tokens && len <= (int64_t(p.s.width) << p.s.page_shift);
  if (!ok) report(p.s.status, STATUS_PLAN);
  return ok;
}

// What the unit is: 256 rows of one (sequence, kv head).
struct Unit {
  int b, head, start, n, len, rows, row0;
  Span span;
  int c0, slot;  // first chunk of this part's; workspace slot, -1: the unit is whole
  int tiles, chunks;

  Unit() = default;
  __device__ __forceinline__ Unit(const AttendParams &p, const UnitRec &r)
      : b(r.b), head(r.head), start(r.start), n(r.n), len(r.len), rows(r.n * p.group), row0(r.row0),
        span(p, r.len - r.n + r.row0 / p.group,
             r.len - r.n + (min(r.row0 + 2 * TILE, r.n * p.group) - 1) / p.group),
        c0(r.c0), slot(r.slot), tiles(rows - r.row0 > TILE ? 2 : 1), chunks(r.c1 - r.c0) {}
};

// What goes with a chunk of codes.
struct ChunkInfo {
  int ek, ev, key0, dead;
};

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}

template <int D, typename T>
__global__ void __launch_bounds__(THREADS, 1) tiles_kernel(const AttendParams p) {
  using L = Layout<D>;
  extern __shared__ uint8_t dyn_raw[];
  uint8_t *const dyn = dyn_raw + ((1024 - (smem_addr(dyn_raw) & 1023)) & 1023);
  __shared__ Bars bars;
  __shared__ uint32_t tmem_slot;
  // Scales (2^ek, ev) of the CTA's chunk c and whether it holds NaN values, in
  // slots c % 4 and c % 8: by the time chunk c + 4 is written there, P V of chunk c + 1 is
  // done and with it every softmax warp past chunk c.
  __shared__ float2 chunk_scale[4];
  __shared__ unsigned stop_word, chunk_nan[8];
  __shared__ ChunkInfo raw_info[RAW];
  volatile unsigned *const stop = &stop_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Seqs &s = p.s;

  grid_dependency_wait();
  if (p.beside && blockIdx.x == 0 && tid == 0)
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p.ready), "r"(1u) : "memory");
  const PlanHead head = *p.plan;
  const UnitRec first_rec = p.units[blockIdx.x];
  grid_dependency_done();
  if (blockIdx.x >= head.units || !plan_fits(p, head, first_rec.b, first_rec.start, first_rec.n, first_rec.len)) return;
  // The units of this CTA: one of each gridDim.x, in turn from the front and
  // from the back, since the longest come first.
  const int units = head.units;
  const auto index_of = [&](int k) {
    return k * int(gridDim.x) + (k & 1 ? int(gridDim.x) - 1 - int(blockIdx.x) : int(blockIdx.x));
  };
  const auto load_unit = [&](int k, Unit &u) {  // false: there is no such unit
    const int i = index_of(k);
    if (i >= units) return false;
    const UnitRec r = p.units[i];
    if (!plan_holds(p, r.start, r.n, r.len)) return false;
    u = Unit(p, r);
    return true;
  };

  // ---- barriers, TMEM ----
  if (tid == 0) {
    bar_init(&bars.q_full[0], 4);  // warps
    bar_init(&bars.q_full[1], 4);
    for (int i = 0; i < STAGES; ++i) {
      bar_init(&bars.kv_full[i], 4);
      bar_init(&bars.kv_empty[i], 2);  // P V of both tiles, and tile B's S, which may have none
    }
    for (int i = 0; i < 8; ++i) chunk_nan[i] = 0;
    for (int i = 0; i < RAW; ++i) {
      bar_init(&bars.raw_full[i], 1);
      bar_init(&bars.raw_empty[i], 4);
    }
    for (int x = 0; x < 2; ++x)
      for (int i = 0; i < 2; ++i) {
        bar_init(&bars.s_full[x][i], 2);
        bar_init(&bars.p_full[x][i], 4);
        bar_init(&bars.pv_done[x][i], 1);
      }
    bar_init(&bars.drain, 3);
    stop_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == W_PV) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;

  bool issuer = false;  // the lane that issued this warp's MMAs
  if (warp < W_SOFTMAX) regs_down<REGS_ISSUE>();
  if (warp == W_PV) {
    // ---- O += P V of both tiles ----
    const uint32_t who = elected();
    bool ok = true;
    Ring kv;
    int n[2] = {0, 0};  // chunks of each tile so far
    Unit u;
    for (int k = 0; ok && load_unit(k, u); ++k)
      for (int g = 0; ok && g < u.chunks; ++g, kv.next(STAGES)) {
        ok = warp_wait(&bars.kv_full[kv.slot], kv.phase, stop, s.status, p.wait_ns);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!ok || x >= u.tiles) break;
          const int buf = n[x] & 1;
          ok = warp_wait(&bars.p_full[x][buf], n[x] >> 1 & 1, stop, s.status, p.wait_ns);
          if (!ok) break;
          ++n[x];
          tc_after();
          // V rows are 128 bytes (64 values of d), the second half of d follows
          // CHUNK rows on; 16 keys are 2 KB
          const uint64_t vd = smem_desc(smem_addr(dyn + L::STAGE0 + kv.slot * 2 * L::KV + L::KV), CHUNK * 128, 1024);
          const uint32_t o = tmem + L::O_COL + x * D, pa = tmem + (2 * x + buf) * CHUNK;
#pragma unroll
          for (int i = 0; i < CHUNK / 16; ++i)
            mma_ts(o, pa + i * 8, vd + (i * 2048 >> 4), IDESC<TILE, D, true>, g > 0 || i > 0, who);
          tc_commit(&bars.pv_done[x][buf], who);
        }
        if (ok) tc_commit(&bars.kv_empty[kv.slot], who);
      }
    if (who) issuer = true;
  } else if (warp == W_FETCH) {
    // ---- bulk copies: K and V of a page's chunk are one contiguous piece
    // each; 32 chunks' pages and exponents are read at once, a lane a chunk ----
    const uint32_t who = elected();
    bool ok = p.stall == 0 || blockIdx.x % p.stall != 0;
    int so_far = 0;
    Ring copied;
    Unit u;
    for (int k = 0; ok && load_unit(k, u); ++k) {
      const int *row = s.table + int64_t(u.b) * s.width;
      ChunkInfo next = {0, 0, 0, 0};
      int64_t next_unit = 0;
      const auto fetch = [&](int g) {  // chunk g into the next slot, which is free
        if ((g & 31) == 0) {
          next = ChunkInfo{0, 0, 0, 0};
          next_unit = 0;
          if (g + lane < u.chunks) {
            next.key0 = u.span.key0(u.c0 + g + lane);
            int page = row[next.key0 >> s.page_shift];
            next.dead = page < 0 || page >= s.pages;
            if (next.dead) {
              report(s.status, STATUS_PAGE);
              page = 0;
            }
            next_unit = int64_t(page) * 2 * s.kv_heads + u.head;
            next.ek = p.exps[next_unit];
            next.ev = p.exps[next_unit + s.kv_heads];
          }
        }
        const int64_t at = __shfl_sync(0xffffffffu, next_unit, g & 31);
        ChunkInfo c;
        c.ek = held_exponent(__shfl_sync(0xffffffffu, next.ek, g & 31));
        c.ev = held_exponent(__shfl_sync(0xffffffffu, next.ev, g & 31));
        c.key0 = __shfl_sync(0xffffffffu, next.key0, g & 31);
        c.dead = __shfl_sync(0xffffffffu, next.dead, g & 31);
        if (who) {
          raw_info[copied.slot] = c;
          const uint8_t *k = p.codes + ((at << s.page_shift) + (c.key0 & ((1 << s.page_shift) - 1))) * D;
          const uint8_t *v = k + (int64_t(s.kv_heads) << s.page_shift) * D;
          const uint32_t dst = smem_addr(dyn + L::RAW0 + copied.slot * L::KV);
          uint64_t *bar = &bars.raw_full[copied.slot];
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(L::KV)
                       : "memory");
          bulk_copy(dst, k, CHUNK * D, bar);
          bulk_copy(dst + CHUNK * D, v, CHUNK * D, bar);
        }
        __syncwarp();
        copied.next(RAW);
      };
      // its query rows on their way into L2
      for (int i = lane; i < min(2 * TILE, u.rows - u.row0); i += 32) {
        const int token = (u.row0 + i) / p.group, h = u.head * p.group + u.row0 + i - token * p.group;
        const T *q = static_cast<const T *>(p.q) + (int64_t(u.start) + token) * p.q_ts + h * p.q_hs;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
        if (D == 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + D / 2));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(q + D - 8));
      }
      for (int g = 0; g < u.chunks; ++g, ++so_far) {
        if (so_far >= RAW) ok = warp_wait(&bars.raw_empty[copied.slot], copied.phase ^ 1, stop, s.status, p.wait_ns);
        if (!ok) break;
        fetch(g);
      }
    }
  } else if (warp < W_SOFTMAX) {
    // ---- S = Q K^T of one tile ----
    const uint32_t who = elected();
    const int x = warp - W_QK;
    const uint64_t qd = smem_desc(smem_addr(dyn + x * L::Q_TILE), 16, 1024);
    bool ok = true;
    Ring kv;
    int n = 0, mine = 0;  // chunks and units of this tile so far
    Unit u;
    for (int k = 0; ok && load_unit(k, u); ++k) {
      if (x < u.tiles) ok = warp_wait(&bars.q_full[x], mine++ & 1, stop, s.status, p.wait_ns);
      for (int g = 0; ok && g < u.chunks; ++g, kv.next(STAGES)) {
        ok = warp_wait(&bars.kv_full[kv.slot], kv.phase, stop, s.status, p.wait_ns);
        if (x == 1 && who) bar_arrive(&bars.kv_empty[kv.slot]);
        if (x >= u.tiles) continue;
        const int buf = n & 1;
        // the buffer holds P of chunk n - 2 until its P V is done
        if (ok && n >= 2) ok = warp_wait(&bars.pv_done[x][buf], (n >> 1 & 1) ^ 1, stop, s.status, p.wait_ns);
        if (!ok) break;
        ++n;
        tc_after();
        const uint64_t kd = smem_desc(smem_addr(dyn + L::STAGE0 + kv.slot * 2 * L::KV), 16, 1024);
        const uint32_t at = tmem + (2 * x + buf) * CHUNK;
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if constexpr (L::Q_TMEM)
              mma_ts(at, tmem + Q_COL + x * (D / 2) + i * 8, kd + (i * 32 >> 4), IDESC<TILE, CHUNK, false>, i > 0, who);
            else
              mma_ss(at, qd + ((h * TILE * 128 + i * 32) >> 4), kd + ((h * CHUNK * 128 + i * 32) >> 4),
                     IDESC<TILE, CHUNK, false>, h > 0 || i > 0, who);
        tc_commit(&bars.s_full[x][buf], who);
        // and one ordinary arrival, which passes on what the loading warps
        // left beside the codes
        if (who) bar_arrive(&bars.s_full[x][buf]);
      }
    }
    if (who) issuer = true;
  } else if (warp >= W_LOAD) {
    regs_down<REGS_LOAD>();
    // ---- codes -> f16 ----
    // A lane's 16-byte pieces of codes become two neighbouring 16-byte pieces
    // of f16.  D = 128: eight lanes that load or store together cover the two
    // halves of d in two neighbouring rows, so that neither the loads (rows of
    // 128 bytes) nor the stores (pieces exchanged by row & 7) meet in a bank.
    constexpr int PASS_ROWS = D == 128 ? 16 : 32, PASSES = CHUNK / PASS_ROWS;
    const int w = warp - W_LOAD, piece = lane & 3, b2 = lane >> 2 & 1;
    const int r0 = D == 128 ? w * 4 + b2 + 2 * (lane >> 4) : w * 8 + (lane >> 2);
    const int half = D == 128 ? b2 ^ (lane >> 3 & 1) : 0;
    const uint32_t from = r0 * D + (half * 4 + piece) * 16;
    const uint32_t to = half * (CHUNK * 128) + swizzled(r0, 2 * piece);
    const auto put = [&](uint8_t *tile, int pass, const uint4 &x) {
      uint8_t *at = tile + pass * (PASS_ROWS * 128);
      *reinterpret_cast<uint4 *>(at + to) =
          make_uint4(e4m3x2_f16x2(x.x), e4m3x2_f16x2(x.x >> 16), e4m3x2_f16x2(x.y), e4m3x2_f16x2(x.y >> 16));
      *reinterpret_cast<uint4 *>(at + (to ^ 16)) =
          make_uint4(e4m3x2_f16x2(x.z), e4m3x2_f16x2(x.z >> 16), e4m3x2_f16x2(x.w), e4m3x2_f16x2(x.w >> 16));
    };
    Ring raw, kv;
    int c = 0;  // chunks so far
    bool ok = true;
    Unit u;
    for (int k = 0; ok && load_unit(k, u); ++k)
      for (int g = 0; g < u.chunks; ++g, ++c, raw.next(RAW), kv.next(STAGES)) {
        ok = warp_wait(&bars.raw_full[raw.slot], raw.phase, stop, s.status, p.wait_ns);
        if (!ok) break;
        const uint8_t *src = dyn + L::RAW0 + raw.slot * L::KV + from;
        uint4 k[PASSES], v[PASSES];
#pragma unroll
        for (int i = 0; i < PASSES; ++i) k[i] = *reinterpret_cast<const uint4 *>(src + i * PASS_ROWS * D);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) v[i] = *reinterpret_cast<const uint4 *>(src + CHUNK * D + i * PASS_ROWS * D);
        const ChunkInfo info = raw_info[raw.slot];
        warp_arrive(&bars.raw_empty[raw.slot]);
        const int st = kv.slot;
        if (c >= STAGES) ok = warp_wait(&bars.kv_empty[st], kv.phase ^ 1, stop, s.status, p.wait_ns);
        if (!ok) break;
        // chunks some row does not see whole: values no row sees are zeroed and
        // a NaN is taken out here (0 * NaN would reach rows it is hidden from)
        // and put into the rows that see it at the end
        if (info.dead || !u.span.all_see(info.key0, info.key0 + CHUNK - 1)) {
#pragma unroll
          for (int i = 0; i < PASSES; ++i) {
            if (info.dead || !u.span.any_sees(info.key0 + r0 + i * PASS_ROWS)) v[i] = make_uint4(0, 0, 0, 0);
            uint32_t *x = &v[i].x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t bad = nan_bytes(x[j]);
              if (bad != 0) {
                x[j] &= ~((bad >> 7) * 0xffu);
                chunk_nan[c & 7] = 1;
              }
            }
          }
        }
        uint8_t *tile = dyn + L::STAGE0 + st * 2 * L::KV;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) put(tile, i, k[i]);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) put(tile + L::KV, i, v[i]);
        if (tid == W_LOAD * 32) {
          chunk_scale[c & 3] = make_float2(info.dead ? 0.0f : pow2(info.ek), float(info.ev));
          chunk_nan[(c + 4) & 7] = 0;  // no loading warp is three chunks ahead
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        warp_arrive(&bars.kv_full[st]);
      }
  } else if (warp >= W_SOFTMAX) {
    // ---- softmax: a thread a row ----
    regs_up<REGS_SOFTMAX>();
    const int x = (warp - W_SOFTMAX) >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lanes = uint32_t(quad * 32) << 16;
    const uint32_t s_at = tmem + lanes + 2 * x * CHUNK, o_at = tmem + lanes + L::O_COL + x * D;
    // the unit from the k-th on that has this tile
    const auto next_unit = [&](int &k, int &before, Unit &u) {
      for (; load_unit(k, u); ++k, before += u.chunks)
        if (x < u.tiles) return true;
      return false;
    };
    struct Row {
      int token, head, pos;
      bool real;
    };
    const auto row_of = [&](const Unit &u) {
      const int row = u.row0 + x * TILE + r, at = min(row, u.rows - 1);
      Row w;
      w.token = at / p.group;
      w.head = u.head * p.group + at - w.token * p.group;
      w.pos = u.len - u.n + w.token;
      w.real = row < u.rows;
      return w;
    };
    // The unit's query rows, f16, scaled by a power of two, the scale's sign in
    // them; returns the factor of the row's scores.  The products that read the
    // rows before are done: their scores were here.
    const auto put_query = [&](const Unit &u, const Row &row) {
      const int64_t mine = (int64_t(u.start) + row.token) * p.q_ts + row.head * p.q_hs;
      const T *const q = static_cast<const T *>(p.q);
      uint4 w[D / 8];
      if constexpr (L::READ4) {
        const T *src[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) src[i] = q + __shfl_sync(0xffffffffu, mine, (lane & ~3) | i) + 8 * (lane & 3);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) w[i] = *reinterpret_cast<const uint4 *>(src[i % 4] + i / 4 * 32);
#pragma unroll
        for (int i = 0; i < D / 8; i += 4) transpose4(*reinterpret_cast<uint4(*)[4]>(&w[i]), lane);
      } else {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) w[i] = *reinterpret_cast<const uint4 *>(q + mine + 8 * i);
      }
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t *v = &w[i].x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a, b;
          unpack2<T>(v[j], a, b);
          a = fabsf(a), b = fabsf(b);
          amax = a < INFINITY ? fmaxf(amax, a) : amax;
          amax = b < INFINITY ? fmaxf(amax, b) : amax;
        }
      }
      const int e = row_exponent(amax);
      const float by = p.scale_log2 < 0.0f ? -pow2(-e) : pow2(-e);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        uint32_t *v = &w[i].x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a, b;
          unpack2<T>(v[j], a, b);
          v[j] = pack2<__half>(a * by, b * by);
        }
        if constexpr (!L::Q_TMEM)
          *reinterpret_cast<uint4 *>(dyn + x * L::Q_TILE + i / 8 * (TILE * 128) + swizzled(r, i % 8)) = w[i];
      }
      if constexpr (L::Q_TMEM) {
        uint32_t all[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) all[i] = (&w[i / 4].x)[i % 4];
        tm_st32(tmem + lanes + Q_COL + x * (D / 2), all);
        tm_wait_st();
        tc_before();
      } else {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      warp_arrive(&bars.q_full[x]);
      return fabsf(p.scale_log2) * pow2(e);
    };
    bool ok = true;
    int k = 0, n = 0, before = 0;  // chunks of this tile, and of all units before this
    Unit u;
    float mult = 0.0f;
    Row at;
    bool more = next_unit(k, before, u);
    if (more) {
      at = row_of(u);
      mult = put_query(u, at);
    }
    while (more) {
      // of the unit only what the loop needs stays in registers
      const int pos = at.pos, chunks = u.chunks, c0 = u.c0, sink_chunks = u.span.sink_chunks, window_chunk0 = u.span.window_chunk0;
      const bool real = at.real;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        *reinterpret_cast<uint32_t *>(dyn + L::NAN_ROWS + (x * TILE + r) * (D / 8) + 4 * i) = 0;
      float m = NONE, l = 0.0f;
      int unit = 0;
      bool nan_seen = false, big = false, rounded = false;
      // chunks whole_lo .. whole_hi - 1 every row sees whole
      int whole_lo = 0, whole_hi = chunks;
      {
        const Span &sp = u.span;
        if (p.window > 0) {
          // from the first window chunk that starts inside the last token's window
          const int low = max(0, sp.last - p.window + 1);
          whole_lo = sp.sink_chunks + max(0, ((low + CHUNK - 1) >> 6) - sp.window_chunk0);
        }
        whole_hi = sp.sink_chunks + ((sp.first + 1) >> 6) - sp.window_chunk0 - u.c0;
        whole_lo -= u.c0;
      }
      for (int g = 0; g < chunks; ++g, ++n) {
        const int buf = n & 1;
        ok = warp_wait(&bars.s_full[x][buf], n >> 1 & 1, stop, s.status, p.wait_ns);
        if (!ok) break;
        if (g == 0 && x == 1) stagger();
        const int c = before + g;  // chunks of the CTA so far
        const float2 sc = chunk_scale[c & 3];
        const int ev = int(sc.y);
        const float rm = rounded ? 1.0f : fmaxf(mult * sc.x, LEAST);
        tc_after();
        uint32_t sv[2][32];
        tm_ld32(sv[0], s_at + buf * CHUNK);
        tm_ld32(sv[1], s_at + buf * CHUNK + 32);
        tm_wait_ld();
        const bool dead = sc.x == 0.0f;
        if (dead || g < whole_lo || g >= whole_hi) {
          const int i0 = c0 + g, key0 = (i0 < sink_chunks ? i0 : i0 - sink_chunks + window_chunk0) << 6;
          // bit i: the row sees key key0 + i
          const auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
          uint64_t see = below(pos - key0 + 1);
          if (p.window > 0) see &= ~below(pos - p.window + 1 - key0) | below(p.sinks - key0);
          if (dead) see = 0;
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (!(see >> i & 1)) sv[i / 32][i % 32] = 0xff800000u;
          if (chunk_nan[c & 7] != 0 && real) {
            // (rare) this chunk holds NaN values: which of them this row sees
            const UnitRec rec = p.units[index_of(k)];
            const int page = s.table[int64_t(rec.b) * s.width + (key0 >> s.page_shift)];
            const int64_t at = (int64_t(page) * 2 + 1) * s.kv_heads + rec.head;
            const uint32_t *v = reinterpret_cast<const uint32_t *>(
                p.codes + ((at << s.page_shift) + (key0 & ((1 << s.page_shift) - 1))) * D);
            uint32_t *bits = reinterpret_cast<uint32_t *>(dyn + L::NAN_ROWS + (x * TILE + r) * (D / 8));
            for (int i = 0; i < CHUNK; ++i)
              if (see >> i & 1)
                for (int w = 0; w < D / 4; ++w) {
                  const uint32_t bad = nan_bytes(v[i * (D / 4) + w]);
                  if (bad != 0)
                    bits[w / 8] |= ((bad >> 7 & 1) | (bad >> 14 & 2) | (bad >> 21 & 4) | (bad >> 28 & 8)) << (w % 8 * 4);
                }
            nan_seen = true;
          }
        }
        const auto score = [&](int i) { return __uint_as_float(sv[i / 32][i % 32]); };
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = score(i);
#pragma unroll
        for (int i = 4; i < 64; i += 2) top[i / 2 & 3] = max3(top[i / 2 & 3], score(i), score(i + 1));
        const float raw = fmaxf(max3(top[0], top[1], top[2]), top[3]), best = raw * rm;
        const int stray = ev - unit;
        const bool first = g == 0, move = stray > UNIT_LAZY || stray < -UNIT_LAZY || big;
        const bool fix = __any_sync(0xffffffffu, best > m + LAZY || move);
        float alpha = 1.0f;
        if (fix) {
          const float to = fmaxf(m, best);
          if (!rounded && __any_sync(0xffffffffu, fabsf(to) > HUGE_SCORE && to != NONE)) {
            // (rare) this chunk again, from products rounded first.  A loop, and the
            // scores' registers left alone: the same unrolled over them cost every
            // call (a prompt of 8191 tokens with a window of 512: 198 for 186 us).
#pragma unroll 1
            for (int c = 0; c < CHUNK; c += 8) {
              uint32_t w[8];
              tm_ld8(w, s_at + buf * CHUNK + c);
              tm_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * rm);
              tm_st8(s_at + buf * CHUNK + c, w);
            }
            tm_wait_st();
            rounded = true;
            --g, --n;
            continue;
          }
          alpha = exp2_fast(m - to);
          m = to;
          l *= alpha;
          big |= is_big(m);
          if (first) unit = ev;
          if (move || big) {
            alpha *= pow2(unit - ev);
            unit = ev;
          }
        }
        const float shift = float(ev - unit) - m;
        const uint64_t rm2 = pair(rm, rm), shift2 = pair(shift, shift);
        uint64_t sum[4] = {};
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float a, b;
          unpair(fma2(pair(score(2 * i), score(2 * i + 1)), rm2, shift2), a, b);
          a = exp2_fast(a);
          b = exp2_fast(b);
          sum[i & 3] = add2(sum[i & 3], pair(a, b));
          pk[i] = pack2<__half>(a, b);
        }
        rounded = false;
        tm_st32(s_at + buf * CHUNK, pk);
        float even, odd;
        unpair(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), even, odd);
        l = fmaf(even + odd, pow2(unit - ev), l);
        tm_wait_st();
        if (fix && !first) {
          // P V of chunk n - 1 is the last to have touched O
          ok = warp_wait(&bars.pv_done[x][(n - 1) & 1], (n - 1) >> 1 & 1, stop, s.status, p.wait_ns);
          if (!ok) break;
          tc_after();
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tm_ld32(o, o_at + c);
            tm_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tm_st32(o_at + c, o);
          }
          tm_wait_st();
        }
        tc_before();
        warp_arrive(&bars.p_full[x][buf]);
      }
      if (!ok) break;
      // the next unit's queries first: its products start under this one's end
      const int i = index_of(k);
      u = Unit(p, p.units[i]);
      at = row_of(u);
      const int slot = u.slot;
      const int64_t to = (int64_t(u.start) + at.token) * p.o_ts + at.head * p.o_hs;
      before += chunks;
      more = next_unit(++k, before, u);
      if (more) {
        at = row_of(u);
        mult = put_query(u, at);
      }
      ok = warp_wait(&bars.pv_done[x][(n - 1) & 1], (n - 1) >> 1 & 1, stop, s.status, p.wait_ns);
      if (!ok) break;
      {
        tc_after();
        const uint32_t reals = __ballot_sync(0xffffffffu, real);
        T *out[4];  // this lane's pieces: of four lanes' rows, or of its own
#pragma unroll
        for (int i = 0; i < 4; ++i)
          out[i] = static_cast<T *>(p.out) +
                   (L::WRITE4 ? __shfl_sync(0xffffffffu, to, (lane & ~3) | i) + 8 * (lane & 3) : to + 8 * i);
        const float by = slot >= 0 ? pow2(unit) : l == 0.0f ? 0.0f : pow2(unit) / l;
        float *const part = p.tile_partial + int64_t(slot) * (D + 2) * (2 * TILE) + x * TILE + r;
        const uint32_t *bits = reinterpret_cast<const uint32_t *>(dyn + L::NAN_ROWS + (x * TILE + r) * (D / 8));
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tm_ld32(o, o_at + c);
          tm_wait_ld();
          const uint32_t nan = nan_seen ? bits[c / 32] : 0;
          if (nan != 0)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (nan >> i & 1) o[i] = 0x7fc00000u;
          if (slot >= 0) {
            // a part: O, and below its maximum and sum, a column of 256 rows each
#pragma unroll
            for (int i = 0; i < 32; ++i) __stcg(&part[(c + i) * (2 * TILE)], __uint_as_float(o[i]) * by);
          } else {
            uint4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              w[i].x = pack2<T>(__uint_as_float(o[8 * i]) * by, __uint_as_float(o[8 * i + 1]) * by);
              w[i].y = pack2<T>(__uint_as_float(o[8 * i + 2]) * by, __uint_as_float(o[8 * i + 3]) * by);
              w[i].z = pack2<T>(__uint_as_float(o[8 * i + 4]) * by, __uint_as_float(o[8 * i + 5]) * by);
              w[i].w = pack2<T>(__uint_as_float(o[8 * i + 6]) * by, __uint_as_float(o[8 * i + 7]) * by);
            }
            if constexpr (L::WRITE4) transpose4(w, lane);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (reals >> (L::WRITE4 ? (lane & ~3) | i : lane) & 1) *reinterpret_cast<uint4 *>(out[i] + c) = w[i];
          }
        }
        if (slot >= 0) {
          __stcg(&part[D * (2 * TILE)], m);
          __stcg(&part[(D + 1) * (2 * TILE)], l);
        }
        tc_before();
      }
    }
  }

  // ---- every MMA issued has completed before the TMEM goes (bounded) ----
  __syncthreads();
  if (*stop != 0 && tid == W_LOAD * 32) {
    // given up: copies in flight land before the block may end (50 ms)
    const unsigned long long t0 = now_ns();
    while (now_ns() - t0 < 50000000ull) {
    }
  }
  if (issuer) {
    tc_commit(&bars.drain, 1);
    if (warp == W_PV) {
      const unsigned long long t0 = now_ns();
      while (!bar_try(smem_addr(&bars.drain), 0))
        if (now_ns() - t0 > WAIT_NS) {
          report(s.status, STATUS_WAIT);
          break;
        }
    }
  }
  __syncthreads();
  if (warp == W_PV) {
    __syncwarp();
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Parts of a cut unit as one, in their order: a CTA takes 8 values of d of the
// unit's 256 rows, a thread a row.
template <int D, typename T>
__global__ void __launch_bounds__(2 * TILE) join_kernel(const AttendParams p) {
  grid_dependency_wait();
  const PlanHead head = *p.plan;
  const JoinRec j = p.joins[blockIdx.x];
  grid_dependency_done();
  if (blockIdx.x >= head.joins || !plan_fits(p, head, j.b, j.start, 0, 0)) return;
  const int row = j.row0 + threadIdx.x, d0 = blockIdx.y * 8;
  if (row >= j.rows) return;
  constexpr int COL = 2 * TILE;
  const float *base = p.tile_partial + int64_t(j.slot0) * (D + 2) * COL + threadIdx.x;
  float m = NONE;
#pragma unroll 8
  for (int c = 0; c < j.parts; ++c) m = fmaxf(m, __ldcg(base + (int64_t(c) * (D + 2) + D) * COL));
  float l = 0.0f, x[8] = {};
#pragma unroll 4
  for (int c = 0; c < j.parts; ++c) {
    const float *at = base + int64_t(c) * (D + 2) * COL;
    const float f = exp2_fast(__ldcg(at + D * COL) - m);
    l += f * __ldcg(at + (D + 1) * COL);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] += f * __ldcg(at + (d0 + i) * COL);
  }
  const float by = l == 0.0f ? 0.0f : 1.0f / l;
  const int token = row / p.group, h = j.head * p.group + row - token * p.group;
  uint4 w;
  w.x = pack2<T>(x[0] * by, x[1] * by);
  w.y = pack2<T>(x[2] * by, x[3] * by);
  w.z = pack2<T>(x[4] * by, x[5] * by);
  w.w = pack2<T>(x[6] * by, x[7] * by);
  *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + (int64_t(j.start) + token) * p.o_ts + h * p.o_hs + d0) = w;
}

template <int D, typename T>
int launch(const AttendParams &p, int device, const PlanShape &shape, cudaStream_t stream) {
  static KernelSetup setup;
  const int rc = setup.ready("emmy_kv8_attend", tiles_kernel<D, T>, device, Layout<D>::DYN, REGS_LAUNCH);
  if (rc != EMMY_OK) return rc;
  return launch_kernel("emmy_kv8_attend", tiles_kernel<D, T>,
                       dim3(unsigned(std::min<int64_t>(shape.most_units, sm_count(device)))), THREADS, Layout<D>::DYN,
                       stream, p);
}
template <int D, typename T>
int launch_join(const AttendParams &p, const PlanShape &shape, cudaStream_t stream) {
  return launch_kernel("emmy_kv8_attend", join_kernel<D, T>, dim3(unsigned(shape.most_joins), D / 8), 2 * TILE, 0,
                       stream, p);
}

}  // namespace

int tiles_attend(const AttendParams &p, const emmy_kv8 &cache, const PlanShape &shape, bool bf16, cudaStream_t stream) {
  const int dev = cache.device;
  if (cache.head_dim == 64)
    return bf16 ? launch<64, __nv_bfloat16>(p, dev, shape, stream) : launch<64, __half>(p, dev, shape, stream);
  return bf16 ? launch<128, __nv_bfloat16>(p, dev, shape, stream) : launch<128, __half>(p, dev, shape, stream);
}

int tiles_join(const AttendParams &p, const emmy_kv8 &cache, const PlanShape &shape, bool bf16, cudaStream_t stream) {
  if (cache.head_dim == 64)
    return bf16 ? launch_join<64, __nv_bfloat16>(p, shape, stream) : launch_join<64, __half>(p, shape, stream);
  return bf16 ? launch_join<128, __nv_bfloat16>(p, shape, stream) : launch_join<128, __half>(p, shape, stream);
}

}  // namespace kv8
