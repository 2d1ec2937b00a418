// Shared by the kernels of the paged 8-bit key/value cache (kv8_*.cu).
//
// A cache layer is a pool of pages codes[page][K or V][kv head][slot][d] in
// e4m3 and one exponent exps[page][K or V][kv head]; a held value is
// code * 2^exp.  The scale is a power of two because e4m3 is a floating
// format: a general scale buys no precision, only a better fit of the top
// binade, while a power of two makes every held value exact in f16 and bf16
// after scaling, makes a change of scale exact above e4m3's subnormals, and
// lets the kernels fold it into exponents they compute anyway.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "emmyrt.h"

namespace kv8 {

// Exponents of a page.  448 * 2^63 = 4e21 is the largest magnitude held.  The
// span of 95 keeps an accumulator of 2^16 terms of 448 with weights of 2^8 (the
// most the running maximum lags) finite in f32 when it moves from the units of
// the largest pages to those of the smallest.
constexpr int E_MIN = -32, E_MAX = 63;

// What a kernel leaves in the status word (0: nothing was wrong).
constexpr unsigned STATUS_PAGE = 0x401;    // a page number outside the pool
constexpr unsigned STATUS_LENGTH = 0x402;  // a sequence longer than its row of the table, or
                                           // more new tokens than keys, than rows given or than max_q
constexpr unsigned STATUS_WAIT = 0x403;    // a bounded wait inside a kernel ran out
constexpr unsigned STATUS_PLAN = 0x404;    // a plan that was made for another call

struct Seqs {
  const int *table;     // [seqs][width] page numbers
  const int *kv_lens;   // [seqs] keys, the new tokens included
  const int *q_starts;  // [seqs + 1] first row of each sequence's new tokens
  unsigned *status;     // may be null
  int seqs, width, pages, tokens, max_q, kv_heads, page_shift;
};

__device__ __forceinline__ void report(unsigned *status, unsigned code) {
  if (status != nullptr) *status = code;
}

// n, or 0 (nothing to do), reported, where the lengths cannot be right.
__device__ __forceinline__ int checked_n(const Seqs &s, int start, int n, int len) {
  if (n >= 0 && n <= len && n <= s.max_q && start >= 0 && start <= s.tokens - n && len <= (int64_t(s.width) << s.page_shift)) return n;
  report(s.status, STATUS_LENGTH);
  return 0;
}
// Lengths of sequence b: first row, new tokens, keys.
__device__ __forceinline__ void lengths(const Seqs &s, int b, int &start, int &n, int &len) {
  start = s.q_starts[b];
  n = s.q_starts[b + 1] - start;
  len = s.kv_lens[b];
  n = checked_n(s, start, n, len);
}

// Two e4m3 codes (bits 0-15 of w) as f16x2; every e4m3 value is exact in f16.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(w)));
  return r;
}

// hi, lo -> packed e4m3x2 (round to nearest even, saturating; NaN -> 0x7f).
__device__ __forceinline__ uint32_t f32x2_e4m3x2(float hi, float lo) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Exponent of a page's side and head as the kernels take it: adopted storage may
// hold any.
__device__ __forceinline__ int held_exponent(int held) { return max(min(held, E_MAX), E_MIN); }

__device__ __forceinline__ float pow2(int e) {  // -126 <= e <= 127
  return __int_as_float((e + 127) << 23);
}

// 0x80 in each byte of w whose code is NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// The kernels start with the end of the one before them in the stream
// (programmatic dependent launch): they wait for it, and for all it wrote,
// before they read anything, and let the next one be set up meanwhile.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_done() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Status of a call, with its message for emmy_last_error().
int fail(int code, const char *what, const char *msg);
int cuda_fail(const char *what, cudaError_t e);

// Makes `device` the runtime's current device for a scope.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    err = cudaGetDevice(&prev_);
    if (err == cudaSuccess && prev_ != device) {
      err = cudaSetDevice(device);
      moved_ = err == cudaSuccess;
    }
  }
  ~OnDevice() {
    if (moved_) cudaSetDevice(prev_);
  }
  cudaError_t err = cudaSuccess;

 private:
  int prev_ = 0;
  bool moved_ = false;
};

// What a kernel needs once on each device: its dynamic shared memory allowed,
// and (regs > 0) the register count that its register split counts on.
class KernelSetup {
 public:
  template <typename K>
  int ready(const char *what, K *kernel, int device, int smem, int regs = 0) {
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (done_.load(std::memory_order_acquire) & bit) return EMMY_OK;
    cudaError_t e = cudaSuccess;
    if (regs > 0) {
      cudaFuncAttributes at;
      e = cudaFuncGetAttributes(&at, kernel);
      if (e == cudaSuccess && at.numRegs != regs)
        return fail(EMMY_ECUDART, what, "the kernel was built with another register count than its split needs");
    }
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(what, e);
    done_.fetch_or(bit, std::memory_order_release);
    return EMMY_OK;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

template <typename... A>
int launch_clusters(const char *what, void (*kernel)(A...), int cluster, dim3 grid, int threads, int smem,
                    cudaStream_t stream, const A &...args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  c.attrs = attr;
  c.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&c, kernel, args...);
  return e == cudaSuccess ? EMMY_OK : cuda_fail(what, e);
}

template <typename... A>
int launch_kernel(const char *what, void (*kernel)(A...), dim3 grid, int threads, int smem, cudaStream_t stream,
                  const A &...args) {
  return launch_clusters(what, kernel, 1, grid, threads, smem, stream, args...);
}

// Checks what every call shares and fills the kernels' view of the sequences.
int check_cache(const char *what, const emmy_kv8 *c);
int check_counts(const char *what, const emmy_kv8 *c);  // of the sequences, without their arrays
int check_seqs(const char *what, const emmy_kv8 *c);
Seqs seqs_of(const emmy_kv8 &c);
int sm_count(int device);
// Counts a call that goes into a capture of `stream` (40 ns a call).
void note_capture(cudaStream_t stream);
// Limit of the kernels' waits, in ns, and the blocks that are to wait in vain.
void wait_limit(unsigned long long &ns, int &stall);
// Whether [a, a + na) and [b, b + nb) share a byte.
inline bool overlap(emmy_dptr a, uint64_t na, emmy_dptr b, uint64_t nb) {
  return a < b + nb && b < a + na;
}

}  // namespace kv8
