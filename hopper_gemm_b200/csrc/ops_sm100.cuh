// Shared by the operators that run next to the GEMM (lora.cu, qk_norm_rope.cu, attn_prompt.cu):
// what they take from hgemm_sm100.cu (device check, status word, tensor maps) and the bounded
// mbarrier wait of their kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "hgemm_b200.h"
#include "ptx_sm100.cuh"

namespace hgemm {

// The current device as an operator's launcher needs it.
struct OpDevice {
  int dev;
  int sm_count;
  unsigned *status_word;          // device status word (see hgemm_device_status)
  unsigned long long timeout_ns;  // bound of one wait in a kernel
};
// Checks that the current device is an sm_100 and fills `out`; returns a status code.
int op_device(OpDevice *out);
// Keeps a call's status for hgemm_last_status() and returns it.
int op_status(int status);
// Tensor map of binary16 elements, 128-byte swizzle, zero fill outside: `rank` dimensions,
// innermost first, byte strides of dimensions 1.. .
bool op_encode(CUtensorMap *map, const void *ptr, int rank, const unsigned long long *dims,
               const unsigned long long *strides, const unsigned *box);
// Opts `kernel` in to `smem` bytes of dynamic shared memory on device `dev`, once until hgemm_release()
// (`done` is the caller's per-kernel array of 64 zeros).
int op_smem(const void *kernel, int smem, int dev, unsigned *done);

// The GEMM with additional k-blocks (the second product of low-rank adapters): row tile i of C gets,
// after the k-blocks of A and B, count[i] entries e = base[i].. of `chunks` k-blocks each, whose A
// rows are low[e][chunk][row of the tile][64] and whose B rows are up[adapter[e]][64 chunk ..].
// A 32 x 64 block of C that leaves with an infinity or NaN is listed (row | column << 32).
struct LoraExt {
  const __half *low;
  const __half *up;       // adapters x rank x N
  int entries, chunks, rank, adapters;
  const int *base, *count, *adapter;
  unsigned *odd_count;
  unsigned long long *odd_list;
};
// Rows of a tile that lora_gemm uses for these sizes (128 or 256).
int lora_gemm_tile_rows(int M, int N, int K, int *rows);
// Launched with programmatic serialization: reads `ext` behind a grid_wait.
int lora_gemm(const __half *A, const __half *B, __half *C, int M, int N, int K, const LoraExt &ext,
              cudaStream_t stream);

// The most rows, columns, sequences or segments of a call: the kernels reckon with them in 32 bits, up to a
// grid's step or a tile behind the last one (a binary search adds two segment numbers).
constexpr int kOpMaxRows = 0x7fffffff - 0xffff;
constexpr int kOpMaxSegments = 1 << 30;
constexpr long long kOpMaxStride = 1ll << 38;  // halves (a tensor map ends at 2^40 bytes)

inline bool op_aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// An operand as rows of bytes; rows of one length next to each other may be one long row.
struct OpRows {
  const void *at;
  long long width, stride, rows;
};
inline OpRows op_dense(const void *at, long long bytes) { return {at, bytes, bytes, 1}; }
// The same of a x b x c elements (sizes that no memory holds end at 2^60 bytes).
inline OpRows op_dense(const void *at, int size, double a, double b = 1.0, double c = 1.0) {
  const double bytes = size * a * b * c, most = 1152921504606846976.0;
  return op_dense(at, static_cast<long long>(bytes < most ? bytes : most));
}
// Halves of `heads` heads for each token.
inline OpRows op_heads(const void *at, long long heads, int head_dim, long long stride, long long tokens) {
  return {at, 2 * heads * head_dim, 2 * stride, tokens};
}
// Whether two operands share a byte. (Rows of two different strides, both with gaps, are taken to
// lie in each other's.)
inline bool op_overlap(OpRows a, OpRows b) {
  if (!a.at || !b.at || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
  for (OpRows *r : {&a, &b}) r->rows = r->rows < (1ll << 60) / r->stride ? r->rows : (1ll << 60) / r->stride + 1;
  for (OpRows *r : {&a, &b})
    if (r->rows == 1 || r->width == r->stride) *r = op_dense(r->at, r->width + (r->rows - 1) * r->stride);
  if (a.rows > 1 && b.rows > 1 && a.stride != b.stride) return false;
  // Row i of a and row j of b meet where k = i - j has d - a.width < k * stride < d + b.width.
  const long long stride = a.rows > 1 ? a.stride : b.stride;
  const long long d = static_cast<long long>(reinterpret_cast<uintptr_t>(b.at)) -
                      static_cast<long long>(reinterpret_cast<uintptr_t>(a.at));
  const long long low = d - a.width;
  long long k = low >= 0 ? low / stride + 1 : -((-low - 1) / stride);  // the first above low
  k = k < 1 - b.rows ? 1 - b.rows : k;
  return k <= a.rows - 1 && k * stride < d + b.width;
}

// Wait sites of the operators' kernels in the device status word (the GEMM uses 1..12).
enum OpWaitSite : unsigned {
  kSiteAttnQ = 32,
  kSiteAttnKvFull = 33,
  kSiteAttnKvEmpty = 34,
  kSiteAttnScores = 35,
  kSiteAttnWeights = 36,
  kSiteAttnOut = 37,
  kSiteLoraEmpty = 40,
  kSiteLoraFull = 41,
  kSiteLoraAcc = 42,
  kSiteLoraFewEmpty = 43,
  kSiteLoraFewFull = 44,
  kSiteLoraFewAcc = 45,
};

// Bounded wait of one thread; false when the CTA is unwinding or the wait ran out (recorded in
// the device status word, and the CTA's abort flag raised so that every role unwinds).
struct OpWait {
  volatile int *abort_flag;  // shared memory
  unsigned *status_word;
  unsigned long long timeout_ns;
};
__device__ __forceinline__ bool op_wait(uint32_t bar, uint32_t parity, const OpWait &w,
                                        unsigned site) {
  // Polls without suspending: a suspended thread comes back late, which a chain of short waits
  // (scores, weights, products) pays at every link.
  if (ptx::mbar_test_wait(bar, parity)) return true;
  const uint64_t t0 = ptx::globaltimer();
  for (uint32_t n = 1;; ++n) {
    if (ptx::mbar_test_wait(bar, parity)) return true;
    if ((n & 255u) == 0) {
      if (*w.abort_flag) return false;
      if (ptx::globaltimer() - t0 > w.timeout_ns) {
        atomicCAS(w.status_word, 0u, 0x100u | site);
        *w.abort_flag = 1;
        return false;
      }
    }
  }
}
// Teardown form: ignores the abort flag and records nothing.
__device__ __forceinline__ void op_drain(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = ptx::globaltimer();
  while (!ptx::mbar_try_wait(bar, parity))
    if (ptx::globaltimer() - t0 > 50000000ull) return;
}

}  // namespace hgemm
