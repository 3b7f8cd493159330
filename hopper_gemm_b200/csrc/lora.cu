// A shared projection with the low-rank adapters of many requests beside it:
//   Y[t,:] = X[t,:] W + scale[a] * (X[t,:] Down[a]) Up[a].
//
// No counterpart in the reference.

#include <algorithm>

#include "ops_sm100.cuh"

namespace hgemm {
namespace {

constexpr int kMaxRank = 256;

struct LoraParams {
  const __half *X, *W, *down, *up;
  __half *Y;
  const float *scale;
  const int *seg_start, *seg_adapter;
  float *low;  // tokens x rank
  int tokens, N, K, rank, adapters, segments;
};

// Adapter of token t, or -1: binary search for the last segment that starts at or before t.
__device__ __forceinline__ int token_adapter(const int *seg_start, const int *seg_adapter,
                                             int segments, int adapters, int t) {
  int lo = 0, hi = segments;  // seg_start[lo] <= t < seg_start[hi], if any segment holds t
  if (segments <= 0 || t < seg_start[0] || t >= seg_start[segments]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (seg_start[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  const int a = seg_adapter[lo];
  return (a >= 0 && a < adapters) ? a : -1;
}

__global__ void __launch_bounds__(256) lora_shrink_rows_kernel(const LoraParams p) {
  const int t = blockIdx.x;
  const int a = token_adapter(p.seg_start, p.seg_adapter, p.segments, p.adapters, t);
  if (a < 0) return;
  const __half *x = p.X + static_cast<long long>(t) * p.K;
  const __half *dn = p.down + static_cast<long long>(a) * p.K * p.rank;
  for (int r = threadIdx.x; r < p.rank; r += 256) {
    float acc = 0.0f;
    for (int k = 0; k < p.K; ++k)
      acc = fmaf(__half2float(x[k]), __half2float(dn[static_cast<long long>(k) * p.rank + r]), acc);
    p.low[static_cast<long long>(t) * p.rank + r] = acc * p.scale[a];
  }
}

// One thread for each output: the shared product and the adapter's part in one fp32 sum.
__global__ void __launch_bounds__(256) lora_rows_kernel(const LoraParams p) {
  const int t = blockIdx.x;
  const int a = token_adapter(p.seg_start, p.seg_adapter, p.segments, p.adapters, t);
  const int n = blockIdx.y * 256 + threadIdx.x;
  if (n >= p.N) return;
  const __half *x = p.X + static_cast<long long>(t) * p.K;
  float acc = 0.0f;
  for (int k = 0; k < p.K; ++k)
    acc = fmaf(__half2float(x[k]), __half2float(p.W[static_cast<long long>(k) * p.N + n]), acc);
  if (a >= 0) {
    const __half *up = p.up + static_cast<long long>(a) * p.rank * p.N;
    for (int r = 0; r < p.rank; ++r)
      acc = fmaf(p.low[static_cast<long long>(t) * p.rank + r],
                 __half2float(up[static_cast<long long>(r) * p.N + n]), acc);
  }
  p.Y[static_cast<long long>(t) * p.N + n] = __float2half_rn(acc);
}

bool sizes_ok(int tokens, int N, int K, int rank, int adapters, int segments) {
  return tokens >= 0 && N >= 0 && K >= 8 && N % 8 == 0 && K % 8 == 0 && rank >= 8 &&
         rank <= kMaxRank && rank % 8 == 0 && adapters >= 0 && segments >= 0;
}

int check(const hgemm_lora_t *a) {
  if (!a || !sizes_ok(a->tokens, a->N, a->K, a->rank, a->adapters, a->segments))
    return HGEMM_ERR_INVALID_ARG;
  if (a->tokens == 0 || a->N == 0) return HGEMM_OK;
  if (!a->X || !a->W || !a->Y || !op_aligned16(a->X) || !op_aligned16(a->W) || !op_aligned16(a->Y))
    return HGEMM_ERR_INVALID_ARG;
  if (a->segments > 0 && (!a->seg_start || !a->seg_adapter)) return HGEMM_ERR_INVALID_ARG;
  if (a->adapters > 0 && a->segments > 0 &&
      (!a->down || !a->up || !a->scale || !op_aligned16(a->down) || !op_aligned16(a->up)))
    return HGEMM_ERR_INVALID_ARG;
  const size_t need = hgemm_lora_workspace_bytes(a->tokens, a->N, a->K, a->rank, a->adapters,
                                                 a->segments);
  if (need > 0 && (!a->workspace || !op_aligned16(a->workspace) || a->workspace_bytes < need))
    return HGEMM_ERR_INVALID_ARG;
  return HGEMM_OK;
}

int run(const hgemm_lora_t *a, cudaStream_t stream) {
  int st = check(a);
  if (st != HGEMM_OK || a->tokens == 0 || a->N == 0) return st;
  OpDevice d;
  st = op_device(&d);
  if (st != HGEMM_OK) return st;
  LoraParams p;
  p.X = a->X;
  p.W = a->W;
  p.down = a->down;
  p.up = a->up;
  p.Y = a->Y;
  p.scale = a->scale;
  p.seg_start = a->seg_start;
  p.seg_adapter = a->seg_adapter;
  p.low = static_cast<float *>(a->workspace);
  p.tokens = a->tokens;
  p.N = a->N;
  p.K = a->K;
  p.rank = a->rank;
  p.adapters = a->adapters;
  p.segments = a->segments;
  if (p.adapters == 0) p.segments = 0;
  if (p.segments > 0) lora_shrink_rows_kernel<<<p.tokens, 256, 0, stream>>>(p);
  lora_rows_kernel<<<dim3(p.tokens, (p.N + 255) / 256), 256, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? HGEMM_OK : HGEMM_ERR_LAUNCH;
}

}  // namespace
}  // namespace hgemm

extern "C" {

int hgemm_lora(const hgemm_lora_t *args, hgemm_stream_t stream) {
  return hgemm::op_status(hgemm::run(args, stream));
}

size_t hgemm_lora_workspace_bytes(int tokens, int N, int K, int rank, int adapters, int segments) {
  if (!hgemm::sizes_ok(tokens, N, K, rank, adapters, segments)) return 0;
  if (adapters == 0 || segments == 0) return 0;
  return static_cast<size_t>(tokens) * rank * sizeof(float);
}

}  // extern "C"
