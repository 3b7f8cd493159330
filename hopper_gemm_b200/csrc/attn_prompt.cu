// Attention over packed sequences with grouped heads (whole prompts, appended prompts, single
// tokens): O = softmax(scale * Q K^T) V for each sequence and head.
//
// No counterpart in the reference.

#include <algorithm>

#include "ops_sm100.cuh"

namespace hgemm {
namespace {

constexpr int kMaxDim = 128;

struct AttnParams {
  const __half *q, *k, *v;
  __half *out;
  float *lse;
  const int *cu_q, *cu_k;
  long long q_stride, k_stride, v_stride, out_stride;
  int total_q, total_k, batch, heads_q, heads_kv, group, head_dim, causal;
  float scale;
};

// Rows [begin, end) of sequence s, cut off at the rows that the tensor holds.
__device__ __forceinline__ void seq_range(const int *cu, int s, int total, int &begin, int &end) {
  begin = min(max(cu[s], 0), total);
  end = min(max(cu[s + 1], begin), total);
}

// One query row over keys [j0, j1) of its sequence, by one warp, in the order of the keys: lane l
// holds elements 4l..4l+3. Leaves the weighted sum relative to the maximum m (log2 units).
__device__ void attn_row(const AttnParams &p, const __half *qrow, const __half *k, const __half *v,
                         int j0, int j1, float (&o)[4], float &m, float &l) {
  const int e0 = 4 * (threadIdx.x & 31);
  const bool live = e0 < p.head_dim;  // head_dim is a multiple of 8
  const float scale2 = p.scale * 1.44269504088896340736f;
  auto load4 = [&](const __half *src, float (&f)[4]) {
    uint2 u = make_uint2(0u, 0u);
    if (live) u = *reinterpret_cast<const uint2 *>(src + e0);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    f[0] = a.x;
    f[1] = a.y;
    f[2] = b.x;
    f[3] = b.y;
  };
  float q[4];
  load4(qrow, q);
  m = -INFINITY;
  l = 0.0f;
  o[0] = o[1] = o[2] = o[3] = 0.0f;
  for (int j = j0; j < j1; ++j) {
    float kk[4], vv[4];
    load4(k + j * p.k_stride, kk);
    load4(v + j * p.v_stride, vv);
    float s = q[0] * kk[0] + q[1] * kk[1] + q[2] * kk[2] + q[3] * kk[3];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= scale2;
    if (s > m) {
      const float f = exp2f(m - s);
      l *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= f;
      m = s;
    }
    const float w = (s == -INFINITY && m == -INFINITY) ? 0.0f : exp2f(s - m);
    l += w;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(w, vv[i], o[i]);
  }
}

// One warp for each (query, head).
__global__ void __launch_bounds__(256) attn_rows_kernel(const AttnParams p) {
  const long long row = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (row >= static_cast<long long>(p.total_q) * p.heads_q) return;
  const int i = static_cast<int>(row / p.heads_q), h = static_cast<int>(row % p.heads_q);
  int s = -1, q0 = 0, q1 = 0;
  for (int b = 0; b < p.batch; ++b) {
    seq_range(p.cu_q, b, p.total_q, q0, q1);
    if (i >= q0 && i < q1) {
      s = b;
      break;
    }
  }
  if (s < 0) return;
  int k0, k1;
  seq_range(p.cu_k, s, p.total_k, k0, k1);
  const int klen = k1 - k0;
  const int seen = p.causal ? max(0, min(klen, i - q0 + 1 + klen - (q1 - q0))) : klen;
  float o[4], m, l;
  const long long hk = static_cast<long long>(h / p.group) * p.head_dim;
  attn_row(p, p.q + i * p.q_stride + static_cast<long long>(h) * p.head_dim,
           p.k + k0 * p.k_stride + hk, p.v + k0 * p.v_stride + hk, 0, seen, o, m, l);
  const float inv = seen > 0 ? 1.0f / l : 0.0f;
  if (4 * lane < p.head_dim) {
    uint2 u;
    const __half2 a = __floats2half2_rn(o[0] * inv, o[1] * inv);
    const __half2 b = __floats2half2_rn(o[2] * inv, o[3] * inv);
    u.x = *reinterpret_cast<const uint32_t *>(&a);
    u.y = *reinterpret_cast<const uint32_t *>(&b);
    *reinterpret_cast<uint2 *>(p.out + i * p.out_stride + static_cast<long long>(h) * p.head_dim +
                               4 * lane) = u;
  }
  if (lane == 0 && p.lse)
    p.lse[row] = seen > 0 ? (m + log2f(l)) * 0.69314718055994530942f : -INFINITY;
}

int check(const hgemm_attn_prompt_t *a) {
  if (!a || a->total_q < 0 || a->total_k < 0 || a->batch < 0) return HGEMM_ERR_INVALID_ARG;
  if (a->heads_kv < 1 || a->heads_q < a->heads_kv || a->heads_q % a->heads_kv != 0 ||
      a->heads_q / a->heads_kv > 128)
    return HGEMM_ERR_INVALID_ARG;
  if (a->head_dim < 8 || a->head_dim > kMaxDim || a->head_dim % 8 != 0)
    return HGEMM_ERR_INVALID_ARG;
  if (!(a->scale >= 0.0f) || a->scale - a->scale != 0.0f) return HGEMM_ERR_INVALID_ARG;
  if (a->total_q == 0 || a->batch == 0) return HGEMM_OK;
  if (!a->q || !a->out || !a->cu_q) return HGEMM_ERR_INVALID_ARG;
  if (!a->cu_k && a->total_k != a->total_q) return HGEMM_ERR_INVALID_ARG;
  if (a->total_k > 0 && (!a->k || !a->v)) return HGEMM_ERR_INVALID_ARG;
  if (!op_aligned16(a->q) || !op_aligned16(a->k) || !op_aligned16(a->v) || !op_aligned16(a->out))
    return HGEMM_ERR_INVALID_ARG;
  const long long qrow = static_cast<long long>(a->heads_q) * a->head_dim;
  const long long krow = static_cast<long long>(a->heads_kv) * a->head_dim;
  if (a->q_stride < qrow || a->out_stride < qrow || a->k_stride < krow || a->v_stride < krow)
    return HGEMM_ERR_INVALID_ARG;
  if (a->q_stride % 8 || a->out_stride % 8 || a->k_stride % 8 || a->v_stride % 8)
    return HGEMM_ERR_INVALID_ARG;
  return HGEMM_OK;
}

int run(const hgemm_attn_prompt_t *a, cudaStream_t stream) {
  int st = check(a);
  if (st != HGEMM_OK || a->total_q == 0 || a->batch == 0) return st;
  OpDevice d;
  st = op_device(&d);
  if (st != HGEMM_OK) return st;
  AttnParams p;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.lse = a->lse;
  p.cu_q = a->cu_q;
  p.cu_k = a->cu_k ? a->cu_k : a->cu_q;
  p.q_stride = a->q_stride;
  p.k_stride = a->k_stride;
  p.v_stride = a->v_stride;
  p.out_stride = a->out_stride;
  p.total_q = a->total_q;
  p.total_k = a->total_k;
  p.batch = a->batch;
  p.heads_q = a->heads_q;
  p.heads_kv = a->heads_kv;
  p.group = a->heads_q / a->heads_kv;
  p.head_dim = a->head_dim;
  p.causal = a->causal != 0;
  p.scale = a->scale;
  const long long blocks = (static_cast<long long>(a->total_q) * a->heads_q + 7) / 8;
  if (blocks > 0x7fffffffll) return HGEMM_ERR_TOO_LARGE;
  attn_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? HGEMM_OK : HGEMM_ERR_LAUNCH;
}

}  // namespace
}  // namespace hgemm

extern "C" {

int hgemm_attn_prompt(const hgemm_attn_prompt_t *args, hgemm_stream_t stream) {
  return hgemm::op_status(hgemm::run(args, stream));
}

size_t hgemm_attn_prompt_workspace_bytes(int total_q, int total_k, int batch, int heads_q,
                                         int heads_kv, int head_dim) {
  (void)total_q, (void)total_k, (void)batch, (void)heads_q, (void)heads_kv, (void)head_dim;
  return 0;
}

}  // extern "C"
