// Norms of queries and keys for each head, with the position rotation in the same pass.
//
//   n = x * rsqrt(mean(x^2) + eps) * w;   (n1, n2) -> (n1 cos a - n2 sin a, n2 cos a + n1 sin a)
//
// Bound: HBM. Every half is read once and written once (4 bytes of traffic an element), against
// about ten fp32 operations, so all that matters is wide loads in flight and no second pass: a
// head lives in the registers of 8, 16 or 32 lanes (8 halves, one 16-byte load, each), the mean
// square is a butterfly over those lanes and the rotation's partner element comes by a shuffle.
// The angles of a token serve all of its heads: one thread per pair forms
// position * inv_freq in fp64 (exact: 31 + 24 bits), reduces it to a turn fraction there and takes sincospi in
// fp32, once per token and CTA, so a far position loses nothing and the fp64 work is 1 / heads of
// what it would be inside the loop.
//
// No counterpart in the reference.

#include <algorithm>

#include "ops_sm100.cuh"

namespace hgemm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalfRot = 128;
constexpr int kMaxTokensPerCta = 4;

struct NormRopeParams {
  const __half *x[2];  // queries, keys
  __half *y[2];
  const __half *w[2];
  long long xs[2], ys[2];
  const int *positions;
  const unsigned char *axis_of;
  const float *inv_freq;
  int tokens, heads_q, heads, head_dim, half_rot, axes;
  float eps, inv_dim;
  int tokens_per_cta, heads_per_cta;
};

__device__ __forceinline__ void unpack8(const uint4 &u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// LANES lanes hold one head, 8 halves each (lanes behind head_dim / 8 hold zeros).
template <int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const NormRopeParams p) {
  constexpr int kGroups = kThreads / LANES;  // heads in flight in this CTA
  __shared__ float s_cos[kMaxTokensPerCta][kMaxHalfRot];
  __shared__ float s_sin[kMaxTokensPerCta][kMaxHalfRot];

  const int t0 = blockIdx.x * p.tokens_per_cta;
  const int nt = min(p.tokens_per_cta, p.tokens - t0);
  for (int i = threadIdx.x; i < nt * p.half_rot; i += kThreads) {
    const int tt = i / p.half_rot, pair = i - tt * p.half_rot;
    const int axis = p.axis_of ? min(static_cast<int>(p.axis_of[pair]), p.axes - 1) : 0;
    const int pos = p.positions[static_cast<long long>(axis) * p.tokens + t0 + tt];
    // angle / pi, reduced to [-1, 1] in fp64.
    const double half_turns =
        static_cast<double>(pos) * static_cast<double>(p.inv_freq[pair]) * 0.31830988618379067154;
    const double r = half_turns - 2.0 * rint(half_turns * 0.5);
    float s, c;
    sincospif(static_cast<float>(r), &s, &c);
    s_cos[tt][pair] = c;
    s_sin[tt][pair] = s;
  }
  __syncthreads();

  const int sub = threadIdx.x % LANES;
  const int e0 = sub * 8;
  const bool live = e0 < p.head_dim;
  const int h0 = blockIdx.y * p.heads_per_cta;
  const int h1 = min(h0 + p.heads_per_cta, p.heads);
  float w[2][8] = {};
  if (live) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      unpack8(__ldg(reinterpret_cast<const uint4 *>(p.w[j] + e0)), w[j]);
  }
  // The rotation of this lane's 8 elements: which angles, and (pairs half a rotation apart) the
  // lane that holds the partners. rot_dim / 2 is a multiple of 8, so a lane's elements are all first
  // halves, all second halves, or all behind the rotation.
  const int rot = 2 * p.half_rot;
  const bool turns = e0 < rot;
  const bool second = !INTERLEAVED && turns && e0 >= p.half_rot;
  const int partner = !turns ? sub : second ? sub - p.half_rot / 8 : sub + p.half_rot / 8;

  for (int tt = 0; tt < nt; ++tt) {
    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      c[j] = 1.0f;
      s[j] = 0.0f;
    }
    if (turns) {
      const int a0 = INTERLEAVED ? e0 / 2 : (second ? e0 - p.half_rot : e0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int a = INTERLEAVED ? a0 + j / 2 : a0 + j;
        c[j] = s_cos[tt][a];
        s[j] = s_sin[tt][a];
        // second element of a pair: n2 cos + n1 sin; first: n1 cos - n2 sin
        const bool sec = INTERLEAVED ? (j & 1) : second;
        if (!sec) s[j] = -s[j];
      }
    }
    const long long token = t0 + tt;
    // Whole passes, so that every lane of a warp takes part in the shuffles. Two heads of a lane
    // group are loaded before either is used.
    for (int hb = h0; hb < h1; hb += 2 * kGroups) {
      uint4 raw[2];
      int head[2];
      bool on[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        head[u] = hb + u * kGroups + static_cast<int>(threadIdx.x) / LANES;
        on[u] = live && head[u] < h1;
        raw[u] = make_uint4(0u, 0u, 0u, 0u);
        if (on[u]) {
          const int j = head[u] >= p.heads_q;
          const int h = head[u] - (j ? p.heads_q : 0);
          raw[u] = *reinterpret_cast<const uint4 *>(
              p.x[j] + token * p.xs[j] + static_cast<long long>(h) * p.head_dim + e0);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x[8], o[8];
        unpack8(raw[u], x);
        float sq = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sq = fmaf(x[j], x[j], sq);
#pragma unroll
        for (int m = LANES / 2; m > 0; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m, LANES);
        const float r = rsqrtf(fmaf(sq, p.inv_dim, p.eps));
        const int jw = head[u] >= p.heads_q;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= r * (jw ? w[1][j] : w[0][j]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y =
              INTERLEAVED ? x[j ^ 1] : __shfl_sync(0xffffffffu, x[j], partner, LANES);
          o[j] = fmaf(x[j], c[j], y * s[j]);
        }
        if (on[u]) {
          const int h = head[u] - (jw ? p.heads_q : 0);
          *reinterpret_cast<uint4 *>(p.y[jw] + token * p.ys[jw] +
                                     static_cast<long long>(h) * p.head_dim + e0) = pack8(o);
        }
      }
    }
  }
}

template <int LANES>
void launch(const NormRopeParams &p, bool interleaved, dim3 grid, cudaStream_t stream) {
  if (interleaved)
    qk_norm_rope_kernel<LANES, true><<<grid, kThreads, 0, stream>>>(p);
  else
    qk_norm_rope_kernel<LANES, false><<<grid, kThreads, 0, stream>>>(p);
}

int check(const hgemm_qk_norm_rope_t *a) {
  if (!a || a->tokens < 0 || a->heads_q < 0 || a->heads_kv < 0) return HGEMM_ERR_INVALID_ARG;
  if (a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8 != 0) return HGEMM_ERR_INVALID_ARG;
  if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 16 != 0)
    return HGEMM_ERR_INVALID_ARG;
  if (a->axes < 1 || (a->axes > 1 && a->rot_dim > 0 && !a->axis_of)) return HGEMM_ERR_INVALID_ARG;
  if (!(a->eps >= 0.0f)) return HGEMM_ERR_INVALID_ARG;
  if (static_cast<long long>(a->heads_q) + a->heads_kv > (1 << 20)) return HGEMM_ERR_TOO_LARGE;
  if (a->tokens == 0 || a->heads_q + a->heads_kv == 0) return HGEMM_OK;
  if (a->rot_dim > 0 && (!a->positions || !a->inv_freq)) return HGEMM_ERR_INVALID_ARG;
  auto operand = [&](const void *in, const void *out, const void *w, long long is, long long os,
                     int heads) {
    if (heads == 0) return true;
    const long long row = static_cast<long long>(heads) * a->head_dim;
    return in && out && w && op_aligned16(in) && op_aligned16(out) && op_aligned16(w) &&
           is % 8 == 0 && os % 8 == 0 && is >= row && os >= row && (in != out || is == os);
  };
  if (!operand(a->q, a->q_out, a->q_weight, a->q_stride, a->q_out_stride, a->heads_q) ||
      !operand(a->k, a->k_out, a->k_weight, a->k_stride, a->k_out_stride, a->heads_kv))
    return HGEMM_ERR_INVALID_ARG;
  return HGEMM_OK;
}

int run(const hgemm_qk_norm_rope_t *a, cudaStream_t stream) {
  int st = check(a);
  if (st != HGEMM_OK || a->tokens == 0 || a->heads_q + a->heads_kv == 0) return st;
  OpDevice d;
  st = op_device(&d);
  if (st != HGEMM_OK) return st;
  NormRopeParams p;
  p.x[0] = a->q;
  p.x[1] = a->k;
  p.y[0] = a->q_out;
  p.y[1] = a->k_out;
  // A side without heads is never indexed by a head, but its weights are loaded.
  p.w[0] = a->heads_q ? a->q_weight : a->k_weight;
  p.w[1] = a->heads_kv ? a->k_weight : a->q_weight;
  p.xs[0] = a->q_stride;
  p.xs[1] = a->k_stride;
  p.ys[0] = a->q_out_stride;
  p.ys[1] = a->k_out_stride;
  p.positions = a->positions;
  p.axis_of = a->axes > 1 ? a->axis_of : nullptr;
  p.inv_freq = a->inv_freq;
  p.tokens = a->tokens;
  p.heads_q = a->heads_q;
  p.heads = a->heads_q + a->heads_kv;
  p.head_dim = a->head_dim;
  p.half_rot = a->rot_dim / 2;
  p.axes = a->axes;
  p.eps = a->eps;
  p.inv_dim = 1.0f / static_cast<float>(a->head_dim);
  const int lanes = a->head_dim <= 64 ? 8 : a->head_dim <= 128 ? 16 : 32;
  const int groups = 2 * kThreads / lanes;
  // A CTA takes whole tokens where there are enough of them to fill the SMs, so that one set of
  // angles serves all heads; with few tokens the heads of one are spread over CTAs (one pass each).
  p.tokens_per_cta =
      std::max(1, std::min(kMaxTokensPerCta, a->tokens / std::max(1, 8 * d.sm_count)));
  p.heads_per_cta = a->tokens >= 2 * d.sm_count ? p.heads : std::min(p.heads, groups);
  const dim3 grid((a->tokens + p.tokens_per_cta - 1) / p.tokens_per_cta,
                  (p.heads + p.heads_per_cta - 1) / p.heads_per_cta);
  if (lanes == 8)
    launch<8>(p, a->interleaved != 0, grid, stream);
  else if (lanes == 16)
    launch<16>(p, a->interleaved != 0, grid, stream);
  else
    launch<32>(p, a->interleaved != 0, grid, stream);
  return cudaGetLastError() == cudaSuccess ? HGEMM_OK : HGEMM_ERR_LAUNCH;
}

}  // namespace
}  // namespace hgemm

extern "C" int hgemm_qk_norm_rope(const hgemm_qk_norm_rope_t *args, hgemm_stream_t stream) {
  return hgemm::op_status(hgemm::run(args, stream));
}
