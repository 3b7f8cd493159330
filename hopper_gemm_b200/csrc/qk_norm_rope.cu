// Norms of queries and keys for each head, with the position rotation in the same pass.
//
//   n = x * rsqrt(mean(x^2) + eps) * w;   (n1, n2) -> (n1 cos a - n2 sin a, n2 cos a + n1 sin a)
//
// Bound: HBM. Every half is read once and written once (4 bytes of traffic an element), against
// about ten fp32 operations, so what matters is loads in flight and few instructions beside them. A
// head lives in the registers of 8, 16 or 32 lanes, 8 halves each: four consecutive ones and the four
// that they turn with (half a rotation away, or next to them when pairs are adjacent), so that the
// rotation needs no other lane and the mean square is the only exchange. Two heads of a lane group are
// loaded while the two before them are worked on.
// The angles of a token serve all of its heads: one thread for each pair forms position * inv_freq in
// fp64 (exact: 31 + 24 bits), reduces it to a turn there and takes sincospi in fp32, once per
// token and CTA, while the first heads are on their way.
//
// No counterpart in the reference.

#include <algorithm>

#include "ops_sm100.cuh"

namespace hgemm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalfRot = 128;
constexpr int kMaxTokensPerCta = 2;
constexpr int kMaxHeads = 1 << 14;  // on each side: item / heads by a 32-bit multiplication is exact

struct NormRopeParams {
  const __half *x[2];  // queries, keys
  __half *y[2];
  const __half *w[2];
  long long xs[2], ys[2];
  int heads[2];
  unsigned magic[2];  // ceil(2^32 / heads): item -> token of this CTA
  const int *positions;
  const unsigned char *axis_of;
  const float *inv_freq;
  int tokens, head_dim, half_rot, axes;
  float eps, inv_dim;
  int tokens_per_cta, parts;  // a token's heads are spread over `parts` CTAs
};

struct Item {
  uint2 a, b;
  __half *y;  // null: nothing to do
  int tt;
};

__device__ __forceinline__ float4 unpack4(const uint2 &u) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
  const __half2 u = __floats2half2_rn(a, b), v = __floats2half2_rn(c, d);
  return make_uint2(*reinterpret_cast<const uint32_t *>(&u), *reinterpret_cast<const uint32_t *>(&v));
}

// LANES lanes hold one head (lanes behind head_dim / 8 hold zeros).
template <int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 4) qk_norm_rope_kernel(const NormRopeParams p) {
  constexpr int kGroups = kThreads / LANES;  // heads in flight in this CTA
  __shared__ __align__(16) float s_cos[kMaxTokensPerCta][kMaxHalfRot];
  __shared__ __align__(16) float s_sin[kMaxTokensPerCta][kMaxHalfRot];

  const int part = blockIdx.x % p.parts;
  const int t0 = blockIdx.x / p.parts * p.tokens_per_cta;
  const int nt = min(p.tokens_per_cta, p.tokens - t0);
  const int sub = threadIdx.x % LANES;
  const bool live = 8 * sub < p.head_dim;
  // This lane's two groups of four elements, and its first angle.
  const bool turns = INTERLEAVED ? 8 * sub < 2 * p.half_rot : 4 * sub < p.half_rot;
  int oa = 8 * sub, ob = 8 * sub + 4;
  if (!INTERLEAVED) {
    // Lanes behind the rotation hold eight elements in a row: 2 half_rot + 8 (sub - half_rot / 4).
    if (turns) {
      oa = 4 * sub;
      ob = p.half_rot + 4 * sub;
    }
  }
  const int first = part * kGroups + static_cast<int>(threadIdx.x) / LANES;
  const int step = kGroups * p.parts;

  auto load = [&](int side, int i) {
    Item it;
    it.a = it.b = make_uint2(0u, 0u);
    it.y = nullptr;
    it.tt = 0;
    if (live && i < nt * p.heads[side]) {
      const int tt = static_cast<int>(__umulhi(static_cast<unsigned>(i), p.magic[side]));
      const int tk = p.heads[side] == 1 ? i : tt;
      const long long col = static_cast<long long>(i - tk * p.heads[side]) * p.head_dim;
      const __half *x = p.x[side] + (t0 + tk) * p.xs[side] + col;
      it.a = *reinterpret_cast<const uint2 *>(x + oa);
      it.b = *reinterpret_cast<const uint2 *>(x + ob);
      it.y = p.y[side] + (t0 + tk) * p.ys[side] + col;
      it.tt = tk;
    }
    return it;
  };
  auto work = [&](const Item &it, const float4 &wa, const float4 &wb) {
    float4 xa = unpack4(it.a), xb = unpack4(it.b);
    float sq = xa.x * xa.x;
    sq = fmaf(xa.y, xa.y, sq);
    sq = fmaf(xa.z, xa.z, sq);
    sq = fmaf(xa.w, xa.w, sq);
    sq = fmaf(xb.x, xb.x, sq);
    sq = fmaf(xb.y, xb.y, sq);
    sq = fmaf(xb.z, xb.z, sq);
    sq = fmaf(xb.w, xb.w, sq);
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m, LANES);
    if (!it.y) return;
    const float r = rsqrtf(fmaf(sq, p.inv_dim, p.eps));
    xa.x *= wa.x * r;
    xa.y *= wa.y * r;
    xa.z *= wa.z * r;
    xa.w *= wa.w * r;
    xb.x *= wb.x * r;
    xb.y *= wb.y * r;
    xb.z *= wb.z * r;
    xb.w *= wb.w * r;
    if (turns) {
      const float4 c = *reinterpret_cast<const float4 *>(&s_cos[it.tt][4 * sub]);
      const float4 s = *reinterpret_cast<const float4 *>(&s_sin[it.tt][4 * sub]);
      if (INTERLEAVED) {
        const float4 ya = xa, yb = xb;
        xa.x = fmaf(ya.x, c.x, -ya.y * s.x);
        xa.y = fmaf(ya.y, c.x, ya.x * s.x);
        xa.z = fmaf(ya.z, c.y, -ya.w * s.y);
        xa.w = fmaf(ya.w, c.y, ya.z * s.y);
        xb.x = fmaf(yb.x, c.z, -yb.y * s.z);
        xb.y = fmaf(yb.y, c.z, yb.x * s.z);
        xb.z = fmaf(yb.z, c.w, -yb.w * s.w);
        xb.w = fmaf(yb.w, c.w, yb.z * s.w);
      } else {
        const float4 ya = xa;
        xa.x = fmaf(ya.x, c.x, -xb.x * s.x);
        xa.y = fmaf(ya.y, c.y, -xb.y * s.y);
        xa.z = fmaf(ya.z, c.z, -xb.z * s.z);
        xa.w = fmaf(ya.w, c.w, -xb.w * s.w);
        xb.x = fmaf(xb.x, c.x, ya.x * s.x);
        xb.y = fmaf(xb.y, c.y, ya.y * s.y);
        xb.z = fmaf(xb.z, c.z, ya.z * s.z);
        xb.w = fmaf(xb.w, c.w, ya.w * s.w);
      }
    }
    *reinterpret_cast<uint2 *>(it.y + oa) = pack4(xa.x, xa.y, xa.z, xa.w);
    *reinterpret_cast<uint2 *>(it.y + ob) = pack4(xb.x, xb.y, xb.z, xb.w);
  };

  Item next[2] = {load(0, first), load(0, first + step)};
  for (int i = threadIdx.x; i < nt * p.half_rot; i += kThreads) {
    const int tt = i >= p.half_rot, pair = i - tt * p.half_rot;
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

#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    float4 wa = make_float4(0.0f, 0.0f, 0.0f, 0.0f), wb = wa;
    if (live && p.heads[side] > 0) {
      wa = unpack4(__ldg(reinterpret_cast<const uint2 *>(p.w[side] + oa)));
      wb = unpack4(__ldg(reinterpret_cast<const uint2 *>(p.w[side] + ob)));
    }
    // Whole passes, so that every lane of a warp takes part in the exchange.
    const int n = nt * p.heads[side];
#pragma unroll 1
    for (int i = first; i - first + part * kGroups < n; i += 2 * step) {
      const Item now[2] = {next[0], next[1]};
      const int j = i + 2 * step;
      const bool more = j - first + part * kGroups < n;
      const int side2 = more ? side : 1, at = more ? j : first;
      if (more || side == 0) {
        next[0] = load(side2, at);
        next[1] = load(side2, at + step);
      }
      work(now[0], wa, wb);
      work(now[1], wa, wb);
    }
    if (side == 0 && part * kGroups >= n) {
      next[0] = load(1, first);  // no queries here: the keys were not yet asked for
      next[1] = load(1, first + step);
    }
  }
}

template <int LANES>
void launch(const NormRopeParams &p, bool interleaved, unsigned grid, cudaStream_t stream) {
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
  if (a->heads_q > kMaxHeads || a->heads_kv > kMaxHeads) return HGEMM_ERR_TOO_LARGE;
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
  p.w[0] = a->q_weight;
  p.w[1] = a->k_weight;
  p.xs[0] = a->q_stride;
  p.xs[1] = a->k_stride;
  p.ys[0] = a->q_out_stride;
  p.ys[1] = a->k_out_stride;
  p.heads[0] = a->heads_q;
  p.heads[1] = a->heads_kv;
  for (int j = 0; j < 2; ++j)
    p.magic[j] = p.heads[j] > 1 ? static_cast<unsigned>((0x100000000ull + p.heads[j] - 1) / p.heads[j]) : 0u;
  p.positions = a->positions;
  p.axis_of = a->axes > 1 ? a->axis_of : nullptr;
  p.inv_freq = a->inv_freq;
  p.tokens = a->tokens;
  p.head_dim = a->head_dim;
  p.half_rot = a->rot_dim / 2;
  p.axes = a->axes;
  p.eps = a->eps;
  p.inv_dim = 1.0f / static_cast<float>(a->head_dim);
  const int lanes = a->head_dim <= 64 ? 8 : a->head_dim <= 128 ? 16 : 32;
  const int groups = kThreads / lanes;
  // Two tokens to a CTA where that still fills the SMs several times over; with few tokens the heads
  // of one are spread over CTAs (one head to a lane group).
  p.tokens_per_cta = a->tokens >= 16 * d.sm_count ? 2 : 1;
  const int most = std::max(a->heads_q, a->heads_kv);
  p.parts = a->tokens >= 2 * d.sm_count ? 1 : (most + groups - 1) / groups;
  const long long ctas =
      static_cast<long long>((a->tokens + p.tokens_per_cta - 1) / p.tokens_per_cta) * p.parts;
  if (ctas > 0x7fffffffll) return HGEMM_ERR_TOO_LARGE;
  const unsigned grid = static_cast<unsigned>(ctas);
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
