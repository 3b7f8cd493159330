// Norms of queries and keys for each head, with the position rotation in the same pass.
//
//   n = x * rsqrt(mean(x^2) + eps) * w;   (n1, n2) -> (n1 cos a - n2 sin a, n2 cos a + n1 sin a)
//
// Bound: loads in flight to HBM (ncu: DRAM and issue at 45% each). Every half is read once and written once (4
// bytes of traffic an element), against about ten fp32 operations, so what matters is loads in flight and few
// instructions beside them.
// Norm weight and rotation are one: element e becomes r (x_e A_e + x_partner B_e), with A and B (weight
// times cos, weight times sin) formed once for a token and side, and two elements go into an
// instruction (fma.rn.f32x2). A warp takes a token: its lane groups of a few lanes hold a head each, 16
// halves a lane: eight consecutive ones and the eight that they turn with (half a rotation away, or
// next to them when pairs are adjacent), so that the rotation needs no other lane, the mean square is
// the only exchange, and A and B stay in registers over all heads of a side. The heads of the next two
// passes are on their way while one is worked on.
// The angles: one lane for each pair forms position * inv_freq / pi in fp64 (three roundings: at a position of 2^31 off by
// 2^-22 of half a turn), reduces it to a turn there and takes sincospi in fp32, while the token's first heads are loaded.
// Forms in which a CTA's warps shared a token (through registers, or a ring of bulk copies) took 37 us
// for 8191 tokens of 40 heads of 128: A and B came from shared memory for every head, whose bandwidth
// was then the bound. Measured: 36 us, 4.6 TB/s (a contiguous copy of the same bytes takes 30 to 31); 2500 tokens
// of 32 heads of 80, where one wave of warps has a token each and latency counts, 12.3 us; a call of 48 tokens 5.4.
//
// No counterpart in the reference.

#include <algorithm>

#include "ops_sm100.cuh"

namespace hgemm {
namespace {

constexpr int kWarps = 4;  // of a CTA
constexpr int kCtasPerSm = 5;
constexpr int kMaxHeads = 1 << 20;

struct NormRopeParams {
  const __half *x[2];  // queries, keys
  __half *y[2];
  const __half *w[2];
  long long xs[2], ys[2];
  const int *positions;
  const unsigned char *axis_of;
  const float *inv_freq;
  int tokens, heads[2], head_dim, half_rot, axes;
  float eps, inv_dim;
  // A warp passes over the heads in steps of one head to a lane group: `passes[0]` over the queries,
  // then those over the keys. A token's passes are shared by `parts` warps.
  int passes[2], parts;
};

__device__ __forceinline__ void unpack8(const uint4 &u, float2 (&f)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
}

__device__ __forceinline__ uint4 pack8(const float2 (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __float22half2_rn(f[i]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// r (x A + y B) for eight elements x with their partners y.
__device__ __forceinline__ uint4 turn8(const float2 (&x)[4], const float2 (&y)[4],
                                       const float2 (&A)[4], const float2 (&B)[4], float2 r) {
  float2 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = __fmul2_rn(__ffma2_rn(x[i], A[i], __fmul2_rn(y[i], B[i])), r);
  return pack8(o);
}

__device__ __forceinline__ void load8(const float *src, float2 (&f)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float4 v = reinterpret_cast<const float4 *>(src)[h];
    f[2 * h] = make_float2(v.x, v.y);
    f[2 * h + 1] = make_float2(v.z, v.w);
  }
}

// LANES lanes hold one head (groups of eight behind head_dim hold zeros). TAIL: some of a head does not
// turn (its own instance, because the care that an infinity needs there costs a head that turns as a whole
// 38.9 us instead of 36.4 for 8191 tokens).
template <int LANES, bool INTERLEAVED, bool TAIL>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm)
    qk_norm_rope_kernel(const NormRopeParams p) {
  constexpr int kGroups = 32 / LANES;  // heads of a pass
  constexpr int kDim = LANES * 16;     // head_dim is at most this
  __shared__ float s_w[2][kDim];
  // A of the queries, B, A of the keys, B of this warp's token.
  __shared__ __align__(16) float s_tab[kWarps][2][2][kDim];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < 2 * kDim; i += kWarps * 32) {
    const int j = i / kDim, e = i % kDim;
    const float w = p.heads[j] > 0 && e < p.head_dim ? __half2float(p.w[j][e]) : 0.0f;
    s_w[j][e] = w;
    if (e >= 2 * p.half_rot)  // behind the rotation: the weight alone, for every token
      for (int x = 0; x < kWarps; ++x) {
        s_tab[x][j][0][e] = w;
        s_tab[x][j][1][e] = 0.0f;
      }
  }
  __syncthreads();

  const int sub = lane % LANES;
  // This lane's two groups of eight: elements oa.. and ob.. .
  int oa = 16 * sub;  // (behind the rotation: 2 half_rot + 16 (sub - half_rot / 8))
  int ob = oa + 8;
  if (!INTERLEAVED && 8 * sub < p.half_rot) {
    oa = 8 * sub;
    ob = p.half_rot + 8 * sub;
  }
  const bool live_a = oa < p.head_dim, live_b = ob < p.head_dim;
  const bool turns = 8 * sub < p.half_rot;  // both groups or neither
  const int gw = blockIdx.x * kWarps + warp, warps = gridDim.x * kWarps;
  const int part = gw % p.parts;
  const int all = p.passes[0] + p.passes[1];
  const int p0 = static_cast<int>(static_cast<long long>(all) * part / p.parts);
  const int p1 = static_cast<int>(static_cast<long long>(all) * (part + 1) / p.parts);

  // Heads [begin, end) of each side are this warp's; its lane groups take them in turn.
  const int group = lane / LANES;
  const int bq = min(p0, p.passes[0]) * kGroups, eq = min(p.heads[0], p1 * kGroups);
  const int bk = max(p0 - p.passes[0], 0) * kGroups;
  const int ek = min(p.heads[1], (p1 - p.passes[0]) * kGroups);
  const int step = kGroups * p.head_dim;
  // Offsets inside a token's row: heads of a token stay below 2^28 halves.
  const int cq = (bq + group) * p.head_dim, ck = (bk + group) * p.head_dim;

  auto load = [&](const __half *x, bool on, uint4 &a, uint4 &b) {
    a = b = make_uint4(0u, 0u, 0u, 0u);
    if (on && live_a) a = *reinterpret_cast<const uint4 *>(x + oa);
    if (on && live_b) b = *reinterpret_cast<const uint4 *>(x + ob);
  };
  // The heads of one side, the first two passes of which are in (a0, b0) and (a1, b1).
  auto walk = [&](int side, const __half *x, __half *y, int begin, int end, uint4 a0, uint4 b0,
                  uint4 a1, uint4 b1) {
    float2 Aa[4], Ba[4], Ab[4], Bb[4];
    load8(&s_tab[warp][side][0][oa], Aa);
    load8(&s_tab[warp][side][1][oa], Ba);
    load8(&s_tab[warp][side][0][ob], Ab);
    load8(&s_tab[warp][side][1][ob], Bb);
    x += 2 * step;
#pragma unroll 1
    for (int left = end - begin - group; left + group > 0; left -= kGroups) {
      const uint4 ra = a0, rb = b0;
      a0 = a1;
      b0 = b1;
      load(x, left > 2 * kGroups, a1, b1);
      x += step;
      float2 xa[4], xb[4];
      unpack8(ra, xa);
      unpack8(rb, xb);
      float2 sa = __fmul2_rn(xa[0], xa[0]), sb = __fmul2_rn(xb[0], xb[0]);
#pragma unroll
      for (int e = 1; e < 4; ++e) {
        sa = __ffma2_rn(xa[e], xa[e], sa);
        sb = __ffma2_rn(xb[e], xb[e], sb);
      }
      sa = __fadd2_rn(sa, sb);
      float sq = sa.x + sa.y;
#pragma unroll
      for (int m = LANES / 2; m > 0; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m, LANES);
      const float r1 = rsqrtf(fmaf(sq, p.inv_dim, p.eps));
      const float2 r = make_float2(r1, r1);
      float2 ya[4], yb[4];  // partners
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ya[e] = INTERLEAVED ? make_float2(xa[e].y, xa[e].x) : xb[e];
        yb[e] = INTERLEAVED ? make_float2(xb[e].y, xb[e].x) : xa[e];
      }
      // B is 0 behind the rotation, but an infinity times 0 is no 0: there an infinite head (the only one
      // that r is 0 for) has no partners. Its finite elements are x * 0 * w.
      if (TAIL && r1 == 0.0f && !turns) {
#pragma unroll
        for (int e = 0; e < 4; ++e) ya[e] = yb[e] = make_float2(0.0f, 0.0f);
      }
      if (left > 0 && live_a) *reinterpret_cast<uint4 *>(y + oa) = turn8(xa, ya, Aa, Ba, r);
      if (left > 0 && live_b) *reinterpret_cast<uint4 *>(y + ob) = turn8(xb, yb, Ab, Bb, r);
      y += step;
    }
  };

#pragma unroll 1
  for (int t = gw / p.parts; t < p.tokens; t += warps / p.parts) {
    const __half *xq = p.x[0] + t * p.xs[0] + cq, *xk = p.x[1] + t * p.xs[1] + ck;
    uint4 a0, b0, a1, b1;
    load(xq, bq + group < eq, a0, b0);
    load(xq + step, bq + kGroups + group < eq, a1, b1);
    __syncwarp();  // the tables of the token before have been read
    for (int pair = lane; pair < p.half_rot; pair += 32) {
      const int axis = p.axis_of ? min(static_cast<int>(p.axis_of[pair]), p.axes - 1) : 0;
      const int pos = p.positions[static_cast<long long>(axis) * p.tokens + t];
      // angle / pi, reduced to [-1, 1] in fp64.
      const double half_turns = static_cast<double>(pos) *
                                static_cast<double>(p.inv_freq[pair]) * 0.31830988618379067154;
      const double r = half_turns - 2.0 * rint(half_turns * 0.5);
      float s, c;
      sincospif(static_cast<float>(r), &s, &c);
      const int e1 = INTERLEAVED ? 2 * pair : pair;
      const int e2 = INTERLEAVED ? 2 * pair + 1 : pair + p.half_rot;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float w1 = s_w[j][e1], w2 = s_w[j][e2];
        s_tab[warp][j][0][e1] = w1 * c;
        s_tab[warp][j][0][e2] = w2 * c;
        s_tab[warp][j][1][e1] = -w2 * s;
        s_tab[warp][j][1][e2] = w1 * s;
      }
    }
    __syncwarp();
    if (eq > bq) walk(0, xq, p.y[0] + t * p.ys[0] + cq, bq, eq, a0, b0, a1, b1);
    if (ek > bk) {
      load(xk, bk + group < ek, a0, b0);
      load(xk + step, bk + kGroups + group < ek, a1, b1);
      walk(1, xk, p.y[1] + t * p.ys[1] + ck, bk, ek, a0, b0, a1, b1);
    }
  }
}

template <int LANES>
void launch(const NormRopeParams &p, bool interleaved, unsigned grid, cudaStream_t stream) {
  const bool tail = 2 * p.half_rot < p.head_dim;
  const auto kernel = interleaved ? tail ? qk_norm_rope_kernel<LANES, true, true> : qk_norm_rope_kernel<LANES, true, false>
                      : tail      ? qk_norm_rope_kernel<LANES, false, true>
                                  : qk_norm_rope_kernel<LANES, false, false>;
  kernel<<<grid, kWarps * 32, 0, stream>>>(p);
}

int check(const hgemm_qk_norm_rope_t *a) {
  if (!a || a->tokens < 0 || a->heads_q < 0 || a->heads_kv < 0) return HGEMM_ERR_INVALID_ARG;
  if (a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8 != 0) return HGEMM_ERR_INVALID_ARG;
  if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 16 != 0)
    return HGEMM_ERR_INVALID_ARG;
  if (a->axes < 1 || (a->axes > 1 && a->rot_dim > 0 && !a->axis_of)) return HGEMM_ERR_INVALID_ARG;
  if (!(a->eps >= 0.0f)) return HGEMM_ERR_INVALID_ARG;
  if (a->heads_q > kMaxHeads || a->heads_kv > kMaxHeads || a->tokens > kOpMaxRows)
    return HGEMM_ERR_TOO_LARGE;
  if (a->tokens == 0 || a->heads_q + a->heads_kv == 0) return HGEMM_OK;
  if (a->rot_dim > 0 && (!a->positions || !a->inv_freq)) return HGEMM_ERR_INVALID_ARG;
  auto operand = [&](const void *in, const void *out, const void *w, long long is, long long os,
                     int heads) {
    if (heads == 0) return true;
    const long long row = static_cast<long long>(heads) * a->head_dim;
    return in && out && w && op_aligned16(in) && op_aligned16(out) && op_aligned16(w) &&
           is % 8 == 0 && os % 8 == 0 && is >= row && os >= row && is <= kOpMaxStride && os <= kOpMaxStride && (in != out || is == os);
  };
  if (!operand(a->q, a->q_out, a->q_weight, a->q_stride, a->q_out_stride, a->heads_q) ||
      !operand(a->k, a->k_out, a->k_weight, a->k_stride, a->k_out_stride, a->heads_kv))
    return HGEMM_ERR_INVALID_ARG;
  const OpRows in[] = {op_heads(a->q, a->heads_q, a->head_dim, a->q_stride, a->tokens),
                       op_heads(a->k, a->heads_kv, a->head_dim, a->k_stride, a->tokens),
                       op_dense(a->q_weight, 2, a->heads_q ? a->head_dim : 0),
                       op_dense(a->k_weight, 2, a->heads_kv ? a->head_dim : 0),
                       op_dense(a->positions, 4, a->rot_dim ? a->axes : 0, a->tokens),
                       op_dense(a->inv_freq, 4, a->rot_dim / 2),
                       op_dense(a->axis_of, 1, a->axes > 1 ? a->rot_dim / 2 : 0)};
  const OpRows out[] = {op_heads(a->q_out, a->heads_q, a->head_dim, a->q_out_stride, a->tokens),
                        op_heads(a->k_out, a->heads_kv, a->head_dim, a->k_out_stride, a->tokens)};
  bool over = op_overlap(out[0], out[1]);
  for (int o = 0; o < 2; ++o)
    for (int i = 0; i < 7; ++i)
      over |= !(i == o && out[o].at == in[i].at) && op_overlap(out[o], in[i]);  // in place, or apart
  return over ? HGEMM_ERR_INVALID_ARG : HGEMM_OK;
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
  p.positions = a->positions;
  p.axis_of = a->axes > 1 ? a->axis_of : nullptr;
  p.inv_freq = a->inv_freq;
  p.tokens = a->tokens;
  p.heads[0] = a->heads_q;
  p.heads[1] = a->heads_kv;
  p.head_dim = a->head_dim;
  p.half_rot = a->rot_dim / 2;
  p.axes = a->axes;
  p.eps = a->eps;
  p.inv_dim = 1.0f / static_cast<float>(a->head_dim);
  const int lanes = a->head_dim <= 64 ? 4 : a->head_dim <= 128 ? 8 : 16;
  const int groups = 32 / lanes;
  p.passes[0] = (a->heads_q + groups - 1) / groups;
  p.passes[1] = (a->heads_kv + groups - 1) / groups;
  // A warp to a token where there are enough tokens for the warps that fit; otherwise a token's passes
  // are shared by as many warps as that leaves, down to a single pass each.
  const int warps = kWarps * kCtasPerSm * d.sm_count;
  p.parts = std::max(1, std::min(p.passes[0] + p.passes[1], warps / a->tokens));
  const long long need = (static_cast<long long>(a->tokens) * p.parts + kWarps - 1) / kWarps;
  const long long grid = std::min<long long>(need, kCtasPerSm * d.sm_count);  // (need, with parts)
  const bool il = a->interleaved != 0;
  if (lanes == 4)
    launch<4>(p, il, static_cast<unsigned>(grid), stream);
  else if (lanes == 8)
    launch<8>(p, il, static_cast<unsigned>(grid), stream);
  else
    launch<16>(p, il, static_cast<unsigned>(grid), stream);
  return cudaGetLastError() == cudaSuccess ? HGEMM_OK : HGEMM_ERR_LAUNCH;
}

}  // namespace
}  // namespace hgemm

extern "C" int hgemm_qk_norm_rope(const hgemm_qk_norm_rope_t *args, hgemm_stream_t stream) {
  return hgemm::op_status(hgemm::run(args, stream));
}
