// Norms of queries and keys for each head, with the position rotation in the same pass.
//
//   n = x * rsqrt(mean(x^2) + eps) * w;   (n1, n2) -> (n1 cos a - n2 sin a, n2 cos a + n1 sin a)
//
// Bound: HBM. Every half is read once and written once (4 bytes of traffic an element), against
// about ten fp32 operations. Loads through registers held too few bytes in flight (two heads to a
// lane group: 37 us for 8191 tokens of 40 heads of 128), so the heads of a token, which are adjacent,
// come by bulk copies into a ring of slots, issued by a warp of their own; the other warps pass
// over the slots each at its own pace, and results leave with 16-byte stores. A CTA takes a range of
// tokens, all CTAs the same number to within one.
// A head then lives in the registers of few lanes, 16 halves each: eight consecutive ones and the
// eight that they turn with (half a rotation away, or next to them when pairs are adjacent), so that the
// rotation needs no other lane and the mean square is the only exchange.
// The angles of a token serve all of its heads: one lane for each pair forms position * inv_freq in
// fp64 (exact: 31 + 24 bits), reduces it to a turn there and takes sincospi in fp32. The copying warp
// does that while the copies are under way, so that a slot is full with its angles and the other
// warps never meet (formed by all of them behind a barrier, they cost 10 us of the 38).
//
// No counterpart in the reference.

#include <algorithm>

#include "ops_sm100.cuh"

namespace hgemm {
namespace {

constexpr int kThreads = 256;  // that pass over the heads; one more warp fills the slots
constexpr int kCtasPerSm = 4;
constexpr int kSlots = 4;
constexpr int kMaxHalfRot = 128;
constexpr int kMaxSlotBytes = 10752;  // kCtasPerSm rings fit an SM
constexpr int kMaxHeads = 1 << 20;

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
  // A CTA takes `part_heads` adjacent heads (queries, then keys) of each of its tokens.
  int part_heads, parts, slot_bytes;
  unsigned *status_word;
  unsigned long long timeout_ns;
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

__device__ __forceinline__ void load8(const float *src, float (&f)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float4 v = reinterpret_cast<const float4 *>(src)[h];
    f[4 * h] = v.x;
    f[4 * h + 1] = v.y;
    f[4 * h + 2] = v.z;
    f[4 * h + 3] = v.w;
  }
}

// LANES lanes hold one head (groups of eight behind head_dim hold zeros).
template <int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads + 32, kCtasPerSm)
    qk_norm_rope_kernel(const NormRopeParams p) {
  constexpr int kGroups = kThreads / LANES;  // heads in flight in this CTA
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(16) float s_cos[kSlots][kMaxHalfRot];
  __shared__ __align__(16) float s_sin[kSlots][kMaxHalfRot];
  __shared__ __align__(16) float s_w[2][256];
  __shared__ __align__(8) uint64_t s_full[kSlots], s_empty[kSlots];
  __shared__ int s_abort;

  const int part = blockIdx.x % p.parts, cta = blockIdx.x / p.parts, ctas = gridDim.x / p.parts;
  const int t0 = static_cast<int>(static_cast<long long>(p.tokens) * cta / ctas);
  const int t1 = static_cast<int>(static_cast<long long>(p.tokens) * (cta + 1) / ctas);
  const int h0 = part * p.part_heads, n = min(p.part_heads, p.heads - h0);
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < kSlots; ++i) {
      ptx::mbar_init(ptx::smem_u32(&s_full[i]), 2);  // the copies; the angles
      ptx::mbar_init(ptx::smem_u32(&s_empty[i]), kThreads / 32);
    }
    ptx::fence_mbar_init_cluster();
  }
  for (int i = threadIdx.x; i < 2 * 256; i += kThreads + 32) {
    const int j = i >> 8, e = i & 255;
    s_w[j][e] = p.w[j] && e < p.head_dim ? __half2float(p.w[j][e]) : 0.0f;
  }
  __syncthreads();
  const OpWait wc{&s_abort, p.status_word, p.timeout_ns};
  const int lane = threadIdx.x & 31;

  if (threadIdx.x >= kThreads) {
    // ---------------------------------------------------------------- copies and angles
    // This part's queries, its keys, or some of both.
    const int split = min(max(p.heads_q, h0), h0 + n);
    const int qbytes = (split - h0) * p.head_dim * 2, kbytes = (h0 + n - split) * p.head_dim * 2;
    const __half *q = p.x[0] + t0 * p.xs[0] + static_cast<long long>(h0) * p.head_dim;
    const __half *k = p.x[1] + t0 * p.xs[1] + static_cast<long long>(split - p.heads_q) * p.head_dim;
    constexpr int kPairs = kMaxHalfRot / 32;  // of a lane: lane, lane + 32, ..
    const int *place[kPairs];                 // positions of the pair's axis
    double freq[kPairs];                      // inv_freq / pi
    int pos[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int pair = lane + 32 * j;
      if (pair >= p.half_rot) continue;
      const int axis = p.axis_of ? min(static_cast<int>(p.axis_of[pair]), p.axes - 1) : 0;
      place[j] = p.positions + static_cast<long long>(axis) * p.tokens + t0;
      freq[j] = static_cast<double>(p.inv_freq[pair]);
      pos[j] = place[j][0];
    }
    int i = 0;
    bool ok = true;
    for (; i < t1 - t0; ++i) {
      const int slot = i % kSlots;
      const uint32_t bar = ptx::smem_u32(&s_full[slot]);
      int okw = 1;
      if (lane == 0) {
        if (i >= kSlots)
          okw = op_wait(ptx::smem_u32(&s_empty[slot]), (i / kSlots - 1) & 1, wc, kSiteNormEmpty);
        if (okw) {
          const uint32_t dst = ptx::smem_u32(ring) + slot * p.slot_bytes;
          ptx::mbar_arrive_expect_tx(bar, qbytes + kbytes);
          if (qbytes) ptx::bulk_load(dst, q + i * p.xs[0], qbytes, bar);
          if (kbytes) ptx::bulk_load(dst + qbytes, k + i * p.xs[1], kbytes, bar);
        }
      }
      ok = __shfl_sync(0xffffffffu, okw, 0) != 0;
      if (!ok) break;
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int pair = lane + 32 * j;
        if (pair >= p.half_rot) continue;
        // angle / pi, reduced to [-1, 1] in fp64.
        const double half_turns = static_cast<double>(pos[j]) * freq[j] * 0.31830988618379067154;
        if (i + 1 < t1 - t0) pos[j] = place[j][i + 1];
        const double r = half_turns - 2.0 * rint(half_turns * 0.5);
        float s, c;
        sincospif(static_cast<float>(r), &s, &c);
        s_cos[slot][pair] = c;
        s_sin[slot][pair] = s;
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar);
    }
    if (!ok && lane == 0)  // unwinding: the copies in flight land before the CTA may exit
      for (int j = max(0, i - kSlots); j < i; ++j)
        op_drain(ptx::smem_u32(&s_full[j % kSlots]), (j / kSlots) & 1);
    return;
  }

  // ------------------------------------------------------------------ norms and rotation
  const int sub = threadIdx.x % LANES;
  // This lane's two groups of eight: elements oa.. and ob.. .
  const bool turns = (INTERLEAVED ? 16 : 8) * sub < (INTERLEAVED ? 2 : 1) * p.half_rot;
  int oa = 16 * sub;  // (behind the rotation: 2 half_rot + 16 (sub - half_rot / 8))
  int ob = oa + 8;
  if (!INTERLEAVED && turns) {
    oa = 8 * sub;
    ob = p.half_rot + 8 * sub;
  }
  const bool live_a = oa < p.head_dim, live_b = ob < p.head_dim;

#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
    const int k = t - t0, slot = k % kSlots;
    // (a wait that ran out leaves the slot's contents unspecified; the status word tells)
    op_wait(ptx::smem_u32(&s_full[slot]), (k / kSlots) & 1, wc, kSiteNormFull);
    const __half *stage = reinterpret_cast<const __half *>(ring + slot * p.slot_bytes);
    // Whole warps, so that every lane takes part in the exchange.
#pragma unroll 1
    for (int i = static_cast<int>(threadIdx.x) / LANES; i - lane / LANES < n; i += kGroups) {
      const bool on = i < n;
      uint4 ra = make_uint4(0u, 0u, 0u, 0u), rb = ra;
      if (on && live_a) ra = *reinterpret_cast<const uint4 *>(stage + i * p.head_dim + oa);
      if (on && live_b) rb = *reinterpret_cast<const uint4 *>(stage + i * p.head_dim + ob);
      float xa[8], xb[8];
      unpack8(ra, xa);
      unpack8(rb, xb);
      float sa = 0.0f, sb = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sa = fmaf(xa[e], xa[e], sa);
        sb = fmaf(xb[e], xb[e], sb);
      }
      float sq = sa + sb;
#pragma unroll
      for (int m = LANES / 2; m > 0; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m, LANES);
      if (!on) continue;
      const int head = h0 + i, side = head >= p.heads_q;
      const float r = rsqrtf(fmaf(sq, p.inv_dim, p.eps));
      float wa[8], wb[8];
      load8(&s_w[side][oa], wa);
      load8(&s_w[side][ob], wb);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xa[e] *= wa[e] * r;
        xb[e] *= wb[e] * r;
      }
      if (turns) {
        float c[8], s[8];
        load8(&s_cos[slot][8 * sub], c);
        load8(&s_sin[slot][8 * sub], s);
        if (INTERLEAVED) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a0 = xa[2 * e], b0 = xb[2 * e];
            xa[2 * e] = fmaf(a0, c[e], -xa[2 * e + 1] * s[e]);
            xa[2 * e + 1] = fmaf(xa[2 * e + 1], c[e], a0 * s[e]);
            xb[2 * e] = fmaf(b0, c[4 + e], -xb[2 * e + 1] * s[4 + e]);
            xb[2 * e + 1] = fmaf(xb[2 * e + 1], c[4 + e], b0 * s[4 + e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a0 = xa[e];
            xa[e] = fmaf(a0, c[e], -xb[e] * s[e]);
            xb[e] = fmaf(xb[e], c[e], a0 * s[e]);
          }
        }
      }
      __half *y = (side ? p.y[1] + t * p.ys[1] : p.y[0] + t * p.ys[0]) +
                  static_cast<long long>(head - (side ? p.heads_q : 0)) * p.head_dim;
      if (live_a) *reinterpret_cast<uint4 *>(y + oa) = pack8(xa);
      if (live_b) *reinterpret_cast<uint4 *>(y + ob) = pack8(xb);
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s_empty[slot]));
  }
}

template <int LANES>
int launch(const NormRopeParams &p, bool interleaved, unsigned grid, int dev, cudaStream_t stream) {
  const auto kernel =
      interleaved ? qk_norm_rope_kernel<LANES, true> : qk_norm_rope_kernel<LANES, false>;
  static bool done[2][64];
  const int st = op_smem(reinterpret_cast<const void *>(kernel), kSlots * kMaxSlotBytes, dev,
                         done[interleaved]);
  if (st != HGEMM_OK) return st;
  kernel<<<grid, kThreads + 32, kSlots * p.slot_bytes, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? HGEMM_OK : HGEMM_ERR_LAUNCH;
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
  p.w[0] = a->heads_q ? a->q_weight : nullptr;
  p.w[1] = a->heads_kv ? a->k_weight : nullptr;
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
  p.status_word = d.status_word;
  p.timeout_ns = d.timeout_ns;
  const int lanes = a->head_dim <= 64 ? 4 : a->head_dim <= 128 ? 8 : 16;
  const int slots = kCtasPerSm * d.sm_count;
  // All heads of a token in one CTA as far as a slot holds them; with fewer tokens than CTAs, one
  // head to a lane group, so that a token's heads are spread over CTAs.
  p.part_heads = std::min(p.heads, kMaxSlotBytes / (2 * a->head_dim));
  if (a->tokens < slots) p.part_heads = std::min(p.part_heads, kThreads / lanes);
  p.parts = (p.heads + p.part_heads - 1) / p.part_heads;
  p.slot_bytes = (p.part_heads * a->head_dim * 2 + 127) / 128 * 128;
  const unsigned grid =
      static_cast<unsigned>(std::min(a->tokens, std::max(1, slots / p.parts)) * p.parts);
  const bool il = a->interleaved != 0;
  return lanes == 4   ? launch<4>(p, il, grid, d.dev, stream)
         : lanes == 8 ? launch<8>(p, il, grid, d.dev, stream)
                      : launch<16>(p, il, grid, d.dev, stream);
}

}  // namespace
}  // namespace hgemm

extern "C" int hgemm_qk_norm_rope(const hgemm_qk_norm_rope_t *args, hgemm_stream_t stream) {
  return hgemm::op_status(hgemm::run(args, stream));
}
