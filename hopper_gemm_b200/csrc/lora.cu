// A shared projection with the low-rank adapters of many requests beside it:
//   Y[t,:] = X[t,:] W + scale[a] * (X[t,:] Down[a]) Up[a],  a the adapter of token t's segment.
//
// Many tokens: two launches (and one that returns at once). lora_shrink_kernel forms H = scale (X Down):
// one tcgen05 product for every (row tile, adapter in it), K split over a cluster, and leaves H as
// operand blocks of the second product: for every adapter of a row tile a block of 64-column rows in
// which the rows of other adapters are zero. The projection's own GEMM kernel (hgemm_sm100.cu) then
// walks those blocks as additional k-blocks behind the k-blocks of X and W, so that Up's product
// lands in the same fp32 accumulators and Y is written and rounded once; an adapter costs its row
// tiles rank / K of the GEMM. H is rounded to binary16 because it is a tcgen05 operand next to Up (the path of few
// tokens keeps it in fp32).
//
// Few tokens (decoding, short batches; few_plan says when): bound by the bytes of W and of the adapters in
// use. W is the M operand of the product, 128 of its columns to a CTA, and the tokens are its N; K is split
// over a cluster, so that every SM pulls weights, and joined through distributed shared memory. The adapters run on the CUDA
// cores in fp32, H in a launch of its own under whose feet the main kernel already starts, and Up's part
// in warps that would otherwise wait for the main loop.
//
// Measured (one B200, eager calls over changing inputs): 1 token x 4096 x 4096, rank 16: 12.3 us, of which W's 33.6 MB
// are 5.2; 48 tokens of as many requests x 4096 x 6144, rank 32: 24.6 us (H 7.5, under which W streams; then every
// token's rows of Up from L2). 1037 tokens x 4096 x 4096 of many adapters: 58 us, the GEMM alone 33.9 and H 20,
// part of it hidden: both take whole SMs' shared memory. 8192 tokens x 4096 x 6144: 381 us (323 in a replayed
// graph), the GEMM alone 291 to 333, H 29: bound by the products and the power limit.
//
// No counterpart in the reference.

#include <algorithm>
#include <cmath>

#include "ops_sm100.cuh"

namespace hgemm {
namespace {

constexpr int kMaxRank = 256;
constexpr int kSms = 148;          // what plans (and with them workspaces) reckon with
constexpr int kTileRows = 128;     // rows of a shrink CTA
constexpr int kMaxTileRows = 256;  // rows of a GEMM tile
constexpr int kSegCache = 1024;    // segment starts kept in shared memory
constexpr int kAdapterCache = 1024;  // adapters whose first row in a tile is kept there
constexpr int kStages = 4;
constexpr int kBlocks = 4;         // 64-column blocks of Down in a stage
constexpr int kABytes = kTileRows * 128;
constexpr int kBBytes = 64 * 128;
constexpr int kStageBytes = kABytes + kBlocks * kBBytes;
constexpr int kSmem = 1024 + kStages * kStageBytes + 256;
constexpr int kPartStride = kBlocks * 64 + 4;  // floats of a partial row, padded for the banks
static_assert(kTileRows * kPartStride * 4 <= kStages * kStageBytes, "partials reuse the stages");
// Warps of a shrink CTA: X's loads, issue, four that join, and one for each 64-column block of Down. A
// thread is held about 400 cycles by a TMA load whatever its size, so every box of a stage has a
// warp of its own (one warp for all five boxes: 30 us for 8192 tokens).
constexpr int kThreads = 32 * (6 + kBlocks);

struct LoraParams {
  const __half *X, *W, *down, *up;
  __half *Y;
  const float *scale;
  const int *seg_start, *seg_adapter;
  int tokens, N, K, rank, adapters, segments;
  int tile_rows, chunks;    // rows of a GEMM tile; 64-column blocks of H
  int groups, per_group;    // adapters of a tile are taken `per_group` at a time by `groups` CTAs
  int ksplit, num_kb;
  int entries, per_tile;    // of all tiles; of each, or 0: as its segments say
  int *base, *count, *adapter;
  __half *low;
  unsigned *odd_count;
  unsigned long long *odd_list;
  unsigned *status_word;
  unsigned long long timeout_ns;
};

// Segments that start at or before token t (binary search; any contents stay in bounds).
__device__ __forceinline__ int starts_upto(const int *seg_start, int segments, int t) {
  int lo = 0, hi = segments;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (seg_start[mid] <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// Adapter of token t, or -1.
__device__ __forceinline__ int token_adapter(const int *seg_start, const int *seg_adapter,
                                             int segments, int adapters, int t) {
  const int s = starts_upto(seg_start, segments, t) - 1;
  if (s < 0 || t >= seg_start[s + 1]) return -1;
  const int a = seg_adapter[s];
  return (a >= 0 && a < adapters) ? a : -1;
}

__global__ void __launch_bounds__(kThreads, 1)
    lora_shrink_kernel(const __grid_constant__ CUtensorMap tmX,
                       const __grid_constant__ CUtensorMap tmDown, const LoraParams p) {
  ptx::grid_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_seg[kSegCache];
  __shared__ int s_first[kAdapterCache];
  __shared__ int s_adapter[kMaxTileRows];
  __shared__ int s_list[kMaxTileRows];
  __shared__ unsigned s_mask[kMaxTileRows / 32];
  __shared__ int s_base;
  __shared__ int s_abort;
  __shared__ uint32_t s_tmem;
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (base - raw);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kStages * kStageBytes);
  const uint32_t full = ptx::smem_u32(bars), empty = full + 8 * kStages, acc = empty + 8 * kStages;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % p.ksplit;
  int idx = blockIdx.x / p.ksplit;
  const int group = idx % p.groups;
  idx /= p.groups;
  const int halves = p.tile_rows / kTileRows;
  const int tile = idx / halves, half = idx % halves;
  const int tile0 = tile * p.tile_rows, row0 = tile0 + half * kTileRows;

  // The adapters of the GEMM tile, in the order of their first row.
  if (warp == 1) {
    ptx::tmem_alloc<1>(ptx::smem_u32(&s_tmem), 256);
    ptx::tmem_relinquish<1>();
  }
  const int *starts = p.seg_start;
  const bool cached = p.adapters <= kAdapterCache;
  if (p.segments < kSegCache) {
    for (int i = threadIdx.x; i <= p.segments; i += kThreads) s_seg[i] = p.seg_start[i];
    starts = s_seg;
  }
  if (cached)
    for (int i = threadIdx.x; i < p.adapters; i += kThreads) s_first[i] = kMaxTileRows;
  const int kb0 = static_cast<int>(static_cast<long long>(p.num_kb) * split / p.ksplit);
  const int kb1 = static_cast<int>(static_cast<long long>(p.num_kb) * (split + 1) / p.ksplit);
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(full + 8 * i, 2);  // X; the blocks of Down
      ptx::mbar_init(empty + 8 * i, 1);
    }
    ptx::mbar_init(acc, 1);
    ptx::fence_mbar_init_cluster();
  }
  __syncthreads();
  // X's first stages are asked for before the adapters are known, by the CTAs that any adapter makes use of.
  const int early = group == 0 && row0 < p.tokens ? min(kStages, kb1 - kb0) : 0;
  if (threadIdx.x == 0)
    for (int it = 0; it < early; ++it) {
      ptx::mbar_arrive_expect_tx(full + 8 * it, kABytes);
      ptx::tma_load_2d(&tmX, base + it * kStageBytes, full + 8 * it, (kb0 + it) * 64, row0);
    }
  __syncwarp();
  for (int i = threadIdx.x; i < p.tile_rows; i += kThreads)
    s_adapter[i] = tile0 + i < p.tokens
                       ? token_adapter(starts, p.seg_adapter, p.segments, p.adapters, tile0 + i)
                       : -1;
  if (threadIdx.x == 0) {
    // Tiles before this one have at most one entry each more than the segments that begin in them.
    s_base = p.per_tile ? tile * p.per_tile : tile + starts_upto(starts, p.segments, tile0 - 1);
  }
  __syncthreads();
  if (cached) {
    for (int i = threadIdx.x; i < p.tile_rows; i += kThreads)
      if (s_adapter[i] >= 0) atomicMin(&s_first[s_adapter[i]], i);
    __syncthreads();
  }
  for (int i0 = warp * 32; i0 < p.tile_rows; i0 += kThreads) {
    const int i = i0 + lane, a = s_adapter[i];
    bool first = a >= 0 && (i == 0 || s_adapter[i - 1] != a);
    if (cached)
      first = first && s_first[a] == i;
    else
      for (int j = 0; first && j < i; ++j) first = s_adapter[j] != a;
    const unsigned m = __ballot_sync(0xffffffffu, first);
    if (lane == 0) s_mask[i0 / 32] = m;
  }
  __syncthreads();
  int n = 0;
  for (int x = 0; x < p.tile_rows / 32; ++x) {
    const unsigned m = s_mask[x];
    if (warp == 0 && ((m >> lane) & 1u))
      s_list[n + __popc(m & ((1u << lane) - 1u))] = s_adapter[32 * x + lane];
    n += __popc(m);
  }
  const int entry0 = min(s_base, p.entries - 1);
  n = min(n, p.entries - entry0);  // (only starts that are not ascending get here with more)
  ptx::tc_fence_before();
  __syncthreads();
  if (half == 0 && split == 0) {
    if (group == 0 && threadIdx.x == 0) {
      p.base[tile] = entry0;
      p.count[tile] = n;
      if (tile == 0) *p.odd_count = 0;
    }
    for (int u = group * p.per_group + threadIdx.x; u < min(n, (group + 1) * p.per_group); u += kThreads)
      p.adapter[entry0 + u] = s_list[u];
  }
  const int u0 = group * p.per_group;
  const int nu = min(n - u0, p.per_group);
  // The same for every CTA of the cluster: no adapters left, or no rows (their products are never
  // stored).
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&s_tmem);
  if (nu <= 0 || row0 >= p.tokens) {
    if (warp == 1) ptx::tmem_dealloc<1>(tmem, 256);
    if (threadIdx.x == 0)
      for (int it = 0; it < early; ++it) {  // the loads in flight land before the CTA may exit
        ptx::mbar_arrive(full + 8 * it);
        op_drain(full + 8 * it, 0);
      }
    return;
  }
  ptx::tc_fence_after();
  const OpWait wc{&s_abort, p.status_word, p.timeout_ns};
  const int cols = p.chunks * 64;  // accumulator columns of an adapter
  bool ok = true;

  const int box = warp - 6;  // of Down
  if (warp == 0 || (box >= 0 && box < nu * p.chunks)) {
    if (lane == 0) {
      const int adapter = box >= 0 ? s_list[u0 + box / p.chunks] : 0;
      int it = box < 0 ? early : 0;
      for (int kb = kb0 + it; kb < kb1; ++kb, ++it) {
        const int st = it % kStages;
        if (it >= kStages &&
            !(ok = op_wait(empty + 8 * st, (it / kStages - 1) & 1, wc, kSiteLoraEmpty)))
          break;
        const uint32_t dst = base + st * kStageBytes, bar = full + 8 * st;
        if (box < 0) {
          ptx::mbar_arrive_expect_tx(bar, kABytes);
          ptx::tma_load_2d(&tmX, dst, bar, kb * 64, row0);
        } else {
          // (the first box's warp announces all of them; bytes may be counted before that)
          if (box == 0) ptx::mbar_arrive_expect_tx(bar, nu * p.chunks * kBBytes);
          ptx::tma_load_3d(&tmDown, dst + kABytes + box * kBBytes, bar, 64 * (box % p.chunks), kb * 64,
                           adapter);
        }
      }
      if (!ok && box < 0)
        for (int j = max(0, it - kStages); j < it; ++j)
          op_drain(full + 8 * (j % kStages), (j / kStages) & 1);
    }
  } else if (warp == 1) {
    // One product for all adapters of the group: their blocks of 64 columns lie one behind the other, and
    // so do their accumulators. The whole warp walks the loop and one lane issues, so that descriptors
    // stay in uniform registers (walked by one lane a product took twice its time to issue).
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const int width = __shfl_sync(0xffffffffu, nu * cols, 0);
    const uint32_t idesc = ptx::umma_idesc_f16_f32(kTileRows, width);
    const bool one = ptx::elect_one();
    int it = 0;
    for (int kb = kb0; kb < kb1; ++kb, ++it) {
      const int st = it % kStages;
      if (!__all_sync(0xffffffffu, op_wait(full + 8 * st, (it / kStages) & 1, wc, kSiteLoraFull))) break;
      ptx::tc_fence_after();
      const uint32_t src = base + st * kStageBytes;
      const uint64_t ad = ptx::umma_desc_sw128(src, 16, 1024);
      const uint64_t bd = ptx::umma_desc_sw128(src + kABytes, kBBytes, 1024);
      if (one) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          ptx::umma_f16<1>(tm, ad + 2 * k, bd + 128 * k, idesc, it > 0 || k > 0);
        if (kb + kStages < kb1) ptx::umma_commit<1>(empty + 8 * st);
      }
    }
    if (one) ptx::umma_commit<1>(acc);
    __syncwarp();
  }
  // Partial sums to shared memory (the stages are free once the last product has retired).
  int okw = 1;
  if (lane == 0) okw = op_wait(acc, 0, wc, kSiteLoraAcc);
  ok = __shfl_sync(0xffffffffu, okw, 0) != 0;
  ptx::tc_fence_after();
  float *part = reinterpret_cast<float *>(smem);
  if (warp >= 2 && warp < 6) {
    const int q = warp & 3;
    const uint32_t t = tmem + (static_cast<uint32_t>(q) << 21);
    float *dst = part + (32 * q + lane) * kPartStride;
    for (int c = 0; ok && c < nu * p.chunks * 2; ++c) {
      uint32_t v[32];
      ptx::tmem_ld_32x32b_x32(t + 32 * c, v);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int g = 0; g < 8; ++g)
        *reinterpret_cast<uint4 *>(dst + 32 * c + 4 * g) =
            make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
    }
  }
  ptx::tc_fence_before();
  if (p.ksplit > 1)
    ptx::cluster_sync();
  else
    __syncthreads();
  // Each CTA of the cluster joins its share of the rows, in split order, and writes the operand
  // blocks: 8 halves at a time, zeros for rows of other adapters and columns behind the rank.
  const int rows = kTileRows / p.ksplit, r0 = split * rows;
  const int per_row = nu * p.chunks * 8;
  const uint32_t part_addr = ptx::smem_u32(part);
  for (int x = threadIdx.x; x < rows * per_row; x += kThreads) {
    const int r = r0 + x / per_row, g = x % per_row;
    const int u = g / (p.chunks * 8), cg = g % (p.chunks * 8);
    uint4 out = make_uint4(0u, 0u, 0u, 0u);
    const int a = s_list[u0 + u];
    if (s_adapter[half * kTileRows + r] == a && 8 * cg < p.rank) {
      float f[8] = {};
      const uint32_t off = part_addr + (r * kPartStride + u * cols + 8 * cg) * 4;
      for (int k = 0; k < p.ksplit; ++k) {
        const uint32_t src = k == split ? off : ptx::mapa(off, k);
        const float4 v = k == split ? ptx::ld_shared_v4f(src) : ptx::ld_shared_cluster_v4f(src);
        const float4 w =
            k == split ? ptx::ld_shared_v4f(src + 16) : ptx::ld_shared_cluster_v4f(src + 16);
        f[0] += v.x;
        f[1] += v.y;
        f[2] += v.z;
        f[3] += v.w;
        f[4] += w.x;
        f[5] += w.y;
        f[6] += w.z;
        f[7] += w.w;
      }
      const float sc = p.scale[a];
      uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __half2 v = __floats2half2_rn(f[2 * e] * sc, f[2 * e + 1] * sc);
        h[e] = *reinterpret_cast<const uint32_t *>(&v);
      }
      out = make_uint4(h[0], h[1], h[2], h[3]);
    }
    const long long block = static_cast<long long>(entry0 + u0 + u) * p.chunks + (cg >> 3);
    *reinterpret_cast<uint4 *>(p.low + (block * p.tile_rows + half * kTileRows + r) * 64 +
                               (cg & 7) * 8) = out;
  }
  if (p.ksplit > 1)
    ptx::cluster_sync();  // nobody reads this CTA's partials any more
  else
    __syncthreads();
  if (warp == 1) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, 256);
  }
}

// Blocks of Y (32 x 64) that left the GEMM with an infinity or NaN. Most of what is not finite there is right: it
// comes of the token's own X, of W or of its own adapter. Only where another adapter of the row tile has an
// infinity or NaN in a column of Up has that column met the zeros that stand for the token's row of H, and is formed
// again from what it depends on alone. So Up's columns are looked at first, rank rows of 128 bytes for each
// adapter of the tile (600 of 1200 tokens NaN, 4096 x 4096: 42 ms when every element was formed again, 0.08
// now, 0.07 with finite ones), and a block is formed again by a CTA, eight rows to a thread, with X's rows in
// shared memory and W read in whole rows. With nothing listed this returns at once.
constexpr int kRepairThreads = 256;
constexpr int kRepairK = 64;  // of X at a time
__global__ void __launch_bounds__(kRepairThreads, 2) lora_repair_kernel(const LoraParams p) {
  __shared__ int s_least[64], s_most[64];  // adapters with an infinity or NaN in a column of Up
  __shared__ int s_own[32], s_entry[32];   // a row's adapter, and its place among the tile's
  __shared__ float s_x[32][kRepairK];
  const unsigned n = *p.odd_count;
  for (unsigned b = blockIdx.x; b < n; b += gridDim.x) {
    const unsigned long long block = p.odd_list[b];
    const int t0 = static_cast<int>(block & 0xffffffffu), c0 = static_cast<int>(block >> 32);
    const int base = p.base[t0 / p.tile_rows], count = p.count[t0 / p.tile_rows];
    __syncthreads();  // the block before is through with the tables
    if (threadIdx.x < 64) {
      s_least[threadIdx.x] = p.adapters;
      s_most[threadIdx.x] = -1;
    }
    __syncthreads();
    bool found = false;
    const int g = 8 * (threadIdx.x & 7);
    for (int u = 0; c0 + g < p.N && u < count; ++u) {
      const int a = p.adapter[base + u];
      for (int r = threadIdx.x >> 3; r < p.rank; r += kRepairThreads / 8) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(
            p.up + (static_cast<long long>(a) * p.rank + r) * p.N + c0 + g));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (((w[e >> 1] >> (16 * (e & 1))) & 0x7c00u) == 0x7c00u) {
            found = true;
            atomicMin(&s_least[g + e], a);
            atomicMax(&s_most[g + e], a);
          }
      }
    }
    if (!__syncthreads_or(found)) continue;
    if (threadIdx.x < 32) {
      const int t = t0 + threadIdx.x;
      const int a = t < p.tokens
                        ? token_adapter(p.seg_start, p.seg_adapter, p.segments, p.adapters, t)
                        : -1;
      int entry = -1;
      for (int u = 0; a >= 0 && u < count; ++u)
        if (p.adapter[base + u] == a) entry = base + u;
      s_own[threadIdx.x] = a;
      s_entry[threadIdx.x] = entry;
    }
    __syncthreads();
    const int col = threadIdx.x & 63, row = threadIdx.x / 64 * 8, c = c0 + col;
    unsigned todo = 0;  // of this thread's eight rows
    if (c < p.N && s_most[col] >= 0)
      for (int i = 0; i < 8; ++i) {
        const int own = s_own[row + i];
        if (t0 + row + i < p.tokens && (s_least[col] != own || s_most[col] != own)) todo |= 1u << i;
      }
    if (!__syncthreads_or(todo != 0)) continue;
    float sum[8] = {};
    for (int k0 = 0; k0 < p.K; k0 += kRepairK) {
      const int xr = threadIdx.x >> 3, xk = 8 * (threadIdx.x & 7);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (t0 + xr < p.tokens && k0 + xk < p.K)  // K is a multiple of 8
        v = __ldg(reinterpret_cast<const uint4 *>(p.X + static_cast<long long>(t0 + xr) * p.K + k0 + xk));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
        s_x[xr][xk + 2 * e] = f.x;
        s_x[xr][xk + 2 * e + 1] = f.y;
      }
      __syncthreads();
      if (todo) {
        const __half *wc = p.W + static_cast<long long>(k0) * p.N + c;
        const int end = min(kRepairK, p.K - k0);
#pragma unroll 8
        for (int k = 0; k < end; ++k) {
          const float wv = __half2float(wc[static_cast<long long>(k) * p.N]);
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[i] = fmaf(s_x[row + i][k], wv, sum[i]);
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (((todo >> i) & 1u) == 0) continue;
      const int t = t0 + row + i, entry = s_entry[row + i];
      if (entry >= 0) {
        // The row of H as the GEMM took it.
        const __half *up = p.up + static_cast<long long>(s_own[row + i]) * p.rank * p.N + c;
        for (int r = 0; r < p.rank; ++r) {
          const long long blk = static_cast<long long>(entry) * p.chunks + (r >> 6);
          const float h = __half2float(p.low[(blk * p.tile_rows + t % p.tile_rows) * 64 + (r & 63)]);
          sum[i] = fmaf(h, __half2float(up[static_cast<long long>(r) * p.N]), sum[i]);
        }
      }
      p.Y[static_cast<long long>(t) * p.N + c] = __float2half_rn(sum[i]);
    }
  }
}

// ------------------------------------------------------------------------------ few tokens
constexpr int kFewTokens = 64;  // of a CTA, at most (the accumulator's columns)
constexpr int kFewCols = 128;   // columns of W in a CTA
constexpr int kAddWarps = 8;    // that form the adapters' part and join the partial sums
constexpr int kLoadWarps = 4;   // two for W, two for X, each every other stage
constexpr int kFewThreads = 32 * (1 + kAddWarps + kLoadWarps);
constexpr int kFewPart = kFewCols + 4;  // floats of a partial row
constexpr int kLowThreads = 256;
constexpr int kMaxSlices = 16;
constexpr int kFewSmem = 104 * 1024;    // two CTAs to an SM

struct LoraFewParams {
  const __half *X, *down, *up;
  __half *Y;
  const float *scale;
  const int *seg_start, *seg_adapter;
  float *low;  // slices x tokens x rank: partial sums of X Down
  int tokens, N, K, rank, adapters, segments;
  int slices, slice_rows;   // K ranges of the first product
  int n16;                  // tokens of a CTA, rounded up to 16
  int ksplit, num_kb, stages, share;  // share: tokens that a CTA of the cluster joins
  int whole_blocks;  // N % 64 == 0: tmW is (64 columns, K, column blocks), one box for 128 columns
  unsigned *status_word;
  unsigned long long timeout_ns;
};

// Adapter of token t, or -1, by one warp: every segment is looked at at once, so that this costs one
// round trip to memory (a binary search with the adapter behind it is a chain of several).
__device__ __forceinline__ int warp_token_adapter(const int *seg_start, const int *seg_adapter,
                                                  int segments, int adapters, int t) {
  int hit = -1, mine = -1;
#pragma unroll 2
  for (int i = threadIdx.x & 31; i < segments; i += 32) {
    const int b = seg_start[i], e = seg_start[i + 1], a = seg_adapter[i];
    if (b <= t && t < e) {
      hit = i;
      mine = a;
    }
  }
  const int last = __reduce_max_sync(0xffffffffu, hit);
  if (last < 0) return -1;
  const int a = __shfl_sync(0xffffffffu, mine, last & 31);
  return (a >= 0 && a < adapters) ? a : -1;
}

// Partial sums of X Down for one token and K range: a thread takes 8 columns of every few rows.
__global__ void __launch_bounds__(kLowThreads) lora_low_kernel(const LoraFewParams p) {
  ptx::grid_launch_dependents();
  __shared__ float s_sum[kLowThreads / 32][kMaxRank];
  const int t = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
  const int a = warp_token_adapter(p.seg_start, p.seg_adapter, p.segments, p.adapters, t);
  if (a < 0) return;
  const int g8 = p.rank / 8;  // 16-byte groups of a row of Down
  const int width = g8 <= 1 ? 1 : 1 << (32 - __clz(g8 - 1));  // lanes of a row, a power of two
  const int g = threadIdx.x & (width - 1), r0 = threadIdx.x / width, rows = kLowThreads / width;
  const int k0 = slice * p.slice_rows, k1 = min(p.K, k0 + p.slice_rows);
  const __half *x = p.X + static_cast<long long>(t) * p.K;
  const __half *dn = p.down + static_cast<long long>(a) * p.K * p.rank + 8 * g;
  float f[8] = {};
  if (g < g8) {
#pragma unroll 8
    for (int k = k0 + r0; k < k1; k += rows) {
      const uint4 u = __ldg(reinterpret_cast<const uint4 *>(dn + static_cast<long long>(k) * p.rank));
      const float xv = __half2float(x[k]);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        f[2 * i] = fmaf(xv, v.x, f[2 * i]);
        f[2 * i + 1] = fmaf(xv, v.y, f[2 * i + 1]);
      }
    }
  }
  for (int m = 16; m >= width; m >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] += __shfl_xor_sync(0xffffffffu, f[i], m);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane < width && g < g8)
#pragma unroll
    for (int i = 0; i < 8; ++i) s_sum[warp][8 * g + i] = f[i];
  __syncthreads();
  if (threadIdx.x < p.rank) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kLowThreads / 32; ++w) sum += s_sum[w][threadIdx.x];
    p.low[(static_cast<long long>(slice) * p.tokens + t) * p.rank + threadIdx.x] = sum;
  }
}

__global__ void __launch_bounds__(kFewThreads, 2)
    lora_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                    const LoraFewParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ float s_low[kAddWarps][kMaxRank];
  __shared__ int s_adapter[kFewTokens];
  __shared__ __align__(8) uint64_t s_full[8], s_empty[8], s_acc;
  __shared__ int s_abort;
  __shared__ uint32_t s_tmem;
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (base - raw);
  const int x_bytes = p.n16 * 128, stage_bytes = 2 * kBBytes + x_bytes;
  float *delta = reinterpret_cast<float *>(smem + p.stages * stage_bytes);  // share x kFewCols
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % p.ksplit, n0 = blockIdx.x / p.ksplit * kFewCols;
  const int first = blockIdx.y * kFewTokens;
  const int kb0 = static_cast<int>(static_cast<long long>(p.num_kb) * split / p.ksplit);
  const int kb1 = static_cast<int>(static_cast<long long>(p.num_kb) * (split + 1) / p.ksplit);
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < p.stages; ++i) {
      ptx::mbar_init(ptx::smem_u32(&s_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&s_empty[i]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(&s_acc), 1);
    ptx::fence_mbar_init_cluster();
  }
  if (warp == 1) {
    ptx::tmem_alloc<1>(ptx::smem_u32(&s_tmem), 64);
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&s_tmem);
  const OpWait wc{&s_abort, p.status_word, p.timeout_ns};
  // Tokens that this CTA joins, adds the adapters' part to and writes.
  const int end = min(p.tokens, first + kFewTokens);
  const int t0 = min(end, first + split * p.share), t1 = min(end, t0 + p.share);

  // Warps 0.. 7 add, 8 issues products, 9.. load. A thread is held 400 to 600 cycles by a TMA load, which
  // for one thread and stages of 16 KB would be a third of what an SM can take in.
  constexpr int kIssueWarp = kAddWarps;
  if (warp > kIssueWarp) {
    const int me = warp - kIssueWarp - 1;
    const bool loads_x = me >= kLoadWarps / 2;
    if (lane == 0) {
      bool ok = true;
      int it = me & 1;
      for (; it < kb1 - kb0; it += 2) {
        const int st = it % p.stages, kb = kb0 + it;
        if (it >= p.stages && !(ok = op_wait(ptx::smem_u32(&s_empty[st]), (it / p.stages - 1) & 1, wc,
                                             kSiteLoraFewEmpty)))
          break;
        const uint32_t bar = ptx::smem_u32(&s_full[st]), dst = base + st * stage_bytes;
        if (loads_x) {
          // (counted on the barrier before or after the bytes are announced)
          ptx::tma_load_2d(&tmX, dst + 2 * kBBytes, bar, kb * 64, first);
        } else {
          ptx::mbar_arrive_expect_tx(bar, stage_bytes);
          if (p.whole_blocks) {
            ptx::tma_load_3d(&tmW, dst, bar, 0, kb * 64, n0 / 64);
          } else {
            ptx::tma_load_2d(&tmW, dst, bar, n0, kb * 64);
            ptx::tma_load_2d(&tmW, dst + kBBytes, bar, n0 + 64, kb * 64);
          }
        }
      }
      if (!ok && !loads_x)
        for (int j = max(me & 1, it - 2 * p.stages); j < it; j += 2)
          op_drain(ptx::smem_u32(&s_full[j % p.stages]), (j / p.stages) & 1);
    }
  } else if (warp == kIssueWarp) {
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t idesc = ptx::umma_idesc_f16_f32(kFewCols, p.n16, true, true);
    const bool one = ptx::elect_one();
    int st = 0, ph = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, op_wait(ptx::smem_u32(&s_full[st]), ph, wc, kSiteLoraFewFull))) break;
      ptx::tc_fence_after();
      const uint32_t src = base + st * stage_bytes;
      // W: columns are M (64-column blocks 8 KB apart), 16 k are 16 rows of 128 bytes. X: K-major.
      const uint64_t wd = ptx::umma_desc_sw128(src, kBBytes, 1024);
      const uint64_t xd = ptx::umma_desc_sw128(src + 2 * kBBytes, 16, 1024);
      if (one) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          ptx::umma_f16<1>(tm, wd + 128 * k, xd + 2 * k, idesc, kb > kb0 || k > 0);
        if (kb + p.stages < kb1) ptx::umma_commit<1>(ptx::smem_u32(&s_empty[st]));
      }
      if (++st == p.stages) {
        st = 0;
        ph ^= 1;
      }
    }
    if (one) ptx::umma_commit<1>(ptx::smem_u32(&s_acc));
    __syncwarp();
  } else {
    // The adapters' part of this CTA's tokens, while the main loop runs: a warp takes a token, 16 lanes
    // its 128 columns, the two halves of the warp every other row of Up.
    const int w = warp, c = 8 * (lane & 15);
    // What does not hang on the first product: whose token it is, and Up's rows into L2.
    for (int t = t0 + w; t < t1; t += kAddWarps) {
      const int a = warp_token_adapter(p.seg_start, p.seg_adapter, p.segments, p.adapters, t);
      if (lane == 0) s_adapter[t - t0] = a;
      if (a >= 0 && n0 + c < p.N)
        for (int r = lane >> 4; r < p.rank; r += 2)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(
              p.up + (static_cast<long long>(a) * p.rank + r) * p.N + n0 + c));
    }
    ptx::grid_wait();
    for (int t = t0 + w; t < t1; t += kAddWarps) {
      __syncwarp();
      const int a = s_adapter[t - t0];
      float f[8] = {};
      if (a >= 0) {
        const float sc = p.scale[a];
        for (int r = lane; r < p.rank; r += 32) {
          float h[kMaxSlices];
#pragma unroll
          for (int s = 0; s < kMaxSlices; ++s)
            h[s] = s < p.slices ? p.low[(static_cast<long long>(s) * p.tokens + t) * p.rank + r] : 0.0f;
          float sum = 0.0f;
#pragma unroll
          for (int s = 0; s < kMaxSlices; ++s) sum += h[s];
          s_low[w][r] = sum * sc;
        }
        __syncwarp();
        if (n0 + c < p.N) {
          const __half *up = p.up + static_cast<long long>(a) * p.rank * p.N + n0 + c;
#pragma unroll 8
          for (int r = lane >> 4; r < p.rank; r += 2) {
            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(up + static_cast<long long>(r) * p.N));
            const float h = s_low[w][r];
            const uint32_t v4[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&v4[i]));
              f[2 * i] = fmaf(h, v.x, f[2 * i]);
              f[2 * i + 1] = fmaf(h, v.y, f[2 * i + 1]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += __shfl_xor_sync(0xffffffffu, f[i], 16);
      }
      if (lane < 16) {
        float *dst = delta + (t - t0) * kFewCols + c;
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = f[i];
      }
    }
  }
  // Partial sums to shared memory (the stages are free once the last product has retired).
  __syncwarp();
  int okw = 1;
  if (lane == 0) okw = op_wait(ptx::smem_u32(&s_acc), 0, wc, kSiteLoraFewAcc);
  const bool ok = __shfl_sync(0xffffffffu, okw, 0) != 0;
  ptx::tc_fence_after();
  float *part = reinterpret_cast<float *>(smem);  // token x column
  const bool adds = warp < kAddWarps;
  if (adds && ok) {
    // (two warps to a lane quarter, every other 16 columns each)
    const int q = warp & 3;
    for (int c = 16 * (warp >> 2); c < p.n16; c += 32) {
      uint32_t v[16];
      ptx::tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(q) << 21) + c, v);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) part[(c + i) * kFewPart + 32 * q + lane] = __uint_as_float(v[i]);
    }
  }
  ptx::tc_fence_before();
  if (p.ksplit > 1)
    ptx::cluster_sync();
  else
    __syncthreads();
  if (adds && ok) {
    constexpr int kAhead = 2, kStep = kAddWarps / 4;  // tokens in flight of a thread; of the CTA
    const int col = threadIdx.x & (kFewCols - 1);
    const uint32_t part_addr = ptx::smem_u32(part) - first * (kFewPart * 4);
    for (int t = t0 + static_cast<int>(threadIdx.x) / kFewCols; t < t1; t += kAhead * kStep) {
      float v[kAhead][8];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int tt = min(t + x * kStep, t1 - 1);
        const uint32_t off = part_addr + (tt * kFewPart + col) * 4;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < p.ksplit) v[x][k] = ptx::ld_shared_cluster_f(ptx::mapa(off, k));
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int tt = t + x * kStep;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < p.ksplit) sum += v[x][k];
        if (tt < t1 && n0 + col < p.N)
          p.Y[static_cast<long long>(tt) * p.N + n0 + col] =
              __float2half_rn(sum + delta[(tt - t0) * kFewCols + col]);
      }
    }
  }
  if (p.ksplit > 1)
    ptx::cluster_sync();  // nobody reads this CTA's partials any more
  else
    __syncthreads();
  if (warp == 1) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, 64);
  }
}

// ------------------------------------------------------------------------------ host side
bool sizes_ok(int tokens, int N, int K, int rank, int adapters, int segments) {
  return tokens >= 0 && N >= 0 && K >= 8 && N % 8 == 0 && K % 8 == 0 && rank >= 8 &&
         rank <= kMaxRank && rank % 8 == 0 && adapters >= 0 && segments >= 0;
}
bool too_large(int tokens, int N, int K, int segments) {
  return tokens > kOpMaxRows || N > kOpMaxRows || K > kOpMaxRows || segments > kOpMaxSegments;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Few tokens: K ranges of the first product, so that the CTAs of all tokens fill the SMs a few times, of
// 64 rows at least (a workspace of `tokens` tokens holds them).
int few_slices(int tokens, int K) {
  return std::max(1, std::min({kMaxSlices, 592 / tokens, K / 64}));
}

struct FewPlan {
  bool use;
  int tiles, chunks, most, n16, num_kb, ksplit, share, stage;
};
// How few tokens are run, and whether: depends on the sizes alone, since the workspace does.
FewPlan few_plan(int tokens, int N, int K, int rank, int adapters, int segments) {
  FewPlan f;
  f.tiles = (N + kFewCols - 1) / kFewCols;
  f.chunks = (tokens + kFewTokens - 1) / kFewTokens;
  f.most = std::min(tokens, kFewTokens);  // of a CTA
  f.n16 = (f.most + 15) / 16 * 16;
  f.num_kb = (K + 63) / 64;
  f.stage = 2 * kBBytes + f.n16 * 128;
  // Two CTAs to an SM, and of K as many ranges as they take, a power of two, with 4 k-blocks or more each
  // (clusters of 6 left CTAs for a second wave: 26 us against 20 us with 4 at N = 6144).
  const long long items = static_cast<long long>(f.tiles) * f.chunks;
  f.ksplit = 1;
  while (f.ksplit < 8 && 2 * f.ksplit * items <= 2 * kSms && f.num_kb >= 8 * f.ksplit) f.ksplit *= 2;
  f.share = (f.most + f.ksplit - 1) / f.ksplit;
  // This path reads Down and Up once for every token, W once for every 64, and splits K; the other takes an
  // adapter's tokens together, in row tiles, and does not split. Both in us, fitted to eager calls of 1 to 512 tokens, ranks
  // of 8 to 128, one to 200 adapters at 36 sizes of K x N from 536 x 1440 to 19192 x 33352 and 4096 x 128256, each in
  // both paths: at 95% of 2774 points the rule takes the faster one or one within 5% of it, on average 0.8% is lost,
  // at worst 55% (200 tokens of as many adapters, rank 8, 5088 x 17840). This path and the other, in us:
  //    K x N          tokens, rank, adapters: us, us
  //    4096 x 4096    1, 16, 1: 13.6, 32.8    128, 16, 1: 21.1, 32.6   256, 64, 32: 70.6, 57.4   512, 16, 1: 57.4, 44.7
  //    4096 x 28672   1, 16, 1: 39.4, 57.7    48, 16, 1: 52.0, 48.9    48, 64, 32: 107, 82       128, 16, 1: 125, 51
  //    14336 x 4096   1, 16, 1: 28.2, 103     48, 64, 32: 53.4, 95.6   192, 64, 32: 131, 116
  //    8192 x 57344   1, 16, 1: 139, 192      48, 16, 1: 191, 166
  const int rows = (tokens + kTileRows - 1) / kTileRows, chunks = (rank + 63) / 64;
  const int distinct = std::min({tokens, adapters, segments});  // adapters, at most
  const double w_mb = 2e-6 * K * N, adapter_mb = 2e-6 * distinct * rank * (static_cast<double>(K) + N);
  const double waves = std::ceil(static_cast<double>(items * f.ksplit) / (2 * kSms));
  const int slices = few_slices(tokens, K);
  const double here = 4.6 + 6.3 * waves +                                    // launches; a CTA's start and end
                      0.10 * waves * f.num_kb / f.ksplit * f.stage / 16384 +  // W and X into an SM
                      0.123 * f.chunks * w_mb + 0.183 * adapter_mb +          // out of memory or L2
                      9.3e-5 * K / slices * rank * std::ceil(tokens * slices / (8.0 * kSms)) +  // Down for each token
                      7.5e-8 * tokens * N * rank + 0.0066 * f.share * rank * waves;             // Up, its sums
  const int of_tile = std::min(distinct, kTileRows);  // adapters of a row tile, at most
  const int per_group = std::max(1, kBlocks / chunks);
  const double shrinks = static_cast<double>((of_tile + per_group - 1) / per_group) * rows;  // products X Down
  double ksplit = 1.0;
  while (ksplit < 8.0 && 2.0 * ksplit * shrinks <= kSms && f.num_kb >= 8.0 * ksplit) ksplit *= 2.0;
  const double tiles = static_cast<double>(rows) * ((N + 255) / 256) / kSms;  // of an SM
  const double other = 6.7 + 9.9 * std::ceil(tiles) +
                       std::max(1.0, tiles) * (0.166 * f.num_kb + 0.60 * chunks * of_tile) +
                       0.122 * w_mb + 0.088 * adapter_mb +
                       0.234 * std::ceil(shrinks * ksplit / kSms) * f.num_kb / ksplit +  // H, the longest
                       0.23 * shrinks * f.num_kb / kSms;                                 // and all of it
  f.use = tokens <= 512 && here <= other;
  return f;
}

// Entries of a call (an adapter of a row tile each): a tile has at most as many as adapters, and all have
// at most one each more than segments that begin in them. The fewer of the two decides (4096 requests of one token over
// 8 adapters at rank 64: 4 MB of operand blocks instead of 135).
struct Entries {
  int per_tile;  // 0: as the segments say
  long long all;
};
Entries entries_of(int tokens, int tile_rows, int adapters, int segments) {
  const long long tiles = (tokens + tile_rows - 1) / tile_rows;
  const int most = std::min(tile_rows, adapters);
  if (tiles * most <= tiles + segments) return {most, tiles * most};
  return {0, tiles + segments};
}

// Workspace, in order: the entries' tables, the list of odd blocks, the operand blocks. Sized for
// 128-row tiles' tables and 256-row tiles' blocks, whichever the GEMM takes.
struct Layout {
  size_t tables, list, low, total;
};
Layout layout(int tokens, int N, int rank, int adapters, int segments) {
  Layout l;
  const long long t128 = (tokens + 127) / 128;
  const long long e128 = entries_of(tokens, 128, adapters, segments).all;
  const long long e256 = entries_of(tokens, 256, adapters, segments).all;
  l.tables = up256(static_cast<size_t>(2 * t128 + std::max(e128, e256) + 1) * sizeof(int));
  l.list = up256(static_cast<size_t>((tokens + 31) / 32) * ((N + 63) / 64) * 8);
  const size_t row = static_cast<size_t>((rank + 63) / 64) * 64 * sizeof(__half);
  l.low = static_cast<size_t>(std::max(e128 * 128, e256 * 256)) * row;
  l.total = l.tables + l.list + l.low;
  return l;
}

int check(const hgemm_lora_t *a) {
  if (!a || !sizes_ok(a->tokens, a->N, a->K, a->rank, a->adapters, a->segments))
    return HGEMM_ERR_INVALID_ARG;
  if (too_large(a->tokens, a->N, a->K, a->segments)) return HGEMM_ERR_TOO_LARGE;
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
  const int A = a->segments > 0 ? a->adapters : 0;
  const OpRows in[] = {op_dense(a->X, 2, a->tokens, a->K), op_dense(a->W, 2, a->K, a->N),
                       op_dense(a->down, 2, A, a->K, a->rank), op_dense(a->up, 2, A, a->rank, a->N),
                       op_dense(a->scale, 4, A), op_dense(a->seg_start, 4, A > 0 ? a->segments + 1 : 0),
                       op_dense(a->seg_adapter, 4, A > 0 ? a->segments : 0)};
  const OpRows Y = op_dense(a->Y, 2, a->tokens, a->N), ws = op_dense(a->workspace, 1, static_cast<double>(need));
  bool over = op_overlap(Y, ws);
  for (const OpRows &x : in) over |= op_overlap(Y, x) || op_overlap(ws, x);
  return over ? HGEMM_ERR_INVALID_ARG : HGEMM_OK;
}

int run_few(const hgemm_lora_t *a, const OpDevice &d, cudaStream_t stream) {
  LoraFewParams p;
  p.X = a->X;
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
  p.slices = few_slices(a->tokens, a->K);
  p.slice_rows = (a->K + p.slices - 1) / p.slices;
  const FewPlan f = few_plan(a->tokens, a->N, a->K, a->rank, a->adapters, a->segments);
  p.n16 = f.n16;
  p.num_kb = f.num_kb;
  p.ksplit = f.ksplit;
  p.share = f.share;
  p.status_word = d.status_word;
  p.timeout_ns = d.timeout_ns;
  const int delta = p.share * kFewCols * 4;
  p.stages = std::min(8, (kFewSmem - 1024 - delta) / f.stage);
  const int smem = 1024 + p.stages * f.stage + delta;
  CUtensorMap tw, tx;
  const unsigned long long wd[2] = {static_cast<unsigned long long>(a->N),
                                    static_cast<unsigned long long>(a->K)};
  const unsigned long long ws[1] = {2ull * a->N};
  const unsigned wb[2] = {64, 64};
  const unsigned long long xd[2] = {static_cast<unsigned long long>(a->K),
                                    static_cast<unsigned long long>(a->tokens)};
  const unsigned long long xs[1] = {2ull * a->K};
  const unsigned xb[2] = {64, static_cast<unsigned>(p.n16)};
  const unsigned long long wd3[3] = {64, static_cast<unsigned long long>(a->K),
                                     static_cast<unsigned long long>(a->N / 64)};
  const unsigned long long ws3[2] = {2ull * a->N, 128};
  const unsigned wb3[3] = {64, 64, 2};
  p.whole_blocks = a->N % 64 == 0;
  if (!(p.whole_blocks ? op_encode(&tw, a->W, 3, wd3, ws3, wb3) : op_encode(&tw, a->W, 2, wd, ws, wb)) ||
      !op_encode(&tx, a->X, 2, xd, xs, xb))
    return HGEMM_ERR_TENSOR_MAP;
  static unsigned done[64];
  const int st = op_smem(reinterpret_cast<const void *>(lora_few_kernel), kFewSmem, d.dev, done);
  if (st != HGEMM_OK) return st;
  lora_low_kernel<<<p.tokens * p.slices, kLowThreads, 0, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return HGEMM_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(f.tiles * f.ksplit), static_cast<unsigned>(f.chunks), 1);
  cfg.blockDim = dim3(kFewThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.ksplit;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.ksplit > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, lora_few_kernel, tw, tx, p) != cudaSuccess) {
    cudaGetLastError();
    return HGEMM_ERR_LAUNCH;
  }
  return HGEMM_OK;
}

int run(const hgemm_lora_t *a, cudaStream_t stream) {
  int st = check(a);
  if (st != HGEMM_OK || a->tokens == 0 || a->N == 0) return st;
  if (a->adapters == 0 || a->segments == 0)
    return hgemm_launch(a->X, a->W, a->Y, a->tokens, a->N, a->K, 1.0f, 0.0f, stream);
  OpDevice d;
  st = op_device(&d);
  if (st != HGEMM_OK) return st;
  if (few_plan(a->tokens, a->N, a->K, a->rank, a->adapters, a->segments).use) return run_few(a, d, stream);
  LoraParams p;
  st = lora_gemm_tile_rows(a->tokens, a->N, a->K, &p.tile_rows);
  if (st != HGEMM_OK) return st;
  p.X = a->X;
  p.W = a->W;
  p.down = a->down;
  p.up = a->up;
  p.Y = a->Y;
  p.scale = a->scale;
  p.seg_start = a->seg_start;
  p.seg_adapter = a->seg_adapter;
  p.tokens = a->tokens;
  p.N = a->N;
  p.K = a->K;
  p.rank = a->rank;
  p.adapters = a->adapters;
  p.segments = a->segments;
  p.chunks = (a->rank + 63) / 64;
  p.num_kb = (a->K + 63) / 64;
  const int tiles = (a->tokens + p.tile_rows - 1) / p.tile_rows;
  const Layout l = layout(a->tokens, a->N, a->rank, a->adapters, a->segments);
  const Entries e = entries_of(a->tokens, p.tile_rows, a->adapters, a->segments);
  if (e.all * p.chunks * p.tile_rows > 0x7fffffffll) return HGEMM_ERR_TOO_LARGE;
  p.per_tile = e.per_tile;
  p.entries = static_cast<int>(e.all);
  char *ws = static_cast<char *>(a->workspace);
  p.odd_count = reinterpret_cast<unsigned *>(ws);
  p.base = reinterpret_cast<int *>(ws) + 1;
  p.count = p.base + tiles;
  p.adapter = p.count + tiles;
  p.odd_list = reinterpret_cast<unsigned long long *>(ws + l.tables);
  p.low = reinterpret_cast<__half *>(ws + l.tables + l.list);
  p.status_word = d.status_word;
  p.timeout_ns = d.timeout_ns;
  p.per_group = std::max(1, kBlocks / p.chunks);
  const int most = std::min(std::min(p.tile_rows, a->segments), a->adapters);
  p.groups = (most + p.per_group - 1) / p.per_group;
  // K is split over a cluster until the CTAs fill the SMs, with at least 4 k-blocks for each.
  const int tiles128 = (a->tokens + kTileRows - 1) / kTileRows;
  p.ksplit = 1;
  while (p.ksplit < 8 && 2ll * p.ksplit * tiles128 * p.groups <= d.sm_count && p.num_kb >= 8 * p.ksplit)
    p.ksplit *= 2;
  const long long ctas =
      static_cast<long long>(tiles) * (p.tile_rows / kTileRows) * p.groups * p.ksplit;
  if (ctas > 0x7fffffffll) return HGEMM_ERR_TOO_LARGE;

  CUtensorMap tx, td;
  const unsigned long long xd[2] = {static_cast<unsigned long long>(a->K),
                                    static_cast<unsigned long long>(a->tokens)};
  const unsigned long long xs[1] = {2ull * a->K};
  const unsigned xb[2] = {64, kTileRows};
  const unsigned long long dd[3] = {static_cast<unsigned long long>(a->rank),
                                    static_cast<unsigned long long>(a->K),
                                    static_cast<unsigned long long>(a->adapters)};
  const unsigned long long ds[2] = {2ull * a->rank, 2ull * a->rank * a->K};
  const unsigned db[3] = {64, 64, 1};
  if (!op_encode(&tx, a->X, 2, xd, xs, xb) || !op_encode(&td, a->down, 3, dd, ds, db))
    return HGEMM_ERR_TENSOR_MAP;
  static unsigned done[64];
  st = op_smem(reinterpret_cast<const void *>(lora_shrink_kernel), kSmem, d.dev, done);
  if (st != HGEMM_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.ksplit;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.ksplit > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, lora_shrink_kernel, tx, td, p) != cudaSuccess) {
    cudaGetLastError();
    return HGEMM_ERR_LAUNCH;
  }
  LoraExt ext;
  ext.low = p.low;
  ext.up = p.up;
  ext.entries = p.entries;
  ext.chunks = p.chunks;
  ext.rank = p.rank;
  ext.adapters = p.adapters;
  ext.base = p.base;
  ext.count = p.count;
  ext.adapter = p.adapter;
  ext.odd_count = p.odd_count;
  ext.odd_list = p.odd_list;
  st = lora_gemm(a->X, a->W, a->Y, a->tokens, a->N, a->K, ext, stream);
  if (st != HGEMM_OK) return st;
  lora_repair_kernel<<<2 * d.sm_count, kRepairThreads, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? HGEMM_OK : HGEMM_ERR_LAUNCH;
}

}  // namespace
}  // namespace hgemm

extern "C" {

int hgemm_lora(const hgemm_lora_t *args, hgemm_stream_t stream) {
  return hgemm::op_status(hgemm::run(args, stream));
}

size_t hgemm_lora_workspace_bytes(int tokens, int N, int K, int rank, int adapters, int segments) {
  if (!hgemm::sizes_ok(tokens, N, K, rank, adapters, segments) ||
      hgemm::too_large(tokens, N, K, segments))
    return 0;
  if (tokens == 0 || N == 0 || adapters == 0 || segments == 0) return 0;
  if (hgemm::few_plan(tokens, N, K, rank, adapters, segments).use)
    return static_cast<size_t>(hgemm::few_slices(tokens, K)) * tokens * rank * sizeof(float);
  return hgemm::layout(tokens, N, rank, adapters, segments).total;
}

}  // extern "C"
