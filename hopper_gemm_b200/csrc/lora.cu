// A shared projection with the low-rank adapters of many requests beside it:
//   Y[t,:] = X[t,:] W + scale[a] * (X[t,:] Down[a]) Up[a],  a the adapter of token t's segment.
//
// Two launches (and one that returns at once). lora_shrink_kernel forms H = scale (X Down): one
// tcgen05 product for every (row tile, adapter in it), K split over a cluster, and leaves H as
// operand blocks of the second product: for every adapter of a row tile a block of 64-column rows in
// which the rows of other adapters are zero. The projection's own GEMM kernel (hgemm_sm100.cu) then
// walks those blocks as additional k-blocks behind the k-blocks of X and W, so that Up's product
// lands in the same fp32 accumulators and Y is written and rounded once; an adapter costs its row
// tiles rank / K of the GEMM. H is rounded to binary16 because it is a tcgen05 operand next to Up.
//
// No counterpart in the reference.

#include <algorithm>

#include "ops_sm100.cuh"

namespace hgemm {
namespace {

constexpr int kMaxRank = 256;
constexpr int kTileRows = 128;     // rows of a shrink CTA
constexpr int kMaxTileRows = 256;  // rows of a GEMM tile
constexpr int kSegCache = 1024;    // segment starts kept in shared memory
constexpr int kStages = 4;
constexpr int kBlocks = 4;         // 64-column blocks of Down in a stage
constexpr int kABytes = kTileRows * 128;
constexpr int kBBytes = 64 * 128;
constexpr int kStageBytes = kABytes + kBlocks * kBBytes;
constexpr int kSmem = 1024 + kStages * kStageBytes + 256;
constexpr int kPartStride = kBlocks * 64 + 4;  // floats of a partial row, padded for the banks
static_assert(kTileRows * kPartStride * 4 <= kStages * kStageBytes, "partials reuse the stages");
constexpr int kThreads = 192;

struct LoraParams {
  const __half *X, *W, *down, *up;
  __half *Y;
  const float *scale;
  const int *seg_start, *seg_adapter;
  int tokens, N, K, rank, adapters, segments;
  int tile_rows, chunks;    // rows of a GEMM tile; 64-column blocks of H
  int groups, per_group;    // adapters of a tile are taken `per_group` at a time by `groups` CTAs
  int ksplit, num_kb;
  int entries;
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
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_seg[kSegCache];
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
  const int *starts = p.seg_start;
  if (p.segments < kSegCache) {
    for (int i = threadIdx.x; i <= p.segments; i += kThreads) s_seg[i] = p.seg_start[i];
    starts = s_seg;
    __syncthreads();
  }
  for (int i = threadIdx.x; i < p.tile_rows; i += kThreads)
    s_adapter[i] = tile0 + i < p.tokens
                       ? token_adapter(starts, p.seg_adapter, p.segments, p.adapters, tile0 + i)
                       : -1;
  if (threadIdx.x == 0) {
    // Tiles before this one have at most one entry each more than the segments that begin in them.
    s_base = tile + starts_upto(starts, p.segments, tile0 - 1);
    s_abort = 0;
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(full + 8 * i, 1);
      ptx::mbar_init(empty + 8 * i, 1);
    }
    ptx::mbar_init(acc, 1);
    ptx::fence_mbar_init_cluster();
  }
  __syncthreads();
  for (int i0 = warp * 32; i0 < p.tile_rows; i0 += kThreads) {
    const int i = i0 + lane, a = s_adapter[i];
    bool first = a >= 0 && (i == 0 || s_adapter[i - 1] != a);
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
  if (nu <= 0 || row0 >= p.tokens) return;

  if (warp == 1) {
    ptx::tmem_alloc<1>(ptx::smem_u32(&s_tmem), 256);
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&s_tmem);
  const int kb0 = static_cast<int>(static_cast<long long>(p.num_kb) * split / p.ksplit);
  const int kb1 = static_cast<int>(static_cast<long long>(p.num_kb) * (split + 1) / p.ksplit);
  const OpWait wc{&s_abort, p.status_word, p.timeout_ns};
  const int cols = p.chunks * 64;  // accumulator columns of an adapter
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int st = it % kStages;
        if (it >= kStages && !op_wait(empty + 8 * st, (it / kStages - 1) & 1, wc, kSiteLoraEmpty)) {
          ok = false;
          break;
        }
        ptx::mbar_arrive_expect_tx(full + 8 * st, kABytes + nu * p.chunks * kBBytes);
        const uint32_t dst = base + st * kStageBytes;
        ptx::tma_load_2d(&tmX, dst, full + 8 * st, kb * 64, row0);
        for (int u = 0; u < nu; ++u)
          for (int c = 0; c < p.chunks; ++c)
            ptx::tma_load_3d(&tmDown, dst + kABytes + (u * p.chunks + c) * kBBytes, full + 8 * st,
                             64 * c, kb * 64, s_list[u0 + u]);
      }
      if (!ok)
        for (int j = max(0, it - kStages); j < it; ++j)
          op_drain(full + 8 * (j % kStages), (j / kStages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const int n16 = (p.rank + 15) / 16 * 16;
      const uint32_t idesc = ptx::umma_idesc_f16_f32(kTileRows, n16);
      int it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int st = it % kStages;
        if (!op_wait(full + 8 * st, (it / kStages) & 1, wc, kSiteLoraFull)) break;
        ptx::tc_fence_after();
        const uint32_t src = base + st * kStageBytes;
        const uint64_t ad = ptx::umma_desc_sw128(src, 16, 1024);
        for (int u = 0; u < nu; ++u) {
          const uint64_t bd =
              ptx::umma_desc_sw128(src + kABytes + u * p.chunks * kBBytes, kBBytes, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            ptx::umma_f16<1>(tmem + u * cols, ad + 2 * k, bd + 128 * k, idesc, it > 0 || k > 0);
        }
        if (kb + kStages < kb1) ptx::umma_commit<1>(empty + 8 * st);
      }
      ptx::umma_commit<1>(acc);
    }
  }
  // Partial sums to shared memory (the stages are free once the last product has retired).
  int okw = 1;
  if (lane == 0) okw = op_wait(acc, 0, wc, kSiteLoraAcc);
  ok = __shfl_sync(0xffffffffu, okw, 0) != 0;
  ptx::tc_fence_after();
  float *part = reinterpret_cast<float *>(smem);
  if (warp >= 2) {
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

// Blocks of Y that left the GEMM with an infinity or NaN: an adapter's own infinities or NaN may have
// reached rows of other adapters in the tile (times their zeros). Such elements are formed again from
// what they depend on alone, by one warp each; with nothing listed this returns at once.
__global__ void __launch_bounds__(256) lora_repair_kernel(const LoraParams p) {
  const unsigned n = *p.odd_count;
  const int lane = threadIdx.x & 31;
  const unsigned warps = gridDim.x * 8;
  for (unsigned long long e = blockIdx.x * 8 + (threadIdx.x >> 5); e < 2048ull * n; e += warps) {
    const unsigned long long block = p.odd_list[e >> 11];
    const int t = static_cast<int>(block & 0xffffffffu) + static_cast<int>((e >> 6) & 31);
    const int c = static_cast<int>(block >> 32) + static_cast<int>(e & 63);
    if (t >= p.tokens || c >= p.N) continue;
    __half *y = p.Y + static_cast<long long>(t) * p.N + c;
    if (__half2float(*y) - __half2float(*y) == 0.0f) continue;  // finite
    const __half *x = p.X + static_cast<long long>(t) * p.K;
    float sum = 0.0f;
    for (int k = lane; k < p.K; k += 32)
      sum = fmaf(__half2float(x[k]), __half2float(p.W[static_cast<long long>(k) * p.N + c]), sum);
    const int a = token_adapter(p.seg_start, p.seg_adapter, p.segments, p.adapters, t);
    if (a >= 0) {
      // The row of H as the GEMM took it: in the tile's entry of this adapter.
      const int tile = t / p.tile_rows;
      for (int u = 0; u < p.count[tile]; ++u) {
        const int entry = p.base[tile] + u;
        if (p.adapter[entry] != a) continue;
        for (int r = lane; r < p.rank; r += 32) {
          const long long blk = static_cast<long long>(entry) * p.chunks + (r >> 6);
          const float h = __half2float(p.low[(blk * p.tile_rows + t % p.tile_rows) * 64 + (r & 63)]);
          sum = fmaf(h, __half2float(p.up[(static_cast<long long>(a) * p.rank + r) * p.N + c]), sum);
        }
      }
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (lane == 0) *y = __float2half_rn(sum);
  }
}

// ------------------------------------------------------------------------------ host side
bool sizes_ok(int tokens, int N, int K, int rank, int adapters, int segments) {
  return tokens >= 0 && N >= 0 && K >= 8 && N % 8 == 0 && K % 8 == 0 && rank >= 8 &&
         rank <= kMaxRank && rank % 8 == 0 && adapters >= 0 && segments >= 0;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Workspace, in order: the entries' tables, the list of odd blocks, the operand blocks. Sized for
// 128-row tiles' tables and 256-row tiles' blocks, whichever the GEMM takes.
struct Layout {
  size_t tables, list, low, total;
  long long entries128, entries256;
};
Layout layout(int tokens, int N, int rank, int segments) {
  Layout l;
  const long long t128 = (tokens + 127) / 128, t256 = (tokens + 255) / 256;
  l.entries128 = t128 + segments;
  l.entries256 = t256 + segments;
  l.tables = up256(static_cast<size_t>(2 * t128 + l.entries128 + 1) * sizeof(int));
  l.list = up256(static_cast<size_t>((tokens + 31) / 32) * ((N + 63) / 64) * 8);
  const size_t row = static_cast<size_t>((rank + 63) / 64) * 64 * sizeof(__half);
  l.low = static_cast<size_t>(std::max(l.entries128 * 128, l.entries256 * 256)) * row;
  l.total = l.tables + l.list + l.low;
  return l;
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
  if (a->adapters == 0 || a->segments == 0)
    return hgemm_launch(a->X, a->W, a->Y, a->tokens, a->N, a->K, 1.0f, 0.0f, stream);
  OpDevice d;
  st = op_device(&d);
  if (st != HGEMM_OK) return st;
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
  const Layout l = layout(a->tokens, a->N, a->rank, a->segments);
  const long long entries = p.tile_rows == 128 ? l.entries128 : l.entries256;
  if (entries * p.chunks * p.tile_rows > 0x7fffffffll) return HGEMM_ERR_TOO_LARGE;
  p.entries = static_cast<int>(entries);
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
  static bool done[64];
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
  lora_repair_kernel<<<d.sm_count, 256, 0, stream>>>(p);
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
  if (tokens == 0 || N == 0 || adapters == 0 || segments == 0) return 0;
  return hgemm::layout(tokens, N, rank, segments).total;
}

}  // extern "C"
