// Attention over packed sequences with grouped heads (whole prompts, appended prompts, single
// tokens): O = softmax(scale * Q K^T) V for each sequence and head, one pass over the keys with a running
// maximum m and sum l of each row:
//   m' = max(m, max_j s_j);  w_j = 2^(s_j - m');  l' = 2^(m - m') l + sum w_j;  O' = 2^(m - m') O + sum w_j v_j,
// s in log2 units, O / l at the end. Scores, statistics and sums are fp32; the weights are rounded to
// binary16 for their product (see `fine` in make_plan), the output once.
//
// A CTA takes a tile of 128 rows: the queries of one key head's whole group, so that keys are loaded
// once for all heads that share them. Both products run on tcgen05: S = Q K^T from shared memory into
// TMEM, a thread to a row for the softmax (no exchange between lanes), the weights back into TMEM in
// the place of their scores, O += W V with W read from TMEM. Keys and values come by TMA, in boxes that may
// reach behind the sequence; what lies there is masked in the scores, and a row that infinities or NaN
// of such places reached (0 times infinity) is formed again over its own keys by attn_row: correct,
// but one row at a time by its warp, 7 keys a microsecond (2048 tokens of 32 heads that all see an infinite
// value: 10 ms instead of 62 us; a NaN score ends its row).
// Causal tiles load the blocks up to their last query's key alone and only blocks that end behind a
// row's limit are masked; the tiles with most keys start first.
//
// Long prompts: bound by the exponentials (64 a row and block, 4 lanes a cycle) beside the products; 16384 tokens
// of 32 heads over 8, head_dim 128, causal: 2.12 ms, 1040 TFLOP/s (1.88 ms in a replayed graph; the GPU's power
// moves both). Prompts of some 700 tokens (12 of 8192 in all) 137 us, where starts and ends of 2100 short CTAs
// count. Single tokens: bound by HBM; 16 over 131072 keys of 8 heads 112 us with the join, 4.8 TB/s. (Eager calls
// over changing inputs; the figures at the choices below compare variants in replayed graphs over one input.)
//
// No counterpart in the reference.

#include <algorithm>

#include "ops_sm100.cuh"

namespace hgemm {
namespace {

constexpr int kMaxDim = 128;
constexpr float kLog2e = 1.44269504088896340736f;

struct AttnParams {
  const __half *q, *k, *v;
  __half *out;
  float *lse;
  const int *cu_q, *cu_k;
  long long q_stride, k_stride, v_stride, out_stride;
  int total_q, total_k, batch, heads_q, heads_kv, group, head_dim, causal;
  float scale2;      // scale * log2(e): scores are kept in log2 units
  int dim16;         // head_dim rounded up to 16
  int tile_q;        // queries of a row tile (each with the group's heads)
  int q_box_bytes;   // bytes of one 64-element block of a tile's queries
  // Blocks of a key range and the most ranges of a sequence; chunk 0: no ranges. With ranges a row's parts
  // are joined by attn_join_kernel.
  int chunk, max_chunks;
  float *part_o;     // max_chunks x total_q x heads_q x dim16, each range's own weighted mean
  float *part_lse;   // max_chunks x total_q x heads_q, log2 of each range's sum
  unsigned *status_word;
  unsigned long long timeout_ns;
};

// Rows [begin, end) of sequence s, cut off at the rows that the tensor holds.
__device__ __forceinline__ void seq_range(const int *cu, int s, int total, int &begin, int &end) {
  begin = min(max(cu[s], 0), total);
  end = min(max(cu[s + 1], begin), total);
}

// One query row over keys [j0, j1) of its sequence, by one warp, in the order of the keys: lane l
// holds elements 4l..4l+3. Leaves the weighted sum relative to the maximum m (log2 units).
struct RowSum {
  float4 o;
  float m, l;
};
__device__ RowSum attn_row(const __half *qrow, const __half *k, const __half *v, long long k_stride,
                           long long v_stride, int head_dim, float scale2, int j0, int j1) {
  constexpr int kAtOnce = 8;  // keys, so that their loads and sums over the lanes overlap
  const int e0 = 4 * (threadIdx.x & 31);
  const bool live = e0 < head_dim;  // head_dim is a multiple of 8
  auto load4 = [&](const __half *src) {
    return live ? *reinterpret_cast<const uint2 *>(src + e0) : make_uint2(0u, 0u);
  };
  auto floats = [](uint2 u, float (&f)[4]) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    f[0] = a.x;
    f[1] = a.y;
    f[2] = b.x;
    f[3] = b.y;
  };
  float q[4];
  floats(load4(qrow), q);
  float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j = j0; j < j1; j += kAtOnce) {
    uint2 vv[kAtOnce];
    float s[kAtOnce], top = -INFINITY, nan = 0.0f;
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      const bool there = j + x < j1;
      float kk[4];
      floats(there ? load4(k + (j + x) * k_stride) : make_uint2(0u, 0u), kk);
      vv[x] = there ? load4(v + (j + x) * v_stride) : make_uint2(0u, 0u);
      s[x] = q[0] * kk[0] + q[1] * kk[1] + q[2] * kk[2] + q[3] * kk[3];
    }
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s[x] += __shfl_xor_sync(0xffffffffu, s[x], d);
      s[x] = j + x < j1 ? s[x] * scale2 : -INFINITY;
      top = fmaxf(top, s[x]);
      if (s[x] != s[x]) nan = s[x];
    }
    if (nan != 0.0f) return {make_float4(nan, nan, nan, nan), nan, nan};  // so is all of the row
    if (top > m) {
      const float f = exp2f(m - top);
      l *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= f;
      m = top;
    }
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      const float w = (s[x] == -INFINITY && m == -INFINITY) ? 0.0f : exp2f(s[x] - m);
      l += w;
      float f[4];
      floats(vv[x], f);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(w, f[i], o[i]);
    }
  }
  return {make_float4(o[0], o[1], o[2], o[3]), m, l};
}

// ------------------------------------------------------------------------------ the kernel
constexpr int kRows = 128;  // (query, head of the group) rows of a tile = TMEM lanes
constexpr int kBlock = 64;  // keys of a block, the unit of the softmax and of the masks
constexpr int kSmemLimit = 232448;
constexpr int kSms = 148;        // what plans (and with them workspaces) reckon with
constexpr int kMaxChunks = 64;   // key ranges of a sequence
// A row's weights are relative to a maximum that may lag the true one by this factor (log2): its
// output is rescaled only when the maximum has grown past it. 2^8 times a weight below 1 stays far
// inside binary16, and the fp32 sums do not care.
constexpr float kLag = 8.0f;
// That maximum is lowered by kRaise: a row's largest weight is 2^7 when the maximum is met and below 2^15 a lag behind
// (binary16 ends at 65504), weights down to 2^-21 of the largest keep all of binary16's 11 bits, and the grid
// of those below it is 2^-31 of it. (With the largest at 1 that grid is 2^-24: 131071 keys 15 below one in their
// logarithm came out 0.2 to 3% off, 17.5 below it they were gone.) Weighted values and sums scale alike.
constexpr float kRaise = 7.0f;

// DB: 64-element blocks of head_dim in shared memory (head_dim <= 64 DB); TILES: row tiles of a CTA,
// each with four softmax warps, a thread to a row; FINE: weights go into their product as two binary16
// numbers each, the second of what the first left over: 22 bits in all, down to 2^-10 of the row's largest
// (the second's own grid is kRaise's 2^-31 of it).
//
// Blocks of 64 keys, because a tile's scores then have two places in TMEM: the next block's scores are
// formed while a block's softmax runs, and no tile ever waits for the way from its weights through two
// products to its next scores. (With blocks of 128 keys in one place that way, 1300 cycles, stood in a
// row with the softmax's 1600: 3800 cycles for two tiles and 128 keys, where the exponentials take 2100 and the
// products 2050.)
template <int DB, int TILES>
struct AttnCfg {
  static constexpr int TILE_BYTES = DB * kRows * 128;   // queries of a tile
  // Blocks of a load. One CTA to an SM has the stages for two at a time, which takes half the loads and
  // announcements (16384 tokens: 1.89 ms against 2.04); two CTAs do not (141 us against 125 for 16 tokens
  // over long keys, with one).
  static constexpr int LOAD = TILES;
  static constexpr int LOAD_ROWS = LOAD * kBlock;
  static constexpr int LOAD_BYTES = DB * LOAD_ROWS * 128;
  static constexpr int CTAS = TILES == 1 ? 2 : 1;      // per SM
  static constexpr int SOFTMAX_WARPS = TILES * 4;
  static constexpr int THREADS = (SOFTMAX_WARPS + 2 + TILES) * 32;  // ... loads of keys, of values, products
  // Barriers, then whole 1024-byte swizzle atoms.
  static constexpr int HEAD = 1024;
  static constexpr int BUDGET = (kSmemLimit - (CTAS - 1) * 1024) / CTAS - HEAD;
  static constexpr int STAGES_FIT = (BUDGET - TILES * TILE_BYTES) / LOAD_BYTES;
  static constexpr int STAGES = STAGES_FIT > 10 ? 10 : STAGES_FIT;
  static constexpr int SMEM = HEAD + TILES * TILE_BYTES + STAGES * LOAD_BYTES;
  // TMEM columns: two blocks of scores of each tile (the weights take the place of their first half),
  // then the outputs.
  static constexpr int O_COL = TILES * 2 * kBlock;
  static constexpr int TMEM_COLS = TILES == 2 ? 512 : 256;
  static_assert(STAGES * LOAD >= 4, "the keys of two blocks, the values of two");
  static_assert(O_COL + TILES * DB * 64 <= TMEM_COLS, "TMEM");
  static_assert(8 * (2 * STAGES + 1 + 6 * TILES) + 32 <= HEAD, "barriers");
};

// log2 of the sum of a key range whose scores are all -infinity: no missing keys, which have -infinity here.
// Beside other ranges it weighs 0 (0 times an infinite value is NaN); a row of nothing else is 0 / 0.
constexpr float kAllMinusInf = -3.402823466e38f;

// Key ranges of a sequence with klen keys.
__device__ __forceinline__ int chunks_of(const AttnParams &p, int klen) {
  if (p.chunk == 0) return 1;
  const int blocks = (klen + kBlock - 1) / kBlock;
  return min(max((blocks + p.chunk - 1) / p.chunk, 1), p.max_chunks);
}

// Work of a CTA: a sequence, a tile of `span` queries in it and a range of its keys.
struct Tile {
  int q0, qlen, k0, klen;
  int tile;  // -1: none (the grid is an upper bound)
  int chunk;
};

// Item w of all sequences one after the other, the last tile (with the most keys to see) of each first, by
// one warp: 32 sequences at a time, with one round trip to memory for all of their four starts.
__device__ __forceinline__ Tile find_tile(const AttnParams &p, int w, int span) {
  const int lane = threadIdx.x & 31;
  Tile t = {0, 0, 0, 0, -1, 0};
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    int q0 = 0, q1 = 0, k0 = 0, k1 = 0, n = 0, chunks = 1;
    if (b0 + lane < p.batch) {
      seq_range(p.cu_q, b0 + lane, p.total_q, q0, q1);
      seq_range(p.cu_k, b0 + lane, p.total_k, k0, k1);
      chunks = chunks_of(p, k1 - k0);
      n = (q1 - q0 + span - 1) / span * chunks;
    }
    int sum = n;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, x);
      if (lane >= x) sum += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, w < sum);
    if (hit) {
      const int src = __ffs(hit) - 1;
      t.q0 = __shfl_sync(0xffffffffu, q0, src);
      t.qlen = __shfl_sync(0xffffffffu, q1, src) - t.q0;
      t.k0 = __shfl_sync(0xffffffffu, k0, src);
      t.klen = __shfl_sync(0xffffffffu, k1, src) - t.k0;
      const int back = __shfl_sync(0xffffffffu, sum, src) - 1 - w;
      chunks = __shfl_sync(0xffffffffu, chunks, src);
      t.tile = back / chunks;
      t.chunk = back % chunks;
      return t;
    }
    w -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return t;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

template <int DB, int TILES, bool FINE>
__global__ void __launch_bounds__(AttnCfg<DB, TILES>::THREADS, AttnCfg<DB, TILES>::CTAS)
    attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const AttnParams p) {
  using Cfg = AttnCfg<DB, TILES>;
  constexpr int S = Cfg::STAGES;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = ptx::smem_u32(smem);
  const uint32_t sQ = base + Cfg::HEAD, sKV = sQ + TILES * Cfg::TILE_BYTES;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem);
  const uint32_t full = ptx::smem_u32(bars);          // [S] keys or values landed
  const uint32_t empty = full + 8 * S;                // [S] the products that read them are done
  const uint32_t qfull = empty + 8 * S;               // [1] queries landed
  const uint32_t sfull = qfull + 8;                   // [TILES][2] scores ready
  const uint32_t pfull = sfull + 16 * TILES;          // [TILES][2] weights ready (and O rescaled)
  const uint32_t odone = pfull + 16 * TILES;          // [TILES] the last block but one is in the output
  const uint32_t ofull = odone + 8 * TILES;           // [TILES] the last one is
  int *misc = reinterpret_cast<int *>(bars + 2 * S + 1 + 6 * TILES);
  volatile int *abort_flag = misc;
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(misc + 1);
  Tile *found = reinterpret_cast<Tile *>(misc + 2);

  if (p.chunk > 0) ptx::grid_launch_dependents();  // attn_join_kernel
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (base & 1023u) {  // swizzle atoms would be off (the declaration asks for this alignment)
    if (threadIdx.x == 0) atomicCAS(p.status_word, 0u, 0x100u | kSiteAttnQ);
    return;
  }
  constexpr int kLoadWarp = Cfg::SOFTMAX_WARPS, kMmaWarp = kLoadWarp + 2;
  const int h = blockIdx.x % p.heads_kv;
  const int w = blockIdx.x / p.heads_kv;
  const int span = TILES * p.tile_q;  // queries of this CTA

  if (warp == 0) {
    const Tile t = find_tile(p, w, span);
    if (lane == 0) *found = t;
  } else if (warp == kLoadWarp) {
    if (lane == 0) {
      ptx::prefetch_tmap(&tmQ);
      ptx::prefetch_tmap(&tmK);
      ptx::prefetch_tmap(&tmV);
      *abort_flag = 0;
      for (int i = 0; i < S; ++i) {
        ptx::mbar_init(full + 8 * i, 1);
        ptx::mbar_init(empty + 8 * i, TILES);
      }
      ptx::mbar_init(qfull, 1);
      for (int i = 0; i < 2 * TILES; ++i) {
        ptx::mbar_init(sfull + 8 * i, 1);
        ptx::mbar_init(pfull + 8 * i, 4);
      }
      for (int i = 0; i < 2 * TILES; ++i) ptx::mbar_init(odone + 8 * i, 1);  // and ofull
      ptx::fence_mbar_init_cluster();
    }
  } else if (warp == kMmaWarp) {
    ptx::tmem_alloc<1>(ptx::smem_u32(tmem_holder), Cfg::TMEM_COLS);
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(tmem_holder);
  const Tile work = *found;
  const int q0 = work.q0, qlen = work.qlen, k0 = work.k0, klen = work.klen, qt = work.tile;
  // Blocks of 64 keys that tile i needs: [0, need_i); this CTA's share is [b0, b0 + count_i).
  auto need_of = [&](int i) {
    const int first = qt * span + i * p.tile_q;
    if (qt < 0 || first >= qlen) return 0;
    const int last = min(first + p.tile_q, qlen) - 1;
    const int seen = p.causal ? max(0, min(klen, last + 1 + klen - qlen)) : klen;
    return (seen + kBlock - 1) / kBlock;
  };
  const int need = max(need_of(0), need_of(TILES - 1));
  const bool whole = chunks_of(p, klen) == 1;  // nothing to join
  const int per = whole ? need : p.chunk;
  const int split = work.chunk, b0 = split * per;
  auto count_of = [&](int i) { return max(0, min(need_of(i) - b0, per)); };
  const int count0 = count_of(0), count1 = TILES == 2 ? count_of(1) : 0;
  const int count = max(count0, count1);
  const int items = (count + Cfg::LOAD - 1) / Cfg::LOAD * 2;  // loads: keys, values, keys, ..
  OpWait wc{abort_flag, p.status_word, p.timeout_ns};

  if (warp == kLoadWarp || warp == kLoadWarp + 1) {
    // A warp for the keys (and queries), one for the values, a lane for each 64-element block: a thread
    // is held about 400 cycles by a TMA load, and one thread for all of them kept the products waiting.
    const bool values = warp != kLoadWarp;
    if (count > 0) {
      if (!values) {
        // Both tiles' queries in one transaction (a tile without blocks is not read).
        if (lane == 0)
          ptx::mbar_arrive_expect_tx(qfull, ((count0 > 0) + (count1 > 0)) * DB * p.q_box_bytes);
        __syncwarp();
        const int i = lane / DB, x = lane % DB;
        if (i < TILES && (i == 0 ? count0 : count1) > 0)
          ptx::tma_load_3d(&tmQ, sQ + i * Cfg::TILE_BYTES + x * (kRows * 128), qfull, 64 * x,
                           h * p.group, q0 + qt * span + i * p.tile_q);
      }
      const CUtensorMap *map = values ? &tmV : &tmK;
      bool ok = true;
      int it = values ? 1 : 0;
      for (; it < items; it += 2) {
        const int st = it % S;
        int okw = 1;
        if (lane == 0) {
          if (it >= S) okw = op_wait(empty + 8 * st, (it / S - 1) & 1, wc, kSiteAttnKvEmpty);
          if (okw) ptx::mbar_arrive_expect_tx(full + 8 * st, Cfg::LOAD_BYTES);
        }
        ok = __shfl_sync(0xffffffffu, okw, 0) != 0;
        if (!ok) break;
        if (lane < DB)
          ptx::tma_load_3d(map, sKV + st * Cfg::LOAD_BYTES + lane * (Cfg::LOAD_ROWS * 128), full + 8 * st,
                           64 * lane, h, k0 + b0 * kBlock + (it >> 1) * Cfg::LOAD_ROWS);
      }
      if (!ok && lane == 0) {
        // Unwinding: the loads in flight land before the CTA may exit.
        if (!values) op_drain(qfull, 0);
        for (int j = max(it & 1, it - 2 * S); j < it; j += 2) op_drain(full + 8 * (j % S), (j / S) & 1);
      }
      __syncwarp();
    }
  } else if (warp >= kMmaWarp) {
    if (count > 0) {
      // A warp for each tile's products, so that one's waits lie under the other's work. The whole warp
      // walks the loop and one lane issues: descriptors then stay in uniform registers. (Walked by one
      // lane, a product took about 130 cycles to issue, twice its time on the tensor core.)
      const int i = __shfl_sync(0xffffffffu, warp - kMmaWarp, 0);
      const int cnt = i == 0 ? count0 : count1;
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t tmS = tm + 2 * i * kBlock, tmO = tm + Cfg::O_COL + i * (DB * 64);
      const uint32_t idesc_s = ptx::umma_idesc_f16_f32(kRows, kBlock, true);
      const uint32_t idesc_o = ptx::umma_idesc_f16_f32(kRows, p.dim16, false);
      const int ksteps = p.dim16 / 16;
      const bool one = ptx::elect_one();
      auto wait = [&](uint32_t bar, int phase, unsigned site) {
        return __all_sync(0xffffffffu, op_wait(bar, phase & 1, wc, site)) != 0;
      };
      auto commit = [&](uint32_t bar) {
        if (one) ptx::umma_commit<1>(bar);
      };
      // Scores of a block, into one of their two places; a 16-element step is 32 bytes of a 128-byte row,
      // the next 64 elements lie a block of rows on.
      const uint64_t qd = ptx::umma_desc_sw128(sQ + i * Cfg::TILE_BYTES, 16, 1024);
      auto scores = [&](int stage, int sub, int place) {
        const uint64_t kd =
            ptx::umma_desc_sw128(sKV + stage * Cfg::LOAD_BYTES + sub * (kBlock * 128), 16, 1024);
        if (one) {
#pragma unroll
          for (int k = 0; k < DB * 4; ++k)
            if (k < ksteps)
              ptx::umma_f16<1>(tmS + place * kBlock, qd + (k >> 2) * (kRows * 128 / 16) + (k & 3) * 2,
                               kd + (k >> 2) * (Cfg::LOAD_ROWS * 128 / 16) + (k & 3) * 2, idesc_s, k > 0);
          ptx::umma_commit<1>(sfull + 16 * i + 8 * place);
        }
      };
      auto output = [&](int stage, int sub, int place, bool first) {
        const uint64_t vd = ptx::umma_desc_sw128(sKV + stage * Cfg::LOAD_BYTES + sub * (kBlock * 128),
                                                 Cfg::LOAD_ROWS * 128, 1024);
        if (one) {
#pragma unroll
          for (int k = 0; k < kBlock / 16; ++k)
            ptx::umma_f16_ts(tmO, tmS + place * kBlock + 8 * k, vd + 128 * k, idesc_o, !(first && k == 0));
          if constexpr (FINE) {
#pragma unroll
            for (int k = 0; k < kBlock / 16; ++k)
              ptx::umma_f16_ts(tmO, tmS + place * kBlock + kBlock / 2 + 8 * k, vd + 128 * k, idesc_o, true);
          }
        }
      };
      // Load `item` lies in stage item % S; it is waited for and given back once by either tile's warp,
      // whether its tile needs it or not (a warp that is through must not give back a stage's next load
      // before this one is there). A stage that nothing is loaded into any more is not announced: no
      // arrival outlives the CTA.
      int st = 0, ph = 0;  // of the next item
      auto arrived = [&](int step) {
        int x = st + step, y = ph;
        if (x >= S) {
          x -= S;
          y ^= 1;
        }
        return wait(full + 8 * x, y, kSiteAttnKvFull);
      };
      auto give_back = [&](int item, int stage) {
        if (item + S < items) commit(empty + 8 * stage);
      };
      constexpr int LOAD = Cfg::LOAD;
      auto last_of_load = [&](int u) { return u % LOAD == LOAD - 1 || u + 1 == count; };
      bool ok = wait(qfull, 0, kSiteAttnQ) && arrived(0);
      if (ok) {
        ptx::tc_fence_after();
        if (cnt > 0) scores(0, 0, 0);
        if (last_of_load(0)) give_back(0, 0);
        constexpr int k1 = 2 * (1 / LOAD);  // load with the keys of block 1
        if (count > 1 && (ok = arrived(k1))) {
          ptx::tc_fence_after();
          if (cnt > 1) scores(k1, 1 % LOAD, 1);
          if (last_of_load(1)) give_back(k1, k1);
        }
      }
      st = 1;
#pragma unroll 1
      for (int u = 0; ok && u < count; ++u) {
        // The values of block u are load 2 (u / LOAD) + 1, at st; the keys of block u + 2 a few further.
        const int item = u / LOAD * 2 + 1;
        if (u % LOAD == 0 && !(ok = arrived(0))) break;
        const int place = u & 1;
        if (u < cnt) {
          if (!(ok = wait(pfull + 16 * i + 8 * place, u >> 1, kSiteAttnWeights))) break;
          ptx::tc_fence_after();
          output(st, u % LOAD, place, u == 0);
          if (u + 2 >= cnt) commit((u + 1 == cnt ? ofull : odone) + 8 * i);
        }
        if (last_of_load(u)) give_back(item, st);
        if (u + 2 < count) {
          constexpr int ahead = LOAD == 1 ? 3 : 1;
          if (u % LOAD == 0 && !(ok = arrived(ahead))) break;
          const int ks = st + ahead >= S ? st + ahead - S : st + ahead;
          // The next scores come behind the product that reads the weights in their place (the tensor
          // core works in issue order), and their announcement tells of that product too.
          if (u + 2 < cnt) {
            ptx::tc_fence_after();
            scores(ks, u % LOAD, place);
          }
          if (last_of_load(u + 2)) give_back(item + ahead, ks);
        }
        if (u % LOAD == LOAD - 1) {
          st += 2;
          if (st >= S) {
            st -= S;
            ph ^= 1;
          }
        }
      }
      if (!ok) {
        // Unwinding: every product retires before TMEM is freed.
        commit(ofull + 8 * i);
        op_drain(ofull + 8 * i, 0);
      }
      __syncwarp();
    }
  } else {
    // ---------------------------------------------------------------- softmax warps
    const int i = warp >> 2;
    const int row = threadIdx.x & 127;
    const int first = qt * span + i * p.tile_q;
    const int n = i == 0 ? count0 : count1;
    const int qi = first + row / p.group;  // query of this row, inside the sequence
    const bool live = qt >= 0 && row < p.tile_q * p.group && qi < qlen;
    // A warp whose 32 rows are no query's (single tokens fill one of the four) only keeps step.
    const bool idle = !__any_sync(0xffffffffu, live);
    const int limit = p.causal ? max(0, min(klen, qi + 1 + klen - qlen)) : klen;
    const uint32_t lane_base = static_cast<uint32_t>(warp & 3) << 21;  // 32 lanes a warp, lane << 16
    const uint32_t tS = tmem + lane_base + i * (2 * kBlock);
    const uint32_t tO = tmem + lane_base + Cfg::O_COL + i * (DB * 64);
    float m = -INFINITY;  // what the weights are relative to (scaled): a maximum less kRaise
    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};  // of the weights, in four parts
    bool ok = true;
    auto wait = [&](uint32_t bar, int phase, unsigned site) {
      int okw = 1;
      if (lane == 0) okw = op_wait(bar, phase & 1, wc, site);
      okw = __shfl_sync(0xffffffffu, okw, 0);
      ptx::tc_fence_after();
      return okw != 0;
    };
#pragma unroll 1
    for (int u = 0; u < n; ++u) {
      const uint32_t place = tS + (u & 1) * kBlock;
      if (!(ok = wait(sfull + 16 * i + 8 * (u & 1), u >> 1, kSiteAttnScores))) break;
      if (idle) {  // whatever stands in its rows of the weights stays in its rows of the output
        if (lane == 0) ptx::mbar_arrive(pfull + 16 * i + 8 * (u & 1));
        continue;
      }
      uint32_t sr[2][32];
      ptx::tmem_ld_32x32b_x32(place, sr[0]);
      ptx::tmem_ld_32x32b_x32(place + 32, sr[1]);
      ptx::tmem_ld_wait();
      const int left = limit - (b0 + u) * kBlock;  // keys of this block that the row sees
      if (__any_sync(0xffffffffu, left < kBlock)) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * c + e >= left) sr[c][e] = 0xff800000u;  // -infinity
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], __uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale2;
      const bool grow = top > m + (kRaise + kLag);  // true of the first key, from -infinity
      const float m_old = m;
      if (grow) m = top - kRaise;
      if (u > 0 && __any_sync(0xffffffffu, grow)) {
        // O comes to rest with the block before: the scores behind this block's are formed after it.
        if (!(ok = u + 1 < n ? wait(sfull + 16 * i + 8 * ((u + 1) & 1), (u + 1) >> 1, kSiteAttnScores)
                             : wait(odone + 8 * i, 0, kSiteAttnOut)))
          break;
        const float f = (grow && m_old != -INFINITY) ? ex2(m_old - m) : 1.0f;
        sum[0].x *= f;
        sum[0].y *= f;
        sum[1].x *= f;
        sum[1].y *= f;
#pragma unroll 1
        for (int c = 0; c < DB * 4; ++c) {
          uint32_t o[16];
          ptx::tmem_ld_32x32b_x16(tO + 16 * c, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          ptx::tmem_st_32x32b_x16(tO + 16 * c, o);
        }
      }
      const float neg1 = m == -INFINITY ? 0.0f : -m;
      const float2 neg = make_float2(neg1, neg1), scale = make_float2(p.scale2, p.scale2);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w2[16], rest[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 x = __ffma2_rn(
              make_float2(__uint_as_float(sr[c][2 * e]), __uint_as_float(sr[c][2 * e + 1])), scale, neg);
          const float2 ab = make_float2(ex2(x.x), ex2(x.y));
          sum[e & 1] = __fadd2_rn(sum[e & 1], ab);
          const __half2 h2 = __float22half2_rn(ab);
          w2[e] = *reinterpret_cast<const uint32_t *>(&h2);
          if constexpr (FINE) {
            const float2 up = __half22float2(h2);
            const __half2 r2 = __float22half2_rn(__fadd2_rn(ab, make_float2(-up.x, -up.y)));
            rest[e] = *reinterpret_cast<const uint32_t *>(&r2);
          }
        }
        ptx::tmem_st_32x32b_x16(place + 16 * c, w2);
        if constexpr (FINE) ptx::tmem_st_32x32b_x16(place + kBlock / 2 + 16 * c, rest);
      }
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(pfull + 16 * i + 8 * (u & 1));
    }
    if (ok && n > 0) ok = wait(ofull + 8 * i, 0, kSiteAttnOut);
    if (ok && !idle) {
      const int kb = b0 * kBlock;                                  // first key of this CTA
      const int ke = min(limit, kb + n * kBlock);                  // behind the last that the row sees
      const bool any = ke > kb;
      const long long orow =
          static_cast<long long>(q0 + qi) * p.heads_q + h * p.group + row % p.group;
      const float l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      const float inv1 = any ? 1.0f / l : 0.0f;
      const float2 inv = make_float2(inv1, inv1), zero = make_float2(0.0f, 0.0f);
      const bool clear = !__all_sync(0xffffffffu, any);  // rows without a key: zeros, whatever stands in O
      float2 check[2] = {zero, zero};  // stays 0 with finite outputs, NaN otherwise
      uint8_t *stage = smem + Cfg::HEAD + i * Cfg::TILE_BYTES;
      float *part = p.part_o + (static_cast<long long>(split) * p.total_q * p.heads_q + orow) * p.dim16;
#pragma unroll
      for (int c = 0; c < DB * 2; ++c) {
        const int col = 32 * c;
        if (col >= p.dim16) break;
        uint32_t o[32];
        if (n > 0) {
          ptx::tmem_ld_32x32b_x32(tO + col, o);
          ptx::tmem_ld_wait();
        }
        float2 f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          f[e] = __fmul2_rn(make_float2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1])), inv);
          if (clear && !any) f[e] = zero;
          // (columns behind dim16 hold nothing)
          if (e < 8 || col + 16 < p.dim16) check[e & 1] = __ffma2_rn(f[e], zero, check[e & 1]);
        }
        if (whole) {
          // Through the tile's own query buffer (its last product has retired), so that rows leave
          // in whole 16-byte groups next to each other.
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const __half2 ab = __float22half2_rn(f[4 * g + x]);
              w[x] = *reinterpret_cast<const uint32_t *>(&ab);
            }
            const int grp = col / 8 + g;
            *reinterpret_cast<uint4 *>(stage + (grp >> 3) * (kRows * 128) + row * 128 +
                                       (((grp & 7) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else if (live && any) {
#pragma unroll
          for (int g = 0; g < 8; ++g)
            if (g < 4 || col + 16 < p.dim16)
              *reinterpret_cast<float4 *>(part + col + 4 * g) =
                  make_float4(f[2 * g].x, f[2 * g].y, f[2 * g + 1].x, f[2 * g + 1].y);
        }
      }
      const float chk = (check[0].x + check[0].y) + (check[1].x + check[1].y);
      const bool odd = any && !(chk == 0.0f && l > 0.0f && l < INFINITY);
      float lse2 = any ? m + log2f(l) : -INFINITY;
      if (whole) {
        __syncwarp();
        // 8 or 16 lanes write a row; where it goes, its own lane knows.
        __half *to = p.out + (q0 + qi) * p.out_stride +
                     static_cast<long long>(h * p.group + row % p.group) * p.head_dim;
        if (!live) to = nullptr;
        constexpr int wide = DB * 8;
        const int grp = lane % wide;
#pragma unroll 4
        for (int r0 = 0; r0 < 32; r0 += 32 / wide) {
          const int r = r0 + lane / wide, rr = (row & ~31) + r;
          __half *dst = reinterpret_cast<__half *>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), r));
          if (dst && 8 * grp < p.head_dim)
            *reinterpret_cast<uint4 *>(dst + 8 * grp) = *reinterpret_cast<const uint4 *>(
                stage + (grp >> 3) * (kRows * 128) + rr * 128 + (((grp & 7) ^ (rr & 7)) << 4));
        }
      }
      __syncwarp();
      // Infinities or NaN: a masked place of the block may have reached the row (0 times infinity
      // is NaN in the second product), or the row sees one. Done again over the keys it sees alone.
      for (unsigned todo = __ballot_sync(0xffffffffu, live && odd); todo; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        const int r = (row & ~31) + src, q = first + r / p.group;
        const int end = __shfl_sync(0xffffffffu, ke, src);
        const int head = h * p.group + r % p.group;
        const RowSum sum1 =
            attn_row(p.q + (q0 + q) * p.q_stride + static_cast<long long>(head) * p.head_dim,
                     p.k + k0 * p.k_stride + static_cast<long long>(h) * p.head_dim,
                     p.v + k0 * p.v_stride + static_cast<long long>(h) * p.head_dim, p.k_stride, p.v_stride,
                     p.head_dim, p.scale2, kb, end);
        // (a range of -infinity alone is handed over as it stands: zeros, or NaN of an infinite value)
        const float ir = !whole && sum1.l == 0.0f ? 1.0f : 1.0f / sum1.l;
        if (4 * lane < p.head_dim) {
          const float4 f = make_float4(sum1.o.x * ir, sum1.o.y * ir, sum1.o.z * ir, sum1.o.w * ir);
          if (whole) {
            const __half2 a = __floats2half2_rn(f.x, f.y);
            const __half2 b = __floats2half2_rn(f.z, f.w);
            *reinterpret_cast<uint2 *>(p.out + (q0 + q) * p.out_stride +
                                       static_cast<long long>(head) * p.head_dim + 4 * lane) =
                make_uint2(*reinterpret_cast<const uint32_t *>(&a),
                           *reinterpret_cast<const uint32_t *>(&b));
          } else {
            float *dst = p.part_o + (static_cast<long long>(split) * p.total_q * p.heads_q +
                                     static_cast<long long>(q0 + q) * p.heads_q + head) * p.dim16;
            *reinterpret_cast<float4 *>(dst + 4 * lane) = f;
          }
        }
        if (lane == src) lse2 = !whole && sum1.l == 0.0f ? kAllMinusInf : sum1.m + log2f(sum1.l);
      }
      if (live) {
        if (!whole)
          p.part_lse[static_cast<long long>(split) * p.total_q * p.heads_q + orow] = lse2;
        else if (p.lse)
          p.lse[orow] = lse2 * 0.69314718055994530942f;
      }
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, Cfg::TMEM_COLS);
  }
}

// Joins the key ranges of a row: one warp for each (query, head).
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnParams p) {
  const long long rows = static_cast<long long>(p.total_q) * p.heads_q;
  const long long row = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (row >= rows) {
    ptx::grid_wait();
    return;
  }
  const int i = static_cast<int>(row / p.heads_q), h = static_cast<int>(row % p.heads_q);
  // Ranges of the row's sequence; rows of no sequence are left as they were.
  int mine = 0;
  for (int b = lane; b < p.batch; b += 32) {
    int q0, q1, k0, k1;
    seq_range(p.cu_q, b, p.total_q, q0, q1);
    seq_range(p.cu_k, b, p.total_k, k0, k1);
    if (i >= q0 && i < q1) mine = chunks_of(p, k1 - k0);
  }
  const int chunks = __reduce_max_sync(0xffffffffu, mine);
  ptx::grid_wait();
  if (chunks <= 1) return;  // written by its only CTA
  // A lane holds the sums of ranges lane, lane + 32, .. .
  constexpr int kEach = kMaxChunks / 32;
  float z[kEach], top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int x = 0; x < kEach; ++x) {
    const int c = lane + 32 * x;
    z[x] = c < chunks ? p.part_lse[c * rows + row] : -INFINITY;
    nan |= z[x] != z[x];
    top = fmaxf(top, z[x]);
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  if (__any_sync(0xffffffffu, nan)) top = __int_as_float(0x7fffffff);
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, l = 0.0f;
  if (top != -INFINITY) {
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
      if (32 * x >= chunks) break;
      const float f = z[x] == -INFINITY ? 0.0f : z[x] == top ? 1.0f : exp2f(z[x] - top);
      const unsigned used = __ballot_sync(0xffffffffu, z[x] != -INFINITY);
      const int end = min(32, chunks - 32 * x);
#pragma unroll 8
      for (int c = 0; c < end; ++c) {
        // (a range without keys for this row has written no output)
        const float fc = __shfl_sync(0xffffffffu, f, c);
        if (((used >> c) & 1u) == 0) continue;
        l += fc;
        if (4 * lane < p.head_dim) {
          const float4 v = *reinterpret_cast<const float4 *>(
              p.part_o + ((c + 32 * x) * rows + row) * p.dim16 + 4 * lane);
          o[0] = fmaf(fc, v.x, o[0]);
          o[1] = fmaf(fc, v.y, o[1]);
          o[2] = fmaf(fc, v.z, o[2]);
          o[3] = fmaf(fc, v.w, o[3]);
        }
      }
    }
  }
  const bool none = top == kAllMinusInf;
  const float inv = none ? __int_as_float(0x7fffffff) : l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
  if (4 * lane < p.head_dim) {
    const __half2 a = __floats2half2_rn(o[0] * inv, o[1] * inv);
    const __half2 b = __floats2half2_rn(o[2] * inv, o[3] * inv);
    *reinterpret_cast<uint2 *>(p.out + i * p.out_stride + static_cast<long long>(h) * p.head_dim +
                               4 * lane) = make_uint2(*reinterpret_cast<const uint32_t *>(&a),
                                                      *reinterpret_cast<const uint32_t *>(&b));
  }
  if (lane == 0 && p.lse) p.lse[row] = none ? -INFINITY : (top + log2f(l)) * 0.69314718055994530942f;
}

// ------------------------------------------------------------------------------ host side
// How a call is run: depends on the sizes alone, so that the workspace does.
struct AttnPlan {
  int tiles;       // row tiles of a CTA
  int tile_q;      // queries of a row tile
  bool fine;       // weights of 22 bits
  int chunk, max_chunks;
  long long items;  // upper bound of (tile, key range) pairs of all sequences
  size_t workspace;
};

AttnPlan make_plan(int total_q, int total_k, int batch, int heads_q, int heads_kv, int head_dim) {
  AttnPlan pl;
  const int group = heads_q / heads_kv;
  pl.tile_q = kRows / group;
  const long long avg_q = (total_q + batch - 1ll) / batch, avg_k = (total_k + batch - 1ll) / batch;
  // Two row tiles to a CTA share the loaded keys, one tile each to two CTAs of an SM lets one's start
  // and end lie under the other's work: measured equal near 6000 keys a sequence at head_dim 128 (4 x 2048
  // tokens 174 and 166 us, 8192 tokens 475 and 495, 16384 tokens 1.89 and 2.06 ms), in favour of
  // one tile at head_dim 64 up to 8192.
  pl.tiles = head_dim > 64 && avg_k >= 6144 && avg_q > pl.tile_q ? 2 : 1;
  // Weights rounded to binary16 leave as much error in an output as its own rounding does, together 1.4 times the
  // latter; with 22 bits the output's own is left. A choice between that and time: small calls, whose few outputs do
  // not average their errors either (1.53 times, 6 rows of 96 seen), take it at 5% (one token over 131072
  // keys 124 us against 118); larger ones do not (16 tokens of 32 heads 106 us instead of 99, a dozen prompts 141 for 122).
  pl.fine = static_cast<long long>(total_q) * heads_q <= 128;
  const int span = pl.tiles * pl.tile_q;
  const long long max_tiles = std::min<long long>(total_q, total_q / span + static_cast<long long>(batch));
  // Key ranges where there are few tiles: of single tokens (whose lengths set the pace) up to two
  // waves of CTAs, of prompts up to half a wave, beyond which writing and joining the parts costs more
  // than the idle SMs. As many as fill one wave at the mean length (longer sequences get more), of 256 keys
  // at least: one token over 2000 keys 12.9 us with 256, 14.2 with 128, 20.0 with 1024; over 131072 keys 97.5
  // us with one wave of ranges, 124 with four shorter ones to a slot, whose starts then cost more than the
  // wave's uneven end.
  const long long slots = kSms * (pl.tiles == 1 ? 2 : 1);
  const long long est_tiles = std::max<long long>((total_q + span - 1) / span, batch);
  const long long units = est_tiles * heads_kv;
  const long long blocks = total_k / kBlock + static_cast<long long>(batch);  // >= those of all sequences
  pl.chunk = 0;
  pl.max_chunks = 1;
  pl.items = max_tiles;
  if (avg_q <= pl.tile_q ? units < 2 * slots : 2 * units <= slots) {
    const long long ranges = std::max<long long>(1, slots / units);  // of a sequence, in one wave
    long long chunk = std::max<long long>(4, (blocks / batch + ranges - 1) / ranges);
    chunk = std::max(chunk, (blocks + kMaxChunks - 1) / kMaxChunks);
    const long long chunks = (blocks + chunk - 1) / chunk;
    if (chunks > 1) {
      pl.chunk = static_cast<int>(chunk);
      pl.max_chunks = static_cast<int>(chunks);
      pl.items = max_tiles + (total_q + span - 1) / span * chunks;
    }
  }
  pl.workspace = 0;
  if (pl.chunk > 0) {
    const size_t rows = static_cast<size_t>(pl.max_chunks) * total_q * heads_q;
    pl.workspace = rows * ((head_dim + 15) / 16 * 16) * sizeof(float) + rows * sizeof(float);
  }
  return pl;
}

int check(const hgemm_attn_prompt_t *a) {
  if (!a || a->total_q < 0 || a->total_k < 0 || a->batch < 0) return HGEMM_ERR_INVALID_ARG;
  if (a->heads_kv < 1 || a->heads_q < a->heads_kv || a->heads_q % a->heads_kv != 0 ||
      a->heads_q / a->heads_kv > 128)
    return HGEMM_ERR_INVALID_ARG;
  if (a->head_dim < 8 || a->head_dim > kMaxDim || a->head_dim % 8 != 0)
    return HGEMM_ERR_INVALID_ARG;
  const float scale2 = a->scale * kLog2e;
  if (!(a->scale >= 0.0f) || scale2 - scale2 != 0.0f) return HGEMM_ERR_INVALID_ARG;
  if (a->total_q > kOpMaxRows || a->total_k > kOpMaxRows || a->batch > kOpMaxRows)
    return HGEMM_ERR_TOO_LARGE;
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
  for (const long long stride : {a->q_stride, a->out_stride, a->k_stride, a->v_stride})
    if (stride % 8 || stride > kOpMaxStride) return HGEMM_ERR_INVALID_ARG;
  const size_t need = hgemm_attn_prompt_workspace_bytes(a->total_q, a->total_k, a->batch, a->heads_q,
                                                        a->heads_kv, a->head_dim);
  if (need > 0 && (!a->workspace || !op_aligned16(a->workspace) || a->workspace_bytes < need))
    return HGEMM_ERR_INVALID_ARG;
  const OpRows in[] = {op_heads(a->q, a->heads_q, a->head_dim, a->q_stride, a->total_q),
                       op_heads(a->k, a->heads_kv, a->head_dim, a->k_stride, a->total_k),
                       op_heads(a->v, a->heads_kv, a->head_dim, a->v_stride, a->total_k),
                       op_dense(a->cu_q, 4, a->batch + 1), op_dense(a->cu_k, 4, a->batch + 1)};
  const OpRows out[] = {op_heads(a->out, a->heads_q, a->head_dim, a->out_stride, a->total_q),
                        op_dense(a->lse, 4, a->total_q, a->heads_q),
                        op_dense(a->workspace, 1, static_cast<double>(need))};
  bool over = op_overlap(out[0], out[1]) || op_overlap(out[0], out[2]) || op_overlap(out[1], out[2]);
  for (const OpRows &o : out)
    for (const OpRows &i : in) over |= op_overlap(o, i);
  return over ? HGEMM_ERR_INVALID_ARG : HGEMM_OK;
}

template <int DB, int TILES, bool FINE>
int launch(const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const AttnParams &p,
           const OpDevice &d, long long ctas, cudaStream_t stream) {
  using Cfg = AttnCfg<DB, TILES>;
  static unsigned done[64];
  const int st = op_smem(reinterpret_cast<const void *>(attn_kernel<DB, TILES, FINE>), Cfg::SMEM, d.dev, done);
  if (st != HGEMM_OK) return st;
  attn_kernel<DB, TILES, FINE>
      <<<static_cast<unsigned>(ctas), Cfg::THREADS, Cfg::SMEM, stream>>>(tq, tk, tv, p);
  return cudaGetLastError() == cudaSuccess ? HGEMM_OK : HGEMM_ERR_LAUNCH;
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
  // scale 0 is a plain mean: any tiny factor gives it without 0 times the masked -infinity.
  p.scale2 = std::max(a->scale * kLog2e, 1e-37f);
  p.dim16 = (a->head_dim + 15) / 16 * 16;
  p.status_word = d.status_word;
  p.timeout_ns = d.timeout_ns;
  const AttnPlan pl = make_plan(a->total_q, a->total_k, a->batch, a->heads_q, a->heads_kv, a->head_dim);
  p.tile_q = pl.tile_q;
  p.q_box_bytes = pl.tile_q * p.group * 128;
  p.chunk = pl.chunk;
  p.max_chunks = pl.max_chunks;
  p.part_o = static_cast<float *>(a->workspace);
  p.part_lse = p.part_o + static_cast<size_t>(pl.max_chunks) * a->total_q * a->heads_q * p.dim16;

  CUtensorMap tq, tk, tv;
  auto encode = [&](CUtensorMap *map, const void *ptr, int heads, int rows, long long stride,
                    int box_heads, int box_rows) {
    const unsigned long long dims[3] = {static_cast<unsigned long long>(a->head_dim),
                                        static_cast<unsigned long long>(heads),
                                        static_cast<unsigned long long>(rows)};
    const unsigned long long strides[2] = {static_cast<unsigned long long>(a->head_dim) * 2,
                                           static_cast<unsigned long long>(stride) * 2};
    const unsigned box[3] = {64, static_cast<unsigned>(box_heads), static_cast<unsigned>(box_rows)};
    return op_encode(map, ptr, 3, dims, strides, box);
  };
  if (!encode(&tq, a->q, a->heads_q, a->total_q, a->q_stride, p.group, pl.tile_q))
    return HGEMM_ERR_TENSOR_MAP;
  if (a->total_k > 0) {
    if (!encode(&tk, a->k, a->heads_kv, a->total_k, a->k_stride, 1, pl.tiles * kBlock) ||
        !encode(&tv, a->v, a->heads_kv, a->total_k, a->v_stride, 1, pl.tiles * kBlock))
      return HGEMM_ERR_TENSOR_MAP;
  } else {
    tk = tv = tq;  // no key: never loaded from
  }
  const long long ctas = pl.items * a->heads_kv;
  const long long joins = (static_cast<long long>(a->total_q) * a->heads_q + 7) / 8;
  if (ctas > 0x7fffffffll || joins > 0x7fffffffll) return HGEMM_ERR_TOO_LARGE;
  if (a->head_dim <= 64)
    st = pl.fine ? launch<1, 1, true>(tq, tk, tv, p, d, ctas, stream)
                 : launch<1, 1, false>(tq, tk, tv, p, d, ctas, stream);
  else if (pl.tiles == 1)
    st = pl.fine ? launch<2, 1, true>(tq, tk, tv, p, d, ctas, stream)
                 : launch<2, 1, false>(tq, tk, tv, p, d, ctas, stream);
  else
    st = launch<2, 2, false>(tq, tk, tv, p, d, ctas, stream);
  if (st != HGEMM_OK || pl.chunk == 0) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(joins), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, attn_join_kernel, p) != cudaSuccess) {
    cudaGetLastError();
    return HGEMM_ERR_LAUNCH;
  }
  return HGEMM_OK;
}

}  // namespace
}  // namespace hgemm

extern "C" {

int hgemm_attn_prompt(const hgemm_attn_prompt_t *args, hgemm_stream_t stream) {
  return hgemm::op_status(hgemm::run(args, stream));
}

size_t hgemm_attn_prompt_workspace_bytes(int total_q, int total_k, int batch, int heads_q,
                                         int heads_kv, int head_dim) {
  if (total_q <= 0 || total_k < 0 || batch <= 0 || heads_kv < 1 || heads_q < heads_kv ||
      heads_q % heads_kv != 0 || heads_q / heads_kv > hgemm::kRows || head_dim < 8 ||
      head_dim > hgemm::kMaxDim || head_dim % 8 != 0 || total_q > hgemm::kOpMaxRows ||
      total_k > hgemm::kOpMaxRows || batch > hgemm::kOpMaxRows)
    return 0;
  return hgemm::make_plan(total_q, total_k, batch, heads_q, heads_kv, head_dim).workspace;
}

}  // extern "C"
