// Attention of longer chunks over a paged cache: tiles of 256 query rows on
// the tensor cores.
//
// Bound by the MMAs (4 * 256 * 128 * D flops per 128-key tile of a unit against
// 2 * 128 * D cache elements).  The pipeline is that of attn_kv.cuh: a cluster
// of two CTAs shares every tcgen05 MMA (cta_group::2: each CTA holds 128 query
// rows, half of each K tile's keys and half of each V tile's columns), scores
// and probabilities live in TMEM, two softmax warpgroups per CTA own a row half
// each and rescale O lazily.  What differs:
//   * Units come from the plan (chunk_plan.cuh): any mix of sequences, each pair
//     walking an equal range of the batch's steps.
//   * K and V are read from pages of any multiple of 16 tokens, through the
//     sequence's table, box by box.
//   * Rows are (token, query head) pairs of a strided Q, gathered by the
//     converter warps instead of TMA; each row sees keys up to its position.
//   * bf16 caches land in operand layout straight from TMA; the converter warps
//     only pass the tile on (and clear V rows past the sequence, which may hold
//     anything: 0 * NaN would reach every row).
//   * An e4m3 cache that many query tiles read is expanded into a bf16 copy first
//     (chunk_expand_kernel; exact, scales included), when the copy is of moderate
//     size: reading it in place converts every key tile again for each 256 rows.
//   * Scaled e4m3 caches: K's 2^e multiplies the scores of its key, V's 2^e the
//     weights, and the softmax reference is kept above score + V exponent, as in
//     chunk_rows.cuh.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include "attn_common.cuh"
#include "attn_softmax.cuh"
#include "chunk_plan.cuh"
#include "conv_geo.cuh"

namespace pcp {

enum : int { kCacheBf16 = 0, kCacheE4m3 = 1, kCacheScaled = 2 };

constexpr int kTilesConvWarps = 4;
constexpr int kTilesConvThreads = 32 * kTilesConvWarps;
constexpr int kTilesConvWarp0 = kMmaWarp + 1;
constexpr int kTilesThreads = kThreads + kTilesConvThreads;  // 448
constexpr uint16_t kChunkBothCtas = 3, kChunkLeader = 1;

template <int D, int kCache>
struct TilesSmem {
  static constexpr bool kFp8 = kCache != kCacheBf16;
  static constexpr int kQBytes = D * 2 * kTileM;
  static constexpr int kOpBytes = 128 * D;  // 16-bit K half [64, D] or V half [128, D/2], swizzled
  static constexpr int kRawBytes = 64 * D;  // e4m3 K half [64][D] or V half [128][D/2]
  static constexpr int kOpStages = kFp8 ? (D == 256 ? 3 : 8) : (D == 256 ? 5 : 11);
  static constexpr int kRawStages = kFp8 ? (D == 256 ? 3 : 6) : 0;
  static constexpr int kLandStages = kFp8 ? kRawStages : kOpStages;  // stages the TMA fills
  static constexpr int kKBox = 64 * 128;
  static constexpr int kVBox = 128 * 128;
  // A tile's scales are rewritten once its P has been consumed: K of tile J + k
  // is converted after item 2 (J + k) - 1 - kOpStages was consumed, V of tile J
  // is item 2 J + 2.
  static constexpr int kScaleBufs = kCache == kCacheScaled ? (kOpStages + 4) / 2 : 0;
  static constexpr int kOpOff = kQBytes;
  static constexpr int kRawOff = kOpOff + kOpStages * kOpBytes;
  static constexpr int kScaleOff = kRawOff + kRawStages * kRawBytes;  // float k[128], v[128], int vmax[4]
  static constexpr int kScaleBuf = 2 * kTileN * 4 + 16;
  static constexpr int kFactorOff = kScaleOff + kScaleBufs * kScaleBuf;  // float[2][128], by segment parity
  static constexpr int kRedOff = kFactorOff + (kFp8 ? 2 * kTileM * 4 : 0);
  static constexpr int kBarOff = kRedOff + 2 * kSoftmaxWarpgroups * kTileM * 4;
  // q_ready, q_empty, rows[2], land_full[NL], land_empty[NR], op_full[NS],
  // op_empty[NS], s_full[2], p_full[2], o_done[2], teardown, red[2], scale[NB]
  static constexpr int kNumBars = 4 + kLandStages + kRawStages + 2 * kOpStages + 9 + kScaleBufs;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kPlanOff = kMiscOff + 16;  // ChunkPlanShared
  static constexpr int kBytes = kPlanOff + sizeof(ChunkPlanShared);
  static_assert(kBytes <= 232448, "exceeds the 227 KB of shared memory per CTA");
  static_assert(kRawOff % 1024 == 0 && kScaleOff % 16 == 0 && kBarOff % 8 == 0, "alignment");
};

// The pages of sequences with tile units as bf16, page lb of sequence s at block
// s * table_width + lb of `copy`, in the payload's layout.  Bound by HBM (1 byte
// read, 2 written an element); a block takes the rows of one head of K or V of a
// page at a time.
struct ExpandParams {
  ChunkParams c;
  __nv_bfloat16* copy;
};

template <int D>
__global__ void __launch_bounds__(256) chunk_expand_kernel(const ExpandParams p) {
  constexpr int kPerRow = D / 16;
  const PoolView& pool = p.c.pool;
  const int per_page = 2 * pool.heads;
  const long long items = static_cast<long long>(p.c.batch.seqs) * p.c.batch.table_width * per_page;
  __shared__ int s_ignored;  // lengths the attention reports itself
  if (threadIdx.x == 0) s_ignored = 0;
  __syncthreads();
  for (long long it = blockIdx.x; it < items; it += gridDim.x) {
    const long long page = it / per_page;
    const int which = static_cast<int>(it - page * per_page);
    const int s = static_cast<int>(page / p.c.batch.table_width), lb = static_cast<int>(page - static_cast<long long>(s) * p.c.batch.table_width);
    const ChunkSeq q = chunk_seq<true>(p.c, s, &s_ignored);
    const int n = min(pool.block_size, q.kvlen - lb * pool.block_size);
    if (q.tiles == 0 || n <= 0) continue;
    const int blk = p.c.batch.tables[s * p.c.batch.table_stride + lb];
    const bool found = blk >= 0 && blk < pool.blocks;
    if (!found && threadIdx.x == 0) atomicCAS(p.c.status, 0, kErrBlockTable);
    const long long src = (static_cast<long long>(found ? blk : 0) * per_page + which) * pool.block_size;
    const uint4* codes = reinterpret_cast<const uint4*>(pool.data + src * D);
    const uint8_t* scales = pool.scales ? pool.scales + src : nullptr;
    uint4* dst = reinterpret_cast<uint4*>(p.copy + (page * per_page + which) * pool.block_size * D);
    for (int e0 = threadIdx.x; e0 < n * kPerRow; e0 += 4 * 256) {
      uint4 x[4];
      uint32_t sc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = e0 + u * 256;
        x[u] = make_uint4(0u, 0u, 0u, 0u);
        sc[u] = 127;
        if (found && e < n * kPerRow) {
          x[u] = codes[e];
          if (scales) sc[u] = scales[e / kPerRow];
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = e0 + u * 256;
        if (e >= n * kPerRow) break;
        uint4 o[2];
        e4m3x16_to_bf16(x[u], sc[u], o);
        dst[2 * e] = o[0];
        dst[2 * e + 1] = o[1];
      }
    }
  }
}

template <int D, int kCache>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTilesThreads, 1)
    chunk_tiles_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const int box_rows, const ChunkParams p) {
  using L = TilesSmem<D, kCache>;
  constexpr bool kFp8 = L::kFp8;
  constexpr bool kScaled = kCache == kCacheScaled;
  constexpr int NS = L::kOpStages, NL = L::kLandStages, NR = L::kRawStages, NB = L::kScaleBufs;

  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  if (sbase & 1023u) {  // identical in both CTAs: neither starts
    if (threadIdx.x == 0) {
      p.work.tile_rec[blockIdx.x].err = kErrSmemAlign;
      clear_record(p.work.tile_rec[blockIdx.x >> 1]);
    }
    return;
  }
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const uint32_t sQ = sbase;
  const uint32_t sOp = sbase + L::kOpOff;
  const uint32_t sRaw = sbase + L::kRawOff;
  const uint32_t bars = sbase + L::kBarOff;
  const uint32_t bar_q_ready = bars;      // leader: Q written in both CTAs (one arrive per converter warp)
  const uint32_t bar_q_empty = bars + 8;  // the segment's last QK^T has read Q (MMA commit, both CTAs)
  // This CTA's row factors written, by segment parity (two: the converters may
  // be a segment ahead of a softmax warp that has not waited yet).
  auto bar_rows = [&](int s) { return bars + 16 + 8u * (s & 1); };
  auto bar_land_full = [&](int s) { return bars + 8u * (4 + s); };
  auto bar_land_empty = [&](int s) { return bars + 8u * (4 + NL + s); };
  auto bar_op_full = [&](int s) { return bars + 8u * (4 + NL + NR + s); };
  auto bar_op_empty = [&](int s) { return bars + 8u * (4 + NL + NR + NS + s); };
  constexpr int kB2 = 4 + NL + NR + 2 * NS;
  auto bar_s_full = [&](int b) { return bars + 8u * (kB2 + b); };
  auto bar_p_full = [&](int b) { return bars + 8u * (kB2 + 2 + b); };
  auto bar_o = [&](int b) { return bars + 8u * (kB2 + 4 + b); };
  const uint32_t bar_td = bars + 8u * (kB2 + 6);
  auto bar_red = [&](int b) { return bars + 8u * (kB2 + 7 + b); };
  auto bar_scale = [&](int b) { return bars + 8u * (kB2 + 9 + b); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  float* red = reinterpret_cast<float*>(smem + L::kRedOff);
  float* factors = reinterpret_cast<float*>(smem + L::kFactorOff);

  ChunkPlanShared& plan = *reinterpret_cast<ChunkPlanShared*>(smem + L::kPlanOff);
  int* err = &plan.err;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (warp == kProducerWarp && lane == 0) {
    mbar_init(bar_q_ready, 2 * kTilesConvWarps);
    mbar_init(bar_q_empty, 1);
    mbar_init(bar_rows(0), kTilesConvWarps);
    mbar_init(bar_rows(1), kTilesConvWarps);
    for (int s = 0; s < NL; ++s) mbar_init(bar_land_full(s), 1);
    for (int s = 0; s < NR; ++s) mbar_init(bar_land_empty(s), kTilesConvWarps);
    for (int s = 0; s < NS; ++s) {
      mbar_init(bar_op_full(s), 2 * kTilesConvWarps);
      mbar_init(bar_op_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_s_full(b), 1);
      mbar_init(bar_p_full(b), 2 * kSoftmaxThreads / 32);  // one arrive per softmax warp of both CTAs
      mbar_init(bar_o(b), 1);
      mbar_init(bar_red(b), kSoftmaxThreads);
    }
    for (int b = 0; b < NB; ++b) mbar_init(bar_scale(b), kTilesConvWarps);
    mbar_init(bar_td, 1);
    *abort_flag = 0;
    plan.err = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc_pair(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // barriers of both CTAs initialised, TMEM allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int pair = blockIdx.x >> 1;
  grid_launch_dependents();  // the merge may wait on the SMs
  chunk_plan<true>(p, plan, p.tile_pairs, pair);

  // Calls body(unit, kt0, kt1) for each part of this pair's range until
  // it returns false; returns false if it did.
  auto for_each_segment = [&](auto&& body) -> bool {
    ChunkWalk<true> walk;
    walk.init(plan);
    ChunkUnit un;
    int kt0, kt1;
    while (walk.next(p, err, un, kt0, kt1))
      if (!body(un, kt0, kt1)) return false;
    return true;
  };
  // Keys of tile kt that the sequence has (may be 0 when it has none at all).
  auto tile_valid = [&](const ChunkUnit& un, int kt) { return min(kTileN, un.kvlen - kt * kTileN); };

  if (warp == kProducerWarp) {
    // ------------------------------------------------------ TMA producer --
    if (lane == 0) {
      uint32_t c = 0;
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      int seq = -1, cached_lb = -1, cached_page = 0;
      auto page_of = [&](const ChunkUnit& un, int lb) -> int {
        if (un.seq == seq && lb == cached_lb) return cached_page;
        int b = lb >= p.batch.table_width ? -1
                : p.batch.tables          ? p.batch.tables[un.seq * p.batch.table_stride + lb]
                                          : un.seq * p.batch.table_width + lb;  // the expanded copy
        if (b < 0 || b >= p.pool.blocks) {  // reported; block 0 keeps the load in bounds
          atomicCAS(err, 0, kErrBlockTable);
          b = 0;
        }
        seq = un.seq;
        cached_lb = lb;
        return cached_page = b;
      };
      // Boxes of [key0, key0 + n) of K or V of one head; row 0 of `dst` is key0.
      auto load_rows = [&](const ChunkUnit& un, bool is_v, int key0, int n, uint32_t dst, uint32_t full) {
        for (int r = 0; r < n; r += box_rows) {
          const int key = key0 + r;
          const int pg = page_of(un, key / p.pool.block_size), at = key % p.pool.block_size;
          if (kFp8) {
            if (is_v)
              tma_load_5d(dst + r * (D / 2), &tm_v, static_cast<int>(rank) * (D / 2), at, un.head, 1, pg, full);
            else
              tma_load_5d(dst + r * D, &tm_k, 0, at, un.head, 0, pg, full);
          } else if (is_v) {
            for (int b = 0; b < D / 128; ++b)
              tma_load_5d(dst + b * L::kVBox + r * 128, &tm_v, static_cast<int>(rank) * (D / 2) + b * 64, at, un.head, 1,
                          pg, full);
          } else {
            for (int b = 0; b < D / 64; ++b)
              tma_load_5d(dst + b * L::kKBox + r * 128, &tm_k, b * 64, at, un.head, 0, pg, full);
          }
        }
      };
      auto issue = [&](const ChunkUnit& un, bool is_v, int kt) {
        const int st = c % NL;
        const uint32_t empty = kFp8 ? bar_land_empty(st) : bar_op_empty(st);
        if (!mbar_wait(empty, ((c / NL) & 1u) ^ 1u, abort_flag, err, kErrWaitKvEmpty)) return false;
        const uint32_t dst = kFp8 ? sRaw + st * L::kRawBytes : sOp + st * L::kOpBytes;
        const int off = is_v ? 0 : 64 * static_cast<int>(rank), most = is_v ? 128 : 64;
        const int n = min(most, max(0, tile_valid(un, kt) - off));
        const int rows = (n + box_rows - 1) / box_rows * box_rows;
        mbar_arrive_expect_tx(bar_land_full(st), rows * (is_v ? D / 2 : D) * (kFp8 ? 1 : 2));
        load_rows(un, is_v, kt * kTileN + off, n, dst, bar_land_full(st));
        ++c;
        return true;
      };
      // Item order = converter and MMA consumption order: per segment K_0,
      // then (K_{j+1}, V_j) per tile.
      const bool ok = for_each_segment([&](const ChunkUnit& un, int kt0, int kt1) -> bool {
        if (!issue(un, false, kt0)) return false;
        for (int kt = kt0; kt < kt1; ++kt) {
          if (kt + 1 < kt1 && !issue(un, false, kt + 1)) return false;
          if (!issue(un, true, kt)) return false;
        }
        return true;
      });
      if (!ok)  // let this CTA's copies still in flight land before it exits
        for (uint32_t i = (c > (uint32_t)NL ? c - NL : 0); i < c; ++i)
          mbar_wait_teardown(bar_land_full(i % NL), (i / NL) & 1u);
    }
    __syncwarp();
  } else if (warp >= kTilesConvWarp0) {
    // ------------------------------- Q gather, e4m3 -> f16, V past the end --
    const int ct = threadIdx.x - kTilesConvWarp0 * 32;
    const int cw = warp - kTilesConvWarp0;
    const ConvGeo geo_k = conv_geo(ct, D / 64, L::kKBox);
    const ConvGeo geo_v = conv_geo(ct, D / 128, L::kVBox);
    uint32_t c = 0, J = 0;
    int segs = 0;
    auto wait_all = [&](uint32_t bar, uint32_t parity, int code) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code));
    };
    auto item = [&](const ChunkUnit& un, bool is_v, int kt) -> bool {
      const int ls = c % NL, os = c % NS;
      const int valid = tile_valid(un, kt);
      if (kFp8) {
        if (kScaled && !is_v) {  // this tile's scales: a key a thread
          const int key = kt * kTileN + ct;
          uint32_t kb = 127, vb = 0;
          if (ct < valid) {
            const int lb = key / p.pool.block_size;
            int pg = lb < p.batch.table_width ? p.batch.tables[un.seq * p.batch.table_stride + lb] : 0;
            if (pg < 0 || pg >= p.pool.blocks) pg = 0;  // the producer reports it
            const uint8_t* sc = p.pool.scales +
                                (static_cast<long long>(pg) * 2 * p.pool.heads + un.head) * p.pool.block_size +
                                key - lb * p.pool.block_size;
            kb = sc[0];
            vb = sc[static_cast<long long>(p.pool.heads) * p.pool.block_size];
          }
          float* sf = reinterpret_cast<float*>(smem + L::kScaleOff + (J % (NB ? NB : 1)) * L::kScaleBuf);
          // (The buffer is free: see kScaleBufs; the item's op stage is waited
          // for below, so wait for it here first.)
          if (!wait_all(bar_op_empty(os), ((c / NS) & 1u) ^ 1u, kErrWaitKvEmpty)) return false;
          sf[ct] = __uint_as_float(kb << 23);
          sf[kTileN + ct] = __uint_as_float(vb << 23);
          const uint32_t vm = __reduce_max_sync(0xffffffffu, vb);
          if (lane == 0) reinterpret_cast<int*>(sf + 2 * kTileN)[cw] = static_cast<int>(vm);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_scale(J % (NB ? NB : 1)));
        }
        if (!is_v) ++J;
        if (!wait_all(bar_land_full(ls), (c / NL) & 1u, kErrWaitKvFull)) return false;
        if (!wait_all(bar_op_empty(os), ((c / NS) & 1u) ^ 1u, kErrWaitKvEmpty)) return false;
        const uint32_t raw = sRaw + ls * L::kRawBytes;
        const uint32_t op = sOp + os * L::kOpBytes;
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        // As attn_kv.cuh: D/32 16-byte chunks a thread, four in flight; rows
        // past the sequence are zeros.
        const ConvGeo& g = is_v ? geo_v : geo_k;
        const int vrows = is_v ? valid : valid - 64 * static_cast<int>(rank);
        const int row_step = is_v ? 64 / (D / 64) : 32 / (D / 64);
        const uint32_t op_step = row_step * 128;
#pragma unroll 1
        for (int m0 = 0; m0 < D / 32; m0 += 4) {
          uint4 x[4];
#pragma unroll
          for (int m = 0; m < 4; ++m)
            x[m] = g.row + (m0 + m) * row_step < vrows ? lds128(raw + g.raw + (m0 + m) * 2048) : zero;
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            uint4 lo, hi;
            e4m3x16_to_f16(x[m], lo, hi);
            const uint32_t o = op + (m0 + m) * op_step;
            sts128(o + g.lo, lo);
            sts128(o + g.hi, hi);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_land_empty(ls));
          mbar_arrive_remote(mapa_shared(bar_op_full(os), 0));
        }
      } else {
        if (!wait_all(bar_land_full(ls), (c / NL) & 1u, kErrWaitKvFull)) return false;
        if (is_v && valid < kTileN) {
          const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
          const uint32_t op = sOp + os * L::kOpBytes;
          for (int i = max(0, valid) * 8 + ct; i < kTileN * 8; i += kTilesConvThreads)
            for (int b = 0; b < D / 128; ++b) sts128(op + b * L::kVBox + i * 16, zero);
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(bar_op_full(os), 0));
      }
      ++c;
      return true;
    };
    for_each_segment([&](const ChunkUnit& un, int kt0, int kt1) -> bool {
      // Q rows into the swizzled operand layout: a row over D / 8 lanes,
      // kFlight loads a lane in flight, the first of them before the wait for the
      // previous segment's QK^T to be done with the buffer.
      constexpr int kSide = 256 / D;  // rows side by side in a warp
      constexpr int kFlight = kFp8 ? 4 : 16;  // (the conversion unrolled 16 times costs the instruction cache more)
      const int side = lane / (D / 8), ch = lane % (D / 8);
#pragma unroll 1
      for (int r0 = cw * 32; r0 < cw * 32 + 32; r0 += kFlight * kSide) {
        uint4 x[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
          const int r = static_cast<int>(rank) * kTileM + r0 + u * kSide + side;
          const int row = un.row0 + r;
          x[u] = make_uint4(0u, 0u, 0u, 0u);
          if (r < un.rows)
            x[u] = *reinterpret_cast<const uint4*>(
                p.q + static_cast<long long>(un.head * p.group + row % p.group) * p.q_head +
                static_cast<long long>(un.q0 + row / p.group) * p.q_row + 8 * ch);
        }
        if (r0 == cw * 32 && segs > 0 && !wait_all(bar_q_empty, (segs - 1) & 1u, kErrWaitQ)) return false;
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
          const int r = r0 + u * kSide + side;
          if (kFp8) {
            float f[8];
            Vec8<__nv_bfloat16>{x[u]}.get(f);
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t a = __float_as_uint(f[i]) & 0x7FFFFFFFu;
              if (a < 0x7F800000u) m = max(m, a);
            }
#pragma unroll
            for (int o = D / 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const int e = m == 0 ? 0 : max(static_cast<int>(m >> 23) - 127 - 14, -112);
            const float down = exp2_of_int(-e);
            if (ch == 0) factors[(segs & 1) * kTileM + r] = p.scale_log2 * exp2_of_int(e);
            x[u] = make_uint4(pack_f16x2(f[0] * down, f[1] * down), pack_f16x2(f[2] * down, f[3] * down),
                              pack_f16x2(f[4] * down, f[5] * down), pack_f16x2(f[6] * down, f[7] * down));
          }
          sts128(sQ + (ch / 8) * kBoxBytes + r * 128 + (((ch % 8) ^ (r & 7)) << 4), x[u]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_rows(segs));
        mbar_arrive_remote(mapa_shared(bar_q_ready, 0));
      }
      ++segs;
      if (!item(un, false, kt0)) return false;
      for (int kt = kt0; kt < kt1; ++kt) {
        if (kt + 1 < kt1 && !item(un, false, kt + 1)) return false;
        if (!item(un, true, kt)) return false;
      }
      return true;
    });
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // --------------------------------------------- MMA issuer (leader only) --
    if (leader && lane == 0) {
      constexpr uint32_t idesc_qk =
          kFp8 ? make_idesc_f16(kUnitRows, kTileN, false, false) : make_idesc_bf16(kUnitRows, kTileN, false, false);
      constexpr uint32_t idesc_pv =
          kFp8 ? make_idesc_f16(kUnitRows, D, false, true) : make_idesc_bf16(kUnitRows, D, false, true);
      uint32_t c = 0;
      uint32_t J = 0;  // tiles of all earlier segments
      int segs = 0;
      auto qk = [&](uint32_t jg) {
        const uint32_t s_tmem = tmem + kTmemS0 + (jg & 1) * kTileN;
        const int st = c % NS;
        if (!mbar_wait(bar_op_full(st), (c / NS) & 1u, abort_flag, err, kErrWaitKvFull)) return false;
        tc_fence_after();
        const uint32_t kbase = sOp + st * L::kOpBytes;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t qa = sQ + (kk / 4) * kBoxBytes + (kk % 4) * 32;
          const uint32_t kb = kbase + (kk / 4) * L::kKBox + (kk % 4) * 32;
          umma_ss_pair(s_tmem, make_sw128_desc(qa, 16, 1024), make_sw128_desc(kb, 16, 1024), idesc_qk,
                       kk != 0 ? 1u : 0u);
        }
        umma_commit_pair(bar_op_empty(st), kChunkBothCtas);
        ++c;
        umma_commit_pair(bar_s_full(jg & 1), kChunkBothCtas);
        return true;
      };
      auto pv = [&](uint32_t jg, bool first) {
        if (!mbar_wait(bar_p_full(jg & 1), (jg >> 1) & 1u, abort_flag, err, kErrWaitPFull)) return false;
        const int st = c % NS;
        if (!mbar_wait(bar_op_full(st), (c / NS) & 1u, abort_flag, err, kErrWaitKvFull)) return false;
        tc_fence_after();
        const uint32_t p_tmem = tmem + kTmemS0 + (jg & 1) * kTileN;
        const uint32_t vbase = sOp + st * L::kOpBytes;
#pragma unroll
        for (int kk = 0; kk < kTileN / 16; ++kk) {
          // A = P (TMEM columns of the S buffer, each warpgroup's in its own
          // half), B = V half, MN-major: 64-dim chunks 16 KB apart, 8-key
          // groups 1 KB apart.
          const uint32_t a_cols = kk * 8 + (kk >= 4 ? 32 : 0);
          umma_ts_pair(tmem, p_tmem + a_cols, make_sw128_desc(vbase + kk * 2048, L::kVBox, 1024), idesc_pv,
                       (!first || kk > 0) ? 1u : 0u);
        }
        umma_commit_pair(bar_op_empty(st), kChunkBothCtas);
        ++c;
        umma_commit_pair(bar_o(jg & 1), kChunkBothCtas);
        return true;
      };
      for_each_segment([&](const ChunkUnit&, int kt0, int kt1) -> bool {
        const uint32_t n = static_cast<uint32_t>(kt1 - kt0);
        // (O of the previous segment has been read out: its softmax warps
        // release P_0 of this segment only after their epilogue.)
        if (!mbar_wait(bar_q_ready, segs & 1u, abort_flag, err, kErrWaitQ)) return false;
        tc_fence_after();
        if (!qk(J)) return false;
        if (n == 1) umma_commit_pair(bar_q_empty, kChunkBothCtas);
        for (uint32_t j = 0; j < n; ++j) {
          if (j + 1 < n) {
            if (!qk(J + j + 1)) return false;
            if (j + 2 == n) umma_commit_pair(bar_q_empty, kChunkBothCtas);  // last QK^T of the segment
          }
          if (!pv(J + j, j == 0)) return false;
        }
        J += n;
        ++segs;
        return true;
      });
      // Drain: completes when every MMA issued above has.
      umma_commit_pair(bar_td, kChunkLeader);
      mbar_wait_teardown(bar_td, 0);
    }
    __syncwarp();
  } else {
    // ---------------------------------------- softmax / correction / epilogue --
    constexpr int kHalfKeys = kTileN / kSoftmaxWarpgroups;  // 64
    constexpr int kOCols = D / kSoftmaxWarpgroups;
    const int wg = warp >> 2;
    const int row = threadIdx.x & (kTileM - 1);  // == TMEM lane
    const uint32_t t_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    uint32_t J = 0;
    int segs = 0;
    // The leader keeps the pair's record.
    ChunkRecord& rec = p.work.tile_rec[pair];
    const bool keeps = leader && threadIdx.x == 0;
    if (keeps) clear_record(rec);
    const bool done = for_each_segment([&](const ChunkUnit& un, int kt0, int kt1) -> bool {
      if (keeps) note_part(rec, un, kt0, kt1);
      bool ok = true;
      const int r = static_cast<int>(rank) * kTileM + row;  // row of the unit
      const bool live = r < un.rows;
      const int at = un.row0 + (live ? r : un.rows - 1);
      const int pos = un.kvlen - un.qlen + at / p.group;  // last key this row sees
      const int n = kt1 - kt0;
      float rf = p.scale_log2;
      if (kFp8) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_rows(segs), (segs >> 1) & 1u, abort_flag, err, kErrWaitQ));
        if (ok) rf = factors[(segs & 1) * kTileM + row];
      }
      ++segs;
      float m_ref = -INFINITY;  // log2 units, V's exponents included
      float l = 0.f;
      for (int j = 0; j < n && ok; ++j) {
        const uint32_t jg = J + j;
        const int b = jg & 1;
        const int key0 = (kt0 + j) * kTileN + wg * kHalfKeys;
        const float* sf = reinterpret_cast<const float*>(smem + L::kScaleOff + (jg % (NB ? NB : 1)) * L::kScaleBuf);
        float ev = 0.f;
        if (kScaled) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar_scale(jg % (NB ? NB : 1)), (jg / (NB ? NB : 1)) & 1u, abort_flag,
                                                 err, kErrWaitKvFull));
          if (!ok) break;
          const int4 vm = *reinterpret_cast<const int4*>(sf + 2 * kTileN);
          ev = static_cast<float>(max(max(vm.x, vm.y), max(vm.z, vm.w)) - 127);
        }
        ok = __all_sync(0xffffffffu, mbar_wait(bar_s_full(b), (jg >> 1) & 1u, abort_flag, err, kErrWaitSFull));
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_s = t_row + kTmemS0 + b * kTileN + wg * kHalfKeys;
        float s[kHalfKeys];
#pragma unroll
        for (int c = 0; c < kHalfKeys / 32; ++c) tmem_ld32(t_s + 32 * c, s + 32 * c);
        tmem_wait_ld();
        if (kScaled) {
          const float4* ks = reinterpret_cast<const float4*>(sf + wg * kHalfKeys);
#pragma unroll
          for (int i = 0; i < kHalfKeys / 4; ++i) {
            const float4 k4 = ks[i];
            s[4 * i] *= k4.x;
            s[4 * i + 1] *= k4.y;
            s[4 * i + 2] *= k4.z;
            s[4 * i + 3] *= k4.w;
          }
        }
        const int visible = pos + 1 - key0;
        if (visible < kHalfKeys) {
#pragma unroll
          for (int i = 0; i < kHalfKeys; ++i)
            if (i >= visible) s[i] = -INFINITY;
        }
        const float pmax = row_max(s);
        red[(b * kSoftmaxWarpgroups + wg) * kTileM + row] = pmax;
        mbar_arrive(bar_red(b));
        // Pass 0 (tiles after the first): speculative P with the current
        // reference, before the other half's maximum is known.  Pass 1:
        // exchange the half maxima; P is recomputed only when some row's
        // moved past the threshold.
        float tile_sum = 0.f;
        float alpha = 1.f;
        bool redo = false;
#pragma unroll 1
        for (int pass = j > 0 ? 0 : 1; pass < 2; ++pass) {
          if (pass == 1) {
            ok = __all_sync(0xffffffffu, mbar_wait(bar_red(b), (jg >> 1) & 1u, abort_flag, err, kErrWaitRed));
            if (!ok) break;
            const float tmax =
                fmaxf(pmax, red[(b * kSoftmaxWarpgroups + (wg ^ 1)) * kTileM + row]) * rf + ev;
            const bool need = tmax > m_ref + kRescaleThreshold;  // from its start as soon as a key is seen
            redo = __any_sync(0xffffffffu, need) || j == 0;
            if (need) {
              alpha = ex2_approx(m_ref - tmax);  // 0 from the start
              m_ref = tmax;
              l *= alpha;
            }
            if (!redo) break;
          }
          // P over this warpgroup's S columns; a row that has seen nothing yet
          // has only -inf scores.
          const float neg = m_ref == -INFINITY ? 0.f : -m_ref;
          float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
          for (int c2 = 0; c2 < kHalfKeys / 32; ++c2) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              float q0 = ex2_approx(fmaf(s[c2 * 32 + 2 * i], rf, neg));
              float q1 = ex2_approx(fmaf(s[c2 * 32 + 2 * i + 1], rf, neg));
              float q2 = ex2_approx(fmaf(s[c2 * 32 + 2 * i + 2], rf, neg));
              float q3 = ex2_approx(fmaf(s[c2 * 32 + 2 * i + 3], rf, neg));
              sum0 += q0 + q2;
              sum1 += q1 + q3;
              if (kScaled) {
                const float4 v4 = *reinterpret_cast<const float4*>(sf + kTileN + wg * kHalfKeys + c2 * 32 + 2 * i);
                q0 *= v4.x;
                q1 *= v4.y;
                q2 *= v4.z;
                q3 *= v4.w;
              }
              pk[i] = kFp8 ? pack_f16x2(q0, q1) : pack_bf16x2(q0, q1);
              pk[i + 1] = kFp8 ? pack_f16x2(q2, q3) : pack_bf16x2(q2, q3);
            }
            tmem_st16(t_s + c2 * 16, pk);
          }
          tmem_wait_st();
          tile_sum = sum0 + sum1;
        }
        if (!ok) break;
        l += tile_sum;
        if (j > 0 && redo) {
          ok = __all_sync(0xffffffffu,
                          mbar_wait(bar_o((jg - 1) & 1), ((jg - 1) >> 1) & 1u, abort_flag, err, kErrWaitODone));
          if (!ok) break;
          tc_fence_after();
          rescale_o<kOCols>(t_row + wg * kOCols, alpha);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(bar_p_full(b), 0));
      }
      if (ok) {
        const uint32_t jl = J + n - 1;
        ok = __all_sync(0xffffffffu, mbar_wait(bar_o(jl & 1), (jl >> 1) & 1u, abort_flag, err, kErrWaitODone));
      }
      ok = named_bar_and(1, kSoftmaxThreads, ok && (*abort_flag == 0));
      if (!ok) return false;
      J += n;
      tc_fence_after();
      red[wg * kTileM + row] = l;
      named_bar_sync(2, kSoftmaxThreads);
      const float l_tot = l + red[(wg ^ 1) * kTileM + row];
      // Both halves read: the next segment may reuse the exchange slots.
      named_bar_sync(2, kSoftmaxThreads);
      const float inv_l = l_tot == 0.f ? 0.f : 1.f / l_tot;  // no key seen: zeros
      const int slot = part_slot(un, kt0, kt1, pair);
      if (slot < 0) {
        store_o_bf16<kOCols>(t_row + wg * kOCols, inv_l,
                             p.out + static_cast<long long>(un.head * p.group + at % p.group) * p.out_head +
                                 static_cast<long long>(un.q0 + at / p.group) * p.out_row + wg * kOCols,
                             live);
      } else {
        const long long pr = static_cast<long long>(slot) * kUnitRows + r;
        store_o_partial<kOCols>(t_row + wg * kOCols, inv_l, p.work.tile_o + pr * D + wg * kOCols, live);
        if (live && wg == 0)
          p.work.tile_lse[pr] = l_tot == 0.f ? -INFINITY : (m_ref == -INFINITY ? 0.f : m_ref) + __log2f(l_tot);
      }
      return true;
    });
    if (keeps && !done) clear_record(rec);  // after a failure nothing is merged
  }

  // Both CTAs: the leader's MMAs (which read the peer's smem and TMEM) are
  // drained, every TMEM read of either CTA is done.
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  if (threadIdx.x == 0) p.work.tile_rec[blockIdx.x].err = *static_cast<volatile int*>(err);
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, kTmemCols);
  }
}

}  // namespace pcp
