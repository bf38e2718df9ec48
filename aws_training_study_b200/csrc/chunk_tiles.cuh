// Attention of longer chunks over a paged cache: tiles of 256 query rows on
// the tensor cores.
//
// 512 tokens over 131072 (32 / 2 heads of 256, e4m3 expanded): 1.55 ms, 1.42
// PFLOP/s, what a long GEMM sustains here; four prompts of 2048 (64 / 8 heads of
// 128, bf16): 280 us, 0.72 PFLOP/s of the causal half, the softmax its limit (per
// tile 1050 cycles of exponentials in some 2200; a quarter of them as polynomials
// on the FMA pipe made it 305 us).
// Bound by the MMAs (4 * 256 * 128 * D flops per 128-key tile of a unit against
// 2 * 128 * D cache elements), with the softmax next: 128 x 128 exponentials a
// CTA and tile take the MUFU 1024 cycles, the MMAs 1024 (D = 128) or 2048.  As in
// attn_kv.cuh a cluster of two CTAs shares every tcgen05 MMA (cta_group::2: each
// CTA holds 128 query rows, half of each K tile's keys and half of each V tile's
// columns), and scores and probabilities live in TMEM.  What differs:
//   * The two softmax warpgroups of a CTA split each tile's keys between them.  (One
//     with the even tiles and one with the odd ones, a thread a whole row, was
//     slower: 400 us for the four prompts where this, otherwise alike, took 358.)
//   * D = 128: TMEM has room for two accumulators, and the converter warps write a
//     finished one out while the softmax warps and the MMAs are at the next unit;
//     Q has two buffers, so that the next unit's first QK^T is issued ahead of the
//     last PV of the one before.
//   * D = 256: one of each; the softmax warps write the output.
//   * Units come from the plan (chunk_plan.cuh): any mix of sequences, each pair
//     walking an equal range of the batch's steps.
//   * K and V are read from pages of any multiple of 16 tokens, through the
//     sequence's table, box by box.
//   * Rows are (token, query head) pairs of a strided Q: boxes of {group, tokens}
//     by TMA (bf16 operands, group a divisor of 128), else gathered by the
//     converter warps; each row sees keys up to its position.
//   * bf16 caches land in operand layout straight from TMA, both CTAs' bytes on
//     the leader's barrier; the converter warps only see V of a unit's last tiles,
//     where they clear the rows that no row sees (they may hold anything: 0 * NaN
//     would reach every row) and values that are not finite (nonfinite8).
//   * An e4m3 cache that many query tiles read is expanded into a bf16 copy first
//     (chunk_expand_kernel; exact, scales included but for a common power of two),
//     when the copy is of moderate size: reading it in place converts every key tile
//     again for each 256 rows.  The weights are rounded to bf16 then, within
//     2^-8 where in place it is 2^-11: an MMA's operands share a type, and f16 does not
//     reach the scaled values.
//   * Scaled e4m3 caches: K's 2^e multiplies the scores of its key, V's e is added to
//     the exponent of its weight, and the softmax reference follows the largest
//     score + V exponent, key by key, as in chunk_rows.cuh.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include <climits>
#include <type_traits>

#include "attn_common.cuh"
#include "attn_softmax.cuh"
#include "chunk_plan.cuh"
#include "conv_geo.cuh"

namespace pcp {

constexpr int kTilesConvWarps = 4;
constexpr int kTilesConvThreads = 32 * kTilesConvWarps;
// Four warpgroups: softmax 0 and 1; K/V copies, MMA, segments and Q, K/V copies;
// converters.  They split the launch's 512 x 128 registers (TilesSmem).
constexpr int kSegmentWarp = 10, kProducerWarp2 = 11;
constexpr int kTilesConvWarp0 = 12;
constexpr int kTilesThreads = 512;
constexpr int kTilesLaunchRegs = 128;
constexpr uint16_t kChunkBothCtas = 3, kChunkLeader = 1;

// A unit; keys from see_all on some rows do not see, from see_any on none does.
struct TileUnit : ChunkUnit {
  int see_all, see_any;
};
// A segment: the part [kt0, kt1) of a unit's key tiles; kt1 = 0 after the last.
struct __align__(16) TileSegment {
  TileUnit un;
  int kt0, kt1;
};
// Segments on their way from the warp that walks the range to the others (each
// walking by itself, the loads and divisions of a step took every role some 1500
// to 2000 cycles a unit).
constexpr int kTileSegments = 4;

template <int D, int kCache>
struct TilesSmem {
  static constexpr bool kFp8 = kCache != kCacheBf16;
  static constexpr int kQBytes = D * 2 * kTileM;
  static constexpr int kOpBytes = 128 * D;  // 16-bit K half [64, D] or V half [128, D/2], swizzled
  static constexpr int kRawBytes = 64 * D;  // e4m3 K half [64][D] or V half [128][D/2]
  static constexpr bool kTwo = D == 128;  // two accumulators and buffers of Q, output by the converter warps
  static constexpr int kSoftmaxRegs = 144, kControlRegs = 112, kConvRegs = 112;
  static_assert(2 * kSoftmaxRegs + kControlRegs + kConvRegs <= 4 * kTilesLaunchRegs, "more than the launch's registers");
  static constexpr int kQBufs = kTwo ? 2 : 1;
  static constexpr int kOpStages = kFp8 ? (D == 256 ? 3 : 5) : (D == 256 ? 5 : 8);
  static constexpr int kRawStages = kFp8 ? (D == 256 ? 3 : 6) : 0;
  static constexpr int kLandStages = kFp8 ? kRawStages : kOpStages;  // stages the TMA fills
  // Warps that issue the copies.  Two: one the even items, one the odd (an item
  // takes a warp some 1000 cycles, as long as half a tile's MMAs take with D = 128),
  // and, with an even number of stages, each sees every filling of its own.
  static constexpr int kProducers = kTwo ? 2 : 1;
  static_assert(kLandStages % kProducers == 0, "a stage has one producer");
  static constexpr int kKBox = 64 * 128;
  static constexpr int kVBox = 128 * 128;
  // A tile's scales are rewritten once its P has been consumed: among the items
  // in their order, V of tile J is at most 2 J + 2, K of tile J + k at least
  // 2 (J + k) - 1, and an item is converted once the one kOpStages before it was
  // consumed.
  static constexpr int kScaleBufs = kCache == kCacheScaled ? (kOpStages + 4) / 2 : 0;
  static constexpr int kOpOff = kQBufs * kQBytes;
  static constexpr int kRawOff = kOpOff + kOpStages * kOpBytes;
  static constexpr int kScaleOff = kRawOff + kRawStages * kRawBytes;  // float k[128] (2^e), v[128] (e)
  static constexpr int kScaleBuf = 2 * kTileN * 4;
  // Row factors of a segment, float[128] each, and (kTwo) its rows' sums of either
  // warpgroup and references.  Q of a segment is written once QK^T of the one
  // kQBufs before it is done, and QK^T of a tile is issued after PV two tiles
  // back: a softmax warpgroup may be three segments (of one tile each) behind Q
  // with kTwo, one without.  The same PV, if it is a segment's first, waits for the
  // output of the segment two before it: the softmax warps are at most three
  // segments ahead of the output.
  static constexpr int kSegBufs = kTwo ? 4 : 2;
  static constexpr int kFactorOff = kScaleOff + kScaleBufs * kScaleBuf;
  static constexpr int kRedOff = kFactorOff + (kFp8 ? kSegBufs * kTileM * 4 : 0);
  // The halves' maxima [tile parity][2][128]: scores, or (scaled) score + exponent, then scores.
  static constexpr int kMaxima = kCache == kCacheScaled ? 8 : 4;
  static constexpr int kSums = kCache == kCacheScaled ? 4 : 3;  // of a segment, kTwo
  static constexpr int kBarOff = kRedOff + (kMaxima + (kTwo ? kSums * kSegBufs : 0)) * kTileM * 4;
  // q_ready[2], q_empty[2], rows[4], o_free[2], sums[4], seg_o[2], land_full[NL],
  // land_empty[NR], op_full[NS], op_empty[NS], s_full[2], p_full[2], o_done[2],
  // teardown, ref[2], scale[NB], seg_full[], seg_empty[]
  static constexpr int kNumBars = 16 + kLandStages + kRawStages + 2 * kOpStages + 9 + kScaleBufs + 2 * kTileSegments;
  static constexpr int kMiscOff = (kBarOff + kNumBars * 8 + 15) / 16 * 16;
  static constexpr int kSegOff = kMiscOff + 16;  // TileSegment[kTileSegments]
  static constexpr int kPlanOff = kSegOff + kTileSegments * sizeof(TileSegment);  // ChunkPlanShared
  static constexpr int kBytes = kPlanOff + sizeof(ChunkPlanShared);
  static_assert(kBytes <= 232448, "exceeds the 227 KB of shared memory per CTA");
  static_assert(kRawOff % 1024 == 0 && kScaleOff % 16 == 0 && kSegOff % 16 == 0 && kBarOff % 8 == 0, "alignment");
};

// 16 rows (lanes l / 4 and l / 4 + 8) of 32 TMEM columns: o[4 i], o[4 i + 1] are
// columns 8 i + 2 (l % 4), + 1 of the first row, o[4 i + 2], o[4 i + 3] of the second.
__device__ __forceinline__ void tmem_ld16x32(uint32_t t, float (&o)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(t));
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = __uint_as_float(r[i]);
}

// A warp's 32 rows (a lane each), O * inv_l of kCols TMEM columns from t_o, to
// `dst` (NULL: not written), bf16 or fp32.  Four lanes hold and store 64 bytes of
// a row (a lane storing its own row touched 32 lines with every instruction: 11600
// cycles a unit, D = 256).
template <int kCols, typename T>
__device__ __forceinline__ void store_rows(uint32_t t_o, float inv_l, T* dst, int lane) {
  constexpr bool kBf16 = sizeof(T) == 2;
  const int q = lane & 3;
  const bool odd = q & 1, high = q & 2;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {  // rows 16 h ..
    float inv[2];
    T* to[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 16 * h + 8 * e + lane / 4;
      inv[e] = __shfl_sync(0xffffffffu, inv_l, r);
      to[e] = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
    }
#pragma unroll 2
    for (int c = 0; c < kCols; c += 32) {
      float o[16];
      tmem_ld16x32(t_o + (static_cast<uint32_t>(16 * h) << 16) + c, o);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (kBf16) {
          // Lane q gets the four words of columns 8 q ..: a 4 x 4 transposition.
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(o[4 * i + 2 * e] * inv[e], o[4 * i + 2 * e + 1] * inv[e]);
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const uint32_t x = __shfl_xor_sync(0xffffffffu, odd ? w[i] : w[i + 1], 1);
            w[i] = odd ? x : w[i];
            w[i + 1] = odd ? w[i + 1] : x;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x = __shfl_xor_sync(0xffffffffu, high ? w[i] : w[i + 2], 2);
            w[i] = high ? x : w[i];
            w[i + 2] = high ? w[i + 2] : x;
          }
          if (to[e]) *reinterpret_cast<uint4*>(to[e] + c + 8 * q) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
          // Even lanes get four columns of group i, odd ones of group i + 1.
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float a0 = o[4 * i + 2 * e] * inv[e], a1 = o[4 * i + 2 * e + 1] * inv[e];
            const float b0 = o[4 * i + 4 + 2 * e] * inv[e], b1 = o[4 * i + 4 + 2 * e + 1] * inv[e];
            const float x = __shfl_xor_sync(0xffffffffu, odd ? a0 : b0, 1);
            const float y = __shfl_xor_sync(0xffffffffu, odd ? a1 : b1, 1);
            if (to[e])
              *reinterpret_cast<float4*>(to[e] + c + 8 * (i + (odd ? 1 : 0)) + 2 * (q & 2)) =
                  odd ? make_float4(x, y, b0, b1) : make_float4(a0, a1, x, y);
          }
        }
      }
    }
  }
}

// How K and V tiles are copied.  A copy costs its issuer 170 cycles and more,
// whatever its size (eight a tile held the kernel at 2900 cycles a tile, D = 256),
// so one brings as many rows, and as many 64-element columns, as the pages allow.
struct TileBoxes {
  int q_copy;          // Q by one copy a segment (bf16 operands, group a divisor of 128); else gathered
  int k_rows, v_rows;  // rows of a copy: K up to 64, V up to 128
  int all_cols;        // bf16: all 64-element columns in a copy (pages of a multiple of 64 tokens)
};

// Values of a scaled cache are copied times 2^-kCopyShift, scores and output are
// multiplied back: 448 * 2^120 is beyond bf16 (a value of 2^128, which an append may
// write, became infinity and, where it passed the converter warps, vanished), and the
// sums of weights up to 2^8 need room in fp32 too.  The least code, 2^-9, at the least
// exponent, -100, is still a normal bf16 number.
constexpr int kCopyShift = 16;

// The pages of sequences with tile units as bf16: sequence s is one block of
// `copy`, [2][Hkv][copy_rows][D].  Bound by HBM (1 byte read, 2 written an
// element); a thread block takes 64 rows of one head of K or V at a time (pages
// of a multiple of 64 tokens; else 16).
struct ExpandParams {
  ChunkParams c;
  __nv_bfloat16* copy;
  int copy_rows;  // table_width * block_size, up to a multiple of 128
  int item_rows;  // 64 or 16
};

template <int D>
__device__ __forceinline__ void expand_item(const ExpandParams& p, int s, int kvlen, long long item) {
  constexpr int kPerRow = D / 16;
  const PoolView& pool = p.c.pool;
  const int per_page = 2 * pool.heads;
  const int piece = static_cast<int>(item / per_page), which = static_cast<int>(item - static_cast<long long>(piece) * per_page);
  const int key0 = piece * p.item_rows, lb = key0 / pool.block_size, row0 = key0 - lb * pool.block_size;
  const int n = min(p.item_rows, kvlen - key0);
  const int blk = p.c.batch.tables[s * p.c.batch.table_stride + lb];
  const bool found = blk >= 0 && blk < pool.blocks;
  if (!found && threadIdx.x == 0) atomicCAS(p.c.status, 0, kErrBlockTable);
  const long long src = (static_cast<long long>(found ? blk : 0) * per_page + which) * pool.block_size + row0;
  const uint4* codes = reinterpret_cast<const uint4*>(pool.data + src * D);
  const uint8_t* scales = pool.scales ? pool.scales + src : nullptr;
  uint4* dst = reinterpret_cast<uint4*>(p.copy + ((static_cast<long long>(s) * per_page + which) * p.copy_rows + key0) * D);
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
      e4m3x16_to_bf16(x[u], scales ? __uint_as_float((min(max(sc[u], kCopyShift + 1u), 254u) - kCopyShift) << 23) : 1.f, o);
      dst[2 * e] = o[0];
      dst[2 * e + 1] = o[1];
    }
  }
}

template <int D>
__global__ void __launch_bounds__(256) chunk_expand_kernel(const ExpandParams p) {
  const int per_page = 2 * p.c.pool.heads, lane = threadIdx.x & 31;
  __shared__ int s_ignored;  // lengths the attention reports itself
  if (threadIdx.x == 0) s_ignored = 0;
  __syncthreads();
  grid_launch_dependents();
  // Items of the sequences with tile units alone, dealt out over the blocks (a
  // table may be far wider than the sequences are long).
  long long next = blockIdx.x;  // this block's next item, from the sequence's first
  for (int s0 = 0; s0 < p.c.batch.seqs; s0 += 32) {
    ChunkSeq mine{};
    if (s0 + lane < p.c.batch.seqs) mine = chunk_seq<true>(p.c, s0 + lane, &s_ignored);
    for (uint32_t with = __ballot_sync(0xffffffffu, mine.tiles > 0); with; with &= with - 1) {
      const int s = s0 + __ffs(with) - 1;
      const int kvlen = __shfl_sync(0xffffffffu, mine.kvlen, s - s0);
      const long long items = static_cast<long long>((kvlen + p.item_rows - 1) / p.item_rows) * per_page;
      for (; next < items; next += gridDim.x) expand_item<D>(p, s, kvlen, next);
      next -= items;
    }
  }
  grid_dependency_wait();  // the small units, as in chunk_tiles_kernel
}

template <int D, int kCache>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTilesThreads, 1)
    chunk_tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v,
                       const TileBoxes box, const ChunkParams p) {
  using L = TilesSmem<D, kCache>;
  constexpr bool kFp8 = L::kFp8;
  constexpr bool kScaled = kCache == kCacheScaled;
  const float v_factor = kFp8 ? 1.f : p.v_factor;
  constexpr int NS = L::kOpStages, NL = L::kLandStages, NR = L::kRawStages, NB = L::kScaleBufs;

  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  if (sbase & 1023u) {  // identical in both CTAs: neither starts
    if (threadIdx.x == 0) {
      p.work.tile_rec[blockIdx.x].err = kErrSmemAlign;
      p.work.tile_rec[blockIdx.x].failed = 1;
      p.work.tile_rec[blockIdx.x].patch = 0;
      clear_record(p.work.tile_rec[blockIdx.x >> 1]);
    }
    grid_dependency_wait();
    return;
  }
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const uint32_t sQ = sbase;
  const uint32_t sOp = sbase + L::kOpOff;
  const uint32_t sRaw = sbase + L::kRawOff;
  const uint32_t bars = sbase + L::kBarOff;
  // By segment parity (the buffers of Q with two; what runs ahead could pass a
  // single barrier by two phases, which its parity does not show):
  // leader: Q written in both CTAs (one arrive per converter warp; a copy: the
  // bytes of both);
  auto bar_q_ready = [&](int sg) { return bars + 8u * (sg & 1); };
  // the segment's last QK^T has read Q (MMA commit, both CTAs);
  auto bar_q_empty = [&](int sg) { return bars + 16 + 8u * (sg & 1); };
  // this CTA's row factors written (kSegBufs of them).
  auto bar_rows = [&](int sg) { return bars + 32 + 8u * (sg & (L::kSegBufs - 1)); };
  // Leader: O of the segment read by every warp of both CTAs that writes it out (two
  // of them with kTwo).
  auto bar_o_free = [&](int sg) { return bars + 64 + 8u * (L::kTwo ? sg & 1 : 0); };
  // kTwo: the segment's sums and references are in shared memory;
  auto bar_sums = [&](int sg) { return bars + 80 + 8u * (sg & (L::kSegBufs - 1)); };
  // its last PV is done (MMA commit, both CTAs).
  auto bar_seg_o = [&](int sg) { return bars + 112 + 8u * (sg & 1); };
  auto bar_land_full = [&](int s) { return bars + 8u * (16 + s); };
  auto bar_land_empty = [&](int s) { return bars + 8u * (16 + NL + s); };
  auto bar_op_full = [&](int s) { return bars + 8u * (16 + NL + NR + s); };
  auto bar_op_empty = [&](int s) { return bars + 8u * (16 + NL + NR + NS + s); };
  constexpr int kB2 = 16 + NL + NR + 2 * NS;
  auto bar_s_full = [&](int b) { return bars + 8u * (kB2 + b); };
  auto bar_p_full = [&](int b) { return bars + 8u * (kB2 + 2 + b); };
  auto bar_o = [&](int b) { return bars + 8u * (kB2 + 4 + b); };
  const uint32_t bar_td = bars + 8u * (kB2 + 6);
  auto bar_ref = [&](int b) { return bars + 8u * (kB2 + 7 + b); };
  auto bar_scale = [&](int b) { return bars + 8u * (kB2 + 9 + b); };
  auto bar_seg_full = [&](int sg) { return bars + 8u * (kB2 + 9 + NB + sg % kTileSegments); };
  auto bar_seg_empty = [&](int sg) { return bars + 8u * (kB2 + 9 + NB + kTileSegments + sg % kTileSegments); };
  TileSegment* segments = reinterpret_cast<TileSegment*>(smem + L::kSegOff);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  // V had values that were taken for zeros (nonfinite8).
  volatile int* patch = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 8);
  float* red = reinterpret_cast<float*>(smem + L::kRedOff);
  float* factors = reinterpret_cast<float*>(smem + L::kFactorOff);

  ChunkPlanShared& plan = *reinterpret_cast<ChunkPlanShared*>(smem + L::kPlanOff);
  int* err = &plan.err;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (warp == kProducerWarp && lane == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_q_ready(b), box.q_copy ? 1 : 2 * kTilesConvWarps);
      mbar_init(bar_q_empty(b), 1);
    }
    for (int b = 0; b < L::kSegBufs; ++b) {
      mbar_init(bar_rows(b), kTilesConvWarps);
      if (L::kTwo) mbar_init(bar_sums(b), 8);
    }
    for (int s = 0; s < NL; ++s) mbar_init(bar_land_full(s), 1);
    for (int s = 0; s < NR; ++s) mbar_init(bar_land_empty(s), kTilesConvWarps);
    for (int s = 0; s < NS; ++s) {
      // e4m3: every converter warp; bf16: the leader's producer twice, with the
      // bytes of both CTAs, or (V of edge tiles) each CTA once.
      mbar_init(bar_op_full(s), kFp8 ? 2 * kTilesConvWarps : 2);
      mbar_init(bar_op_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_s_full(b), 1);
      mbar_init(bar_p_full(b), 2 * 8);  // one arrive per softmax warp of both CTAs
      mbar_init(bar_o(b), 1);
      mbar_init(bar_ref(b), 256);
      if (L::kTwo || b == 0) mbar_init(bar_o_free(b), L::kTwo ? 2 * kTilesConvWarps : 2 * 8);
      mbar_init(bar_seg_o(b), 1);
    }
    for (int b = 0; b < NB; ++b) mbar_init(bar_scale(b), kTilesConvWarps);
    for (int b = 0; b < kTileSegments; ++b) {
      mbar_init(bar_seg_full(b), 1);
      mbar_init(bar_seg_empty(b), 8 + L::kProducers + 1 + kTilesConvWarps);  // every warp that reads them
    }
    mbar_init(bar_td, 1);
    *abort_flag = 0;
    *patch = 0;
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

  // Segment sg of this pair's range, for a whole warp; false after the last (or
  // when the kernel gives up).
  auto get_segment = [&](int sg, TileUnit& un, int& kt0, int& kt1) -> bool {
    if (!__all_sync(0xffffffffu, mbar_wait(bar_seg_full(sg), (sg / kTileSegments) & 1u, abort_flag, err, kErrWaitQ)))
      return false;
    const TileSegment& s = segments[sg % kTileSegments];
    un = s.un;
    kt0 = s.kt0;
    kt1 = s.kt1;
    return kt1 > 0;
  };
  auto put_back = [&](int sg) {  // read by this warp
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_seg_empty(sg));
  };
  // Calls body(unit, kt0, kt1, segment) for each segment until it returns false;
  // returns false if it did.
  auto for_each_segment = [&](auto&& body) -> bool {
    TileUnit un;
    int kt0, kt1;
    for (int sg = 0; get_segment(sg, un, kt0, kt1); ++sg) {
      put_back(sg);
      if (!body(un, kt0, kt1, sg)) return false;
    }
    return *abort_flag == 0;
  };
  // V of tile kt passes through the converter warps (bf16): rows to be cleared, or
  // to be looked through.
  auto edge = [&](const TileUnit& un, int kt) { return (kt + 1) * kTileN > un.see_all; };
  // Keys of tile kt that the sequence has (may be 0 when it has none at all).
  auto tile_valid = [&](const TileUnit& un, int kt) { return min(kTileN, un.kvlen - kt * kTileN); };
  // The items of the range in the order of their loads, conversions and MMAs: K of
  // a tile ahead of V of the tile before it (one buffer of Q: within a segment).
  // body(is_v, unit, tile, tiles before it, segment, the segment's first tile, its
  // last) until it returns false.
  auto for_each_item = [&](auto&& body) -> bool {
    if constexpr (!L::kTwo) {
      uint32_t J = 0;
      return for_each_segment([&](const TileUnit& un, int kt0, int kt1, int sg) -> bool {
        if (!body(false, un, kt0, J, sg, true, kt0 + 1 == kt1)) return false;
#pragma unroll 1
        for (int kt = kt0; kt < kt1; ++kt, ++J) {
          if (kt + 1 < kt1 && !body(false, un, kt + 1, J + 1, sg, false, kt + 2 == kt1)) return false;
          if (!body(true, un, kt, J, sg, kt == kt0, kt + 1 == kt1)) return false;
        }
        return true;
      });
    } else {
      TileUnit k, v;
      int k0, k1, v0, v1, kseg = 0, vseg = 0;
      uint32_t kj = 0, vj = 0;
      if (!get_segment(0, k, k0, k1)) return *abort_flag == 0;
      put_back(0);
      v = k;
      v0 = k0;
      v1 = k1;
      int kt = k0;
      bool more = true;
      while (true) {
        for (int vt = v0; vt < v1; ++vt, ++vj) {
#pragma unroll 1
          while (more && kj <= vj + 1) {
            if (!body(false, k, kt, kj, kseg, kt == k0, kt + 1 == k1)) return false;
            ++kj;
            if (++kt == k1) {
              more = get_segment(++kseg, k, k0, k1);
              kt = k0;
            }
          }
          if (!body(true, v, vt, vj, vseg, vt == v0, vt + 1 == v1)) return false;
        }
        if (!get_segment(++vseg, v, v0, v1)) return *abort_flag == 0;
        put_back(vseg);
      }
    }
  };
  // V's 64-element columns in an operand stage: each of 128 rows, or (copied 64
  // rows at a time) all columns of keys 0-63, then of 64-127.
  const bool v_halves = !kFp8 && box.all_cols && box.v_rows == 64;
  const uint32_t v_col = v_halves ? L::kVBox / 2 : L::kVBox;
  const uint32_t v_half = v_halves ? (D / 128) * (L::kVBox / 2) - 64 * 128 : 0;  // beyond 64 rows

  if (warp >= kProducerWarp && warp < kTilesConvWarp0) {
    setmaxnreg_dec<L::kControlRegs>();
    // Both roles walk with the whole warp and issue from one elected lane: in
    // code that only one lane runs, every operand of an MMA or a copy takes its
    // way through a vector register (100 cycles an MMA; the tensor cores waited).
    const bool elected = elect_one();
    if (warp == kProducerWarp || (L::kProducers == 2 && warp == kProducerWarp2)) {
      // --------------------------------------------------- TMA producers --
      // Their instructions set the pace of short tiles (with two divisions, a table
      // entry loaded and a modulus a copy, 1400 cycles an item): where a cursor
      // stands is carried on from item to item.
      const uint32_t mine = warp == kProducerWarp ? 0 : 1;
      if (elected) {
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
      }
      if (!p.batch.tables) grid_dependency_wait();  // the expanded copy is there
      const int bs = p.pool.block_size;
      // Where K and V (a tile behind) stand: a lane holds one of 32 entries of the
      // sequence's table from `first`; row `at` of page `lb` is next.
      struct Cursor {
        int seq = -1, first = 0, page = 0, key = -1, lb = 0, at = 0;
      } cur_k, cur_v;
      auto page_of = [&](Cursor& w) -> int {
        if (!p.batch.tables) return w.seq;  // the expanded copy
        if (w.lb < w.first || w.lb >= w.first + 32) {
          w.first = w.lb;
          w.page = w.lb + lane < p.batch.table_width ? p.batch.tables[w.seq * p.batch.table_stride + w.lb + lane] : -1;
        }
        int b = __shfl_sync(0xffffffffu, w.page, w.lb - w.first);
        if (b < 0 || b >= p.pool.blocks) {  // reported; block 0 keeps the load in bounds
          if (elected) atomicCAS(err, 0, kErrBlockTable);
          b = 0;
        }
        return b;
      };
      // Rows [key0, key0 + n) of K or V of one head; row 0 of `dst` is key0.
      // bf16: `full` is a cluster address.
      auto load_rows = [&](auto v, Cursor& w, const TileUnit& un, int key0, int n, uint32_t dst, uint32_t full) {
        constexpr bool is_v = decltype(v)::value;
        const int step = is_v ? box.v_rows : box.k_rows;
        if (w.seq != un.seq || w.key != key0) {
          if (w.seq != un.seq) w.first = INT_MIN;
          w.seq = un.seq;
          w.lb = key0 / bs;
          w.at = key0 - w.lb * bs;
        }
        for (int r = 0; r < n; r += step) {
          const int pg = page_of(w);
          if (elected) {
            if (kFp8) {
              if (is_v)
                tma_load_5d(dst + r * (D / 2), &tm_v, static_cast<int>(rank) * (D / 2), w.at, un.head, 1, pg, full);
              else
                tma_load_5d(dst + r * D, &tm_k, 0, w.at, un.head, 0, pg, full);
            } else if (box.all_cols) {  // {64 elements, rows, columns, head, 2 page + K/V}
              if (is_v)
                tma_load_5d_pair(dst + r * D, &tm_v, 0, w.at, static_cast<int>(rank) * (D / 128), un.head, 2 * pg + 1, full);
              else
                tma_load_5d_pair(dst, &tm_k, 0, w.at, 0, un.head, 2 * pg, full);
            } else if (is_v) {
              for (int b = 0; b < D / 128; ++b)
                tma_load_5d_pair(dst + b * L::kVBox + r * 128, &tm_v, 0, w.at, static_cast<int>(rank) * (D / 128) + b,
                                 un.head, 2 * pg + 1, full);
            } else {
              for (int b = 0; b < D / 64; ++b)
                tma_load_5d_pair(dst + b * L::kKBox + r * 128, &tm_k, 0, w.at, b, un.head, 2 * pg, full);
            }
          }
          w.at += step;  // a divisor of the page's rows
          if (w.at == bs) {
            w.at = 0;
            ++w.lb;
          }
        }
        w.key = -1;
        if (n == (is_v ? 128 : 64)) {  // on to the next tile
          w.key = key0 + kTileN;
          if (!is_v)
            for (w.at += 64; w.at >= bs; w.at -= bs) ++w.lb;
        }
      };
      uint32_t c = 0, parity = 1;
      int st = 0;
      const uint32_t own_bars = kFp8 ? bars : mapa_shared(bars, rank), leader_bars = mapa_shared(bars, 0);
      auto issue = [&](auto v, Cursor& w, const TileUnit& un, int kt) {
        constexpr bool is_v = decltype(v)::value;
        if (c % L::kProducers != mine) return true;
        const uint32_t empty = kFp8 ? bar_land_empty(st) : bar_op_empty(st);
        if (!__all_sync(0xffffffffu, mbar_wait(empty, parity, abort_flag, err, kErrWaitKvEmpty))) return false;
        const uint32_t dst = kFp8 ? sRaw + st * L::kRawBytes : sOp + st * L::kOpBytes;
        constexpr int row_bytes = (is_v ? D / 2 : D) * (kFp8 ? 1 : 2), most = is_v ? 128 : 64;
        const int valid = tile_valid(un, kt);
        const int off = is_v ? 0 : 64 * static_cast<int>(rank);
        const int n = min(most, max(0, valid - off));
        // Bytes of CTA rk's half, in whole copies (a power of two of rows).
        auto bytes_of = [&](int rk) {
          const int step = is_v ? box.v_rows : box.k_rows;
          return ((min(most, max(0, valid - (is_v ? 0 : 64 * rk))) + step - 1) & -step) * row_bytes;
        };
        uint32_t full;
        if (kFp8 || (is_v && edge(un, kt))) {  // to this CTA's converters
          if (elected) mbar_arrive_expect_tx(bar_land_full(st), bytes_of(static_cast<int>(rank)));
          full = own_bars + (bar_land_full(st) - bars);
        } else {
          if (leader && elected) {
            mbar_arrive_expect_tx(bar_op_full(st), valid >= kTileN ? 2 * most * row_bytes : bytes_of(0) + bytes_of(1));
            mbar_arrive(bar_op_full(st));
          }
          full = leader_bars + (bar_op_full(st) - bars);
        }
        load_rows(v, w, un, kt * kTileN + off, n, dst, full);
        return true;
      };
      const bool ok = for_each_item([&](bool is_v, const TileUnit& un, int kt, uint32_t, int, bool, bool) {
        if (!(is_v ? issue(std::true_type(), cur_v, un, kt) : issue(std::false_type(), cur_k, un, kt))) return false;
        ++c;
        if (++st == NL) {
          st = 0;
          parity ^= 1u;
        }
        return true;
      });
      // After a failure: let the copies still in flight land (bf16: those of both
      // CTAs are counted on the leader).
      if (!ok && elected && (kFp8 || leader))
        for (uint32_t i = (c > (uint32_t)NL ? c - NL : 0); i < c; ++i)
          if (i % L::kProducers == mine) mbar_wait_teardown(kFp8 ? bar_land_full(i % NL) : bar_op_full(i % NL), (i / NL) & 1u);
    }
    if (warp == kSegmentWarp) {
      // ------------- walks the range; Q, where a copy brings it --
      // Rows token * group + head of a unit as boxes of {64 elements, group, 128 /
      // group tokens, two columns}; tokens past the sequence bring other rows,
      // whose results nobody reads.  Both CTAs' bytes count on the leader.
      ChunkWalk<true> walk;
      walk.init(p, plan, err);
      TileUnit un;
      int kt0, kt1, sg = 0, landed = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, kErrWaitQ));
      };
      for (;; ++sg) {
        const bool more = walk.next(p, err, un, kt0, kt1);
        if (more) {
          un.see_all = keys_all_see(un.kvlen, un.qlen, un.row0, p.group);
          un.see_any = keys_all_see(un.kvlen, un.qlen, un.row0 + un.rows - 1, p.group);
        }
        if (sg >= kTileSegments) ok = wait(bar_seg_empty(sg), ((sg / kTileSegments) & 1u) ^ 1u);
        if (!ok) break;
        if (elected) {
          TileSegment& s = segments[sg % kTileSegments];
          s.un = un;
          s.kt0 = kt0;
          s.kt1 = more ? kt1 : 0;
          mbar_arrive(bar_seg_full(sg));
        }
        if (!more) break;
        if (!box.q_copy) continue;
        if (sg >= L::kQBufs) ok = wait(bar_q_empty(sg - L::kQBufs), ((sg - L::kQBufs) >> 1) & 1u);
        if (!ok) break;
        if (elected) {
          if (leader) mbar_arrive_expect_tx(bar_q_ready(sg), 2 * L::kQBytes);
          const int token = un.q0 + un.row0 / p.group + static_cast<int>(rank) * (kTileM / p.group);
          for (int b = 0; b < D / 64; b += 2)
            tma_load_5d_pair(sQ + (L::kQBufs > 1 ? (sg & 1) * L::kQBytes : 0) + b * kBoxBytes, &tm_q, 0, 0, token, b,
                             un.head, mapa_shared(bar_q_ready(sg), 0));
        }
        landed = sg + 1;
      }
      // Let the copies land, if nobody waits for them any more.
      if ((!ok || *abort_flag) && leader && elected)
        for (int i = max(0, landed - L::kQBufs); i < landed; ++i) mbar_wait_teardown(bar_q_ready(i), (i >> 1) & 1u);
    }
    if (warp == kMmaWarp && !leader) for_each_segment([](const TileUnit&, int, int, int) { return true; });
    if (warp == kMmaWarp && leader) {
      // ------------------------------------------ MMA issuer (leader only) --
      constexpr uint32_t idesc_qk =
          kFp8 ? make_idesc_f16(kUnitRows, kTileN, false, false) : make_idesc_bf16(kUnitRows, kTileN, false, false);
      constexpr uint32_t idesc_pv =
          kFp8 ? make_idesc_f16(kUnitRows, D, false, true) : make_idesc_bf16(kUnitRows, D, false, true);
      uint32_t c = 0;
      auto wait = [&](uint32_t bar, uint32_t parity, int code) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code));
      };
      // Descriptors of the first k step; the others differ in the address alone.
      const uint64_t q_desc0 = make_sw128_desc(sQ, 16, 1024);
      const uint64_t k_desc = make_sw128_desc(sOp, 16, 1024);
      const uint64_t v_desc = make_sw128_desc(sOp, v_col, 1024);
      auto qk = [&](uint32_t jg, int seg) {
        const uint64_t q_desc = q_desc0 + (L::kQBufs > 1 ? (seg & 1) * (L::kQBytes >> 4) : 0);
        const uint32_t s_tmem = tmem + kTmemS0 + (jg & 1) * kTileN;
        const int st = c % NS;
        if (!wait(bar_op_full(st), (c / NS) & 1u, kErrWaitKvFull)) return false;
        tc_fence_after();
        const uint64_t kd = k_desc + static_cast<uint32_t>(st) * (L::kOpBytes >> 4);
        if (elected) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_ss_pair(s_tmem, q_desc + (((kk / 4) * kBoxBytes + (kk % 4) * 32) >> 4),
                         kd + (((kk / 4) * L::kKBox + (kk % 4) * 32) >> 4), idesc_qk, kk != 0 ? 1u : 0u);
          umma_commit_pair(bar_op_empty(st), kChunkBothCtas);
          umma_commit_pair(bar_s_full(jg & 1), kChunkBothCtas);
        }
        ++c;
        return true;
      };
      auto pv = [&](uint32_t jg, bool first, bool last, int seg) {
        // The output of the segment that had this accumulator has been read.
        constexpr int kO = L::kTwo ? 2 : 1;
        if (first && seg >= kO && !wait(bar_o_free(seg - kO), ((seg - kO) / kO) & 1u, kErrWaitODone)) return false;
        if (!wait(bar_p_full(jg & 1), (jg >> 1) & 1u, kErrWaitPFull)) return false;
        const int st = c % NS;
        if (!wait(bar_op_full(st), (c / NS) & 1u, kErrWaitKvFull)) return false;
        tc_fence_after();
        const uint32_t p_tmem = tmem + kTmemS0 + (jg & 1) * kTileN;
        const uint32_t o_tmem = tmem + (L::kTwo ? (seg & 1) * D : 0);
        const uint64_t vd = v_desc + static_cast<uint32_t>(st) * (L::kOpBytes >> 4);
        const uint64_t vd2 = vd + (v_half >> 4);
        if (elected) {
#pragma unroll
          for (int kk = 0; kk < kTileN / 16; ++kk) {
            // A = P (over S, each warpgroup's in its own half), B = V half, MN-major:
            // 64-dim chunks v_col apart, 8-key groups 1 KB apart.
            umma_ts_pair(o_tmem, p_tmem + kk * 8 + (kk >= 4 ? 32 : 0), (kk >= 4 ? vd2 : vd) + kk * (2048 >> 4),
                         idesc_pv, (!first || kk > 0) ? 1u : 0u);
          }
          umma_commit_pair(bar_op_empty(st), kChunkBothCtas);
          umma_commit_pair(bar_o(jg & 1), kChunkBothCtas);
          if (L::kTwo && last) umma_commit_pair(bar_seg_o(seg), kChunkBothCtas);
        }
        ++c;
        return true;
      };
      for_each_item([&](bool is_v, const TileUnit&, int, uint32_t J, int seg, bool first, bool last) {
        if (is_v) return pv(J, first, last, seg);
        if (first) {
          if (!wait(bar_q_ready(seg), (seg >> 1) & 1u, kErrWaitQ)) return false;
          tc_fence_after();
        }
        if (!qk(J, seg)) return false;
        if (last && elected) umma_commit_pair(bar_q_empty(seg), kChunkBothCtas);
        return true;
      });
      // Drain: completes when every MMA issued above has.
      if (elected) {
        umma_commit_pair(bar_td, kChunkLeader);
        mbar_wait_teardown(bar_td, 0);
      }
    }
    __syncwarp();
  } else if (warp >= kTilesConvWarp0) {
    setmaxnreg_dec<L::kConvRegs>();
    // ----------- Q gather, e4m3 -> f16, V past the end; D = 128: the output --
    const int ct = threadIdx.x - kTilesConvWarp0 * 32;
    const int cw = warp - kTilesConvWarp0;
    const ConvGeo geo_k = conv_geo(ct, D / 64, L::kKBox);
    const ConvGeo geo_v = conv_geo(ct, D / 128, L::kVBox);
    uint32_t c = 0, J = 0;
    int segs = 0;
    auto wait_all = [&](uint32_t bar, uint32_t parity, int code) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code));
    };
    auto item = [&](const TileUnit& un, bool is_v, int kt) -> bool {
      const int ls = c % NL, os = c % NS;
      const int valid = tile_valid(un, kt);
      if (kFp8) {
        if (kScaled && !is_v) {  // this tile's scales: a key a thread
          const int key = kt * kTileN + ct;
          uint32_t kb = 127, vb = 127;
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
          sf[kTileN + ct] = exponent_of_scale(vb);
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
        const int vrows = is_v ? min(valid, un.see_any - kt * kTileN) : valid - 64 * static_cast<int>(rank);
        const int look = is_v ? un.see_all - kt * kTileN : kTileN;  // rows to look through
        bool found = false;
        const int row_step = is_v ? 64 / (D / 64) : 32 / (D / 64);
        const uint32_t op_step = row_step * 128;
#pragma unroll 1
        for (int m0 = 0; m0 < D / 32; m0 += 4) {
          uint4 x[4];
#pragma unroll
          for (int m = 0; m < 4; ++m)
            x[m] = g.row + (m0 + m) * row_step < vrows ? lds128(raw + g.raw + (m0 + m) * 2048) : zero;
          if (look < kTileN) {
#pragma unroll
            for (int m = 0; m < 4; ++m)
              if (g.row + (m0 + m) * row_step >= look) found |= drop_nonfinite<true>(x[m]);
          }
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            uint4 lo, hi;
            e4m3x16_to_f16(x[m], lo, hi);
            const uint32_t o = op + (m0 + m) * op_step;
            sts128(o + g.lo, lo);
            sts128(o + g.hi, hi);
          }
        }
        if (found) *patch = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_land_empty(ls));
          mbar_arrive_remote(mapa_shared(bar_op_full(os), 0));
        }
      }
      ++c;
      return true;
    };
    auto gather_q = [&](const TileUnit& un) -> bool {
      // Q rows into the swizzled operand layout: a row over D / 8 lanes,
      // kFlight loads a lane in flight, the first of them before the wait for the
      // previous segment's QK^T to be done with the buffer.
      constexpr int kSide = 256 / D;  // rows side by side in a warp
      constexpr int kFlight = 4;
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
        if (r0 == cw * 32 && segs >= L::kQBufs && !wait_all(bar_q_empty(segs - L::kQBufs), ((segs - L::kQBufs) >> 1) & 1u, kErrWaitQ))
          return false;
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
            if (ch == 0) factors[(segs & (L::kSegBufs - 1)) * kTileM + r] = p.scale_log2 * exp2_of_int(e);
            x[u] = make_uint4(pack_f16x2(f[0] * down, f[1] * down), pack_f16x2(f[2] * down, f[3] * down),
                              pack_f16x2(f[4] * down, f[5] * down), pack_f16x2(f[6] * down, f[7] * down));
          }
          sts128(sQ + (L::kQBufs > 1 ? (segs & 1) * L::kQBytes : 0) + (ch / 8) * kBoxBytes + r * 128 + (((ch % 8) ^ (r & 7)) << 4), x[u]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_rows(segs));
        mbar_arrive_remote(mapa_shared(bar_q_ready(segs), 0));
      }
      ++segs;
      return true;
    };
    // kTwo: the output of segment sg.  Called once all that its last PV waits for is
    // on its way, Q and the first K of the next segment included.
    const float* seg_sums = red + L::kMaxima * kTileM;  // [kSegBufs]{l of either warpgroup, its reference, (scaled) m}[128]
    auto write_out = [&](const TileUnit& un, int kt0, int kt1, int sg) -> bool {
      if (!wait_all(bar_sums(sg), (sg / L::kSegBufs) & 1u, kErrWaitRed) ||
          !wait_all(bar_seg_o(sg), (sg >> 1) & 1u, kErrWaitODone))
        return false;
      tc_fence_after();
      const float* sums = seg_sums + (sg & (L::kSegBufs - 1)) * L::kSums * kTileM;
      const float l = sums[ct] + sums[kTileM + ct], ref = sums[2 * kTileM + ct];
      // No key seen: zeros.
      const float inv_l = l == 0.f ? 0.f : kScaled ? output_factor(sums[(L::kSums - 1) * kTileM + ct], ref, l)
                                                  : v_factor / l;
      const int r = static_cast<int>(rank) * kTileM + ct;  // row of the unit
      const bool live = r < un.rows;
      const uint32_t t_o = tmem + (static_cast<uint32_t>(cw * 32) << 16) + (sg & 1) * D;
      const int slot = part_slot(un, kt0, kt1, pair);
      if (slot < 0) {
        const int at = un.row0 + r;
        __nv_bfloat16* out = p.out + static_cast<long long>(un.head * p.group + at % p.group) * p.out_head +
                             static_cast<long long>(un.q0 + at / p.group) * p.out_row;
        store_rows<D>(t_o, inv_l, live ? out : nullptr, lane);
      } else {
        const long long pr = static_cast<long long>(slot) * kUnitRows + r;
        if (live) p.work.tile_lse[pr] = l == 0.f ? -INFINITY : ref + __log2f(l);
        store_rows<D>(t_o, inv_l, live ? p.work.tile_o + pr * D : nullptr, lane);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(mapa_shared(bar_o_free(sg), 0));
      return true;
    };
    TileUnit last_un;
    int last0 = 0, last1 = 0, last_seg = -1;
    auto write_last = [&]() { return !L::kTwo || last_seg < 0 || write_out(last_un, last0, last1, last_seg); };
    bool ok;
    if constexpr (kFp8) {
      ok = for_each_item([&](bool is_v, const TileUnit& un, int kt, uint32_t, int seg, bool first, bool last) {
        if (!is_v && first && !gather_q(un)) return false;
        if (!item(un, is_v, kt)) return false;
        if (L::kTwo && is_v) {
          if (first) {
            if (!write_last()) return false;
            last_un = un;
            last0 = kt;
            last_seg = seg;
          }
          if (last) last1 = kt + 1;
        }
        return true;
      });
    } else {
      // V of edge tiles: rows that no row of the unit sees become zeros (those
      // past the sequence's end may hold anything), values that are not finite
      // in rows that only some see too.  An item's stage follows from its place
      // in the order of for_each_item.
      const uint32_t tiles = static_cast<uint32_t>(plan.end - plan.x);
      uint32_t J = 0, used = 0;  // bit st: parity of stage st's landings so far
      ok = for_each_segment([&](const TileUnit& un, int kt0, int kt1, int seg) -> bool {
        if (!box.q_copy && !gather_q(un)) return false;
        if (L::kTwo) {
          if (!write_last()) return false;
          last_un = un;
          last0 = kt0;
          last1 = kt1;
          last_seg = seg;
        }
        for (int kt = max(kt0, max(0, un.see_all) / kTileN); kt < kt1; ++kt) {
          const uint32_t j = kt - kt0;
          const uint32_t at = L::kTwo ? J + j + min(J + j + 2, tiles) : 2 * (J + j) + (kt + 1 < kt1 ? 2 : 1);
          const int st = at % NS;
          if (!wait_all(bar_land_full(st), (used >> st) & 1u, kErrWaitKvFull)) return false;
          used ^= 1u << st;
          const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
          const uint32_t op = sOp + st * L::kOpBytes;
          bool found = false;
          for (int i = max(0, un.see_all - kt * kTileN) * 8 + ct; i < kTileN * 8; i += kTilesConvThreads) {
            const bool seen = kt * kTileN + i / 8 < un.see_any;
            for (int b = 0; b < D / 128; ++b) {
              const uint32_t a = op + b * v_col + (i >= 64 * 8 ? v_half : 0) + i * 16;
              uint4 x = seen ? lds128(a) : zero;
              if (seen) {
                if (!drop_nonfinite<false>(x)) continue;
                found = true;
              }
              sts128(a, x);
            }
          }
          if (found) *patch = 1;
          fence_proxy_async_smem();
          named_bar_sync(3, kTilesConvThreads);
          if (ct == 0) mbar_arrive_remote(mapa_shared(bar_op_full(st), 0));
        }
        J += kt1 - kt0;
        return true;
      });
    }
    if (ok) write_last();
    __syncwarp();
  } else {
    setmaxnreg_inc<L::kSoftmaxRegs>();
    // ---------------------------------------- softmax / correction / epilogue --
    constexpr int kOCols = D / 2;
    constexpr int kKeys = kTileN / 2;  // a thread's keys of a tile
    const int wg = warp >> 2;
    const int row = threadIdx.x & (kTileM - 1);  // == TMEM lane
    const uint32_t t_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float* sums = red;  // (one accumulator: a segment's sums, once its maxima were read)
    uint32_t J = 0;
    // The leader keeps the pair's record.
    ChunkRecord& rec = p.work.tile_rec[pair];
    const bool keeps = leader && threadIdx.x == 0;
    if (keeps) clear_record(rec);
    for_each_segment([&](const TileUnit& un, int kt0, int kt1, int seg) -> bool {
      if (keeps) note_part(rec, un, kt0, kt1);
      bool ok = true;
      const int r = static_cast<int>(rank) * kTileM + row;  // row of the unit
      const bool live = r < un.rows;
      const int at = un.row0 + (live ? r : un.rows - 1);
      const int pos = un.kvlen - un.qlen + at / p.group;  // last key this row sees
      const uint32_t Jend = J + (kt1 - kt0);
      const uint32_t t_o = t_row + (L::kTwo ? (seg & 1) * D : 0) + wg * kOCols;
      float rf = p.scale_log2;
      if (kFp8) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_rows(seg), (seg / L::kSegBufs) & 1u, abort_flag, err, kErrWaitQ));
        if (ok) rf = factors[(seg & (L::kSegBufs - 1)) * kTileM + row];
      }
      float m = -INFINITY;  // reference of both halves, log2 units (kScaled: V's exponents included)
      float ref = -INFINITY;  // kScaled: l's own reference (chunk_rows.cuh), scores alone
      float l = 0.f;          // this half's weights, over 2^m or 2^ref

      // This thread's scores of tile jg: loaded, keys past the row's position at
      // -inf; kScaled: in log2 units (the row's factor first: it is below 1 for queries up
      // to 2^17, so that large K scales do not overflow), else without the row's factor.
      const uint32_t first_key = wg * kKeys;
      auto scores = [&](uint32_t jg, float (&s)[kKeys]) -> bool {
        if (!__all_sync(0xffffffffu, mbar_wait(bar_s_full(jg & 1), (jg >> 1) & 1u, abort_flag, err, kErrWaitSFull)))
          return false;
        tc_fence_after();
        const uint32_t t_s = t_row + kTmemS0 + (jg & 1) * kTileN + first_key;
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) tmem_ld32(t_s + 32 * c, s + 32 * c);
        tmem_wait_ld();
        if (kScaled) {
          if (!__all_sync(0xffffffffu, mbar_wait(bar_scale(jg % (NB ? NB : 1)), (jg / (NB ? NB : 1)) & 1u, abort_flag,
                                                 err, kErrWaitKvFull)))
            return false;
          const float* sf = reinterpret_cast<const float*>(smem + L::kScaleOff + (jg % (NB ? NB : 1)) * L::kScaleBuf);
          const float4* ks = reinterpret_cast<const float4*>(sf + first_key);
          const f32x2 rf2 = pcp::pair(rf, rf);
#pragma unroll
          for (int i = 0; i < kKeys / 4; ++i) {
            const float4 k4 = ks[i];
            split(mul2(mul2(pcp::pair(s[4 * i], s[4 * i + 1]), rf2), pcp::pair(k4.x, k4.y)), s[4 * i], s[4 * i + 1]);
            split(mul2(mul2(pcp::pair(s[4 * i + 2], s[4 * i + 3]), rf2), pcp::pair(k4.z, k4.w)), s[4 * i + 2],
                  s[4 * i + 3]);
          }
        }
        const int visible = pos + 1 - (kt0 + static_cast<int>(jg - J)) * kTileN - static_cast<int>(first_key);
        if (visible < kKeys) {
#pragma unroll
          for (int i = 0; i < kKeys; ++i)
            if (i >= visible) s[i] = -INFINITY;
        }
        return true;
      };
      // The largest score + V exponent of this thread's keys of tile jg (kScaled).
      auto top = [&](uint32_t jg, const float (&s)[kKeys]) -> float {
        const float4* ve = reinterpret_cast<const float4*>(smem + L::kScaleOff + (jg % (NB ? NB : 1)) * L::kScaleBuf) +
                           (kTileN + first_key) / 4;
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < kKeys / 4; ++i) {
          const float4 e = ve[i];
          mx0 = fmaxf(mx0, fmaxf(s[4 * i] + e.x, s[4 * i + 1] + e.y));
          mx1 = fmaxf(mx1, fmaxf(s[4 * i + 2] + e.z, s[4 * i + 3] + e.w));
        }
        return fmaxf(mx0, mx1);
      };
      // P = 2^(s rf - m), kScaled 2^(s + V's exponent - m), into TMEM columns
      // [t_p, t_p + kKeys / 2); returns the sum of P, kScaled of 2^(s - ref).
      // A row that has seen nothing yet has only -inf scores.
      auto probs = [&](uint32_t jg, const float (&s)[kKeys], uint32_t t_p) -> float {
        const float* sf = reinterpret_cast<const float*>(smem + L::kScaleOff + (jg % (NB ? NB : 1)) * L::kScaleBuf);
        const float neg = m == -INFINITY ? 0.f : -m, neg_ref = ref == -INFINITY ? 0.f : -ref;
        const f32x2 rf2 = pcp::pair(rf, rf), neg2 = pcp::pair(neg, neg), neg_ref2 = pcp::pair(neg_ref, neg_ref);
        f32x2 sum = pcp::pair(0.f, 0.f);
#pragma unroll
        for (int c2 = 0; c2 < kKeys / 32; ++c2) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float q0, q1, q2, q3;
            const f32x2 s0 = pcp::pair(s[c2 * 32 + 2 * i], s[c2 * 32 + 2 * i + 1]);
            const f32x2 s1 = pcp::pair(s[c2 * 32 + 2 * i + 2], s[c2 * 32 + 2 * i + 3]);
            split(kScaled ? add2(s0, neg_ref2) : fma2(s0, rf2, neg2), q0, q1);
            split(kScaled ? add2(s1, neg_ref2) : fma2(s1, rf2, neg2), q2, q3);
            q0 = ex2_approx(q0);
            q1 = ex2_approx(q1);
            q2 = ex2_approx(q2);
            q3 = ex2_approx(q3);
            sum = add2(sum, add2(pcp::pair(q0, q1), pcp::pair(q2, q3)));
            if (kScaled) {
              const float4 e = *reinterpret_cast<const float4*>(sf + kTileN + first_key + c2 * 32 + 2 * i);
              split(add2(add2(s0, pcp::pair(e.x, e.y)), neg2), q0, q1);
              split(add2(add2(s1, pcp::pair(e.z, e.w)), neg2), q2, q3);
              q0 = ex2_approx(q0);
              q1 = ex2_approx(q1);
              q2 = ex2_approx(q2);
              q3 = ex2_approx(q3);
            }
            pk[i] = kFp8 ? pack_f16x2(q0, q1) : pack_bf16x2(q0, q1);
            pk[i + 1] = kFp8 ? pack_f16x2(q2, q3) : pack_bf16x2(q2, q3);
          }
          tmem_st16(t_p + c2 * 16, pk);
        }
        tmem_wait_st();
        float sum0, sum1;
        split(sum, sum0, sum1);
        return sum0 + sum1;
      };
      auto release = [&](uint32_t jg) {  // tile jg's P is in place
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(bar_p_full(jg & 1), 0));
      };
      // The reference moves when a tile's largest weight would pass 2^8 (and
      // from its start, as soon as a key is seen); O of the tiles before goes
      // over to the new one once their last product is in it.
      for (uint32_t jg = J; jg < Jend && ok; ++jg) {
        const int b = jg & 1;
        float s[kKeys];
        ok = scores(jg, s);
        if (!ok) break;
        const float pmax = kScaled ? top(jg, s) : row_max(s);
        const float smax = kScaled ? row_max(s) : pmax;
        red[(b * 2 + wg) * kTileM + row] = pmax;
        if (kScaled) red[(4 + b * 2 + wg) * kTileM + row] = smax;
        mbar_arrive(bar_ref(b));
        // Pass 0 (tiles after the first): speculative P with the current
        // reference, before the other half's maximum is known.  Pass 1:
        // exchange the half maxima; P is recomputed only when some row's
        // moved past the threshold.
        float tile_sum = 0.f;
        float alpha = 1.f;
        bool moved = false;
#pragma unroll 1
        for (int pass = jg > J ? 0 : 1; pass < 2; ++pass) {
          if (pass == 1) {
            ok = __all_sync(0xffffffffu, mbar_wait(bar_ref(b), (jg >> 1) & 1u, abort_flag, err, kErrWaitRed));
            if (!ok) break;
            const float both = fmaxf(pmax, red[(b * 2 + (wg ^ 1)) * kTileM + row]);
            const float tmax = kScaled ? both : both * rf;
            const bool need = tmax > m + kRescaleThreshold;
            moved = __any_sync(0xffffffffu, need);
            bool redo = moved || jg == J;
            if (need) {
              alpha = ex2_approx(m - tmax);  // 0 from the start
              m = tmax;
              if (!kScaled) l *= alpha;
            }
            if (kScaled) {
              const float most = fmaxf(smax, red[(4 + b * 2 + (wg ^ 1)) * kTileM + row]);
              const bool raise = most > ref + kRescaleThreshold;
              redo |= __any_sync(0xffffffffu, raise);
              if (raise) {
                l *= ex2_approx(ref - most);
                ref = most;
              }
            }
            if (!redo) break;
          }
          tile_sum = probs(jg, s, t_row + kTmemS0 + b * kTileN + wg * kKeys);
        }
        if (!ok) break;
        l += tile_sum;
        if (jg > J && moved) {
          ok = __all_sync(0xffffffffu,
                          mbar_wait(bar_o((jg - 1) & 1), ((jg - 1) >> 1) & 1u, abort_flag, err, kErrWaitODone));
          if (!ok) break;
          tc_fence_after();
          rescale_o<kOCols>(t_o, alpha);
        }
        release(jg);
      }
      const uint32_t jl = Jend - 1;  // the last tile
      J = Jend;
      if constexpr (L::kTwo) {
        if (!ok) return false;
        float* part = red + (L::kMaxima + (seg & (L::kSegBufs - 1)) * L::kSums) * kTileM;
        part[wg * kTileM + row] = l;
        if (wg == 0) part[2 * kTileM + row] = kScaled ? ref : m;
        if (wg == 0 && kScaled) part[3 * kTileM + row] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_sums(seg));
        return true;
      } else {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar_o(jl & 1), (jl >> 1) & 1u, abort_flag, err, kErrWaitODone));
        sums[wg * kTileM + row] = l;
        ok = named_bar_and(1, kSoftmaxThreads, ok && (*abort_flag == 0));
        if (!ok) return false;
        tc_fence_after();
        l += sums[(wg ^ 1) * kTileM + row];
        // Both read: the next segment may reuse the slots.
        named_bar_sync(2, kSoftmaxThreads);
        const float inv_l = l == 0.f ? 0.f : kScaled ? output_factor(m, ref, l) : v_factor / l;  // no key seen: zeros
        const int slot = part_slot(un, kt0, kt1, pair);
        if (slot < 0) {
          __nv_bfloat16* out = p.out + static_cast<long long>(un.head * p.group + at % p.group) * p.out_head +
                               static_cast<long long>(un.q0 + at / p.group) * p.out_row;
          store_rows<kOCols>(t_o, inv_l, live ? out + wg * kOCols : nullptr, lane);
        } else {
          const long long pr = static_cast<long long>(slot) * kUnitRows + r;
          if (live && wg == 0) p.work.tile_lse[pr] = l == 0.f ? -INFINITY : (kScaled ? ref : m) + __log2f(l);
          store_rows<kOCols>(t_o, inv_l, live ? p.work.tile_o + pr * D + wg * kOCols : nullptr, lane);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(bar_o_free(seg), 0));
        return true;
      }
    });
  }

  // Both CTAs: the leader's MMAs (which read the peer's smem and TMEM) are
  // drained, every TMEM read of either CTA is done.
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  grid_dependency_wait();  // the small units: the merge waits for them through this kernel
  if (threadIdx.x == 0) {
    p.work.tile_rec[blockIdx.x].err = *static_cast<volatile int*>(err);
    p.work.tile_rec[blockIdx.x].failed = *abort_flag;  // (nothing of the range is merged then)
    p.work.tile_rec[blockIdx.x].patch = *patch;
  }
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, kTmemCols);
  }
}

}  // namespace pcp
