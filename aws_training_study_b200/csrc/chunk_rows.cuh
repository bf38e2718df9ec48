// Attention of a few query rows (a KV head's group of queries of one token, or
// of a few drafted ones: at most kSmallRows) over a long paged cache.
//
// Bound by reading the cache: 4 rows' flops a byte are far below what the
// tensor cores need, so the cache must stream at HBM's rate and everything else
// hide behind it.  A 128-row tcgen05 tile would spend its time on empty rows
// (the tile kernel reads 2.4 TB/s on such a unit); here a warp's mma.sync tile is
// 16 rows, which one token's group of heads fills, and warps split the KEYS:
//   * A producer warp streams 32 KB stages (K and V of one head) through a ring of
//     four or five with TMA.  A copy and what surrounds it cost its issuer some 300 cycles
//     whatever its size, and the SM's share of HBM is 7 KB in that time: so one
//     copy brings all of a stage's rows that share a page (16 to 128: pages of any
//     multiple of 16 tokens), K and V together, 128-byte columns swizzled for the
//     MMAs.
//   * Teams of D / 128 warps take 16 keys each in turn: a team scores its keys
//     against all rows and adds P V into its own accumulators, with its own running
//     maximum, so teams exchange nothing until the unit ends.  Within a team of
//     two each warp has half the columns: half the terms of the scores, which
//     are summed through shared memory, and half the output.  128 columns are
//     what lets 12 such warps live on an SM (64 accumulators a thread): one
//     warp with all 256 columns at two warps a scheduler spilled, and read 2.0
//     TB/s where this reads 3.9.  17 to 32 rows are two row tiles, each with half
//     the teams, on the same stages.
//   * The teams' (m, l, O) are merged through shared memory when the unit's part
//     ends, into bf16 rows or an fp32 partial.
// 64 sequences of 4096 (bf16, 32 / 8 heads of 128): 5.6 TB/s, 86 % of a copy's rate.
// 16 of 32768 (e4m3 with scales, 32 / 2 heads of 256): 3.8 TB/s, bound by issue and
// latency (half of the issue slots; conversions and MMAs are half the instructions).
// Multiplying a visit's scores under the softmax of the one before held the stages
// longer and was slower (87 to 100 us, bf16 129 to 153).
//
// e4m3 codes become f16 in registers (exact) on their way into the MMA.  No
// ldmatrix: the order of an MMA's k index is free as long as both operands
// agree, so a lane takes 16 consecutive bytes of a K row as four k steps (Q's
// fragments are laid out to match), and of a V row as 16 output columns (pairs
// of keys are zipped with byte permutes).  All accesses hit distinct banks.
// Scales: K's 2^e multiplies its key's score, V's 2^e its key's weight, as part of
// the exponent: 2^(s + e - m), where m follows the largest s + e, key by key, that
// the row sees.  So the weights that enter f16 are at most 2^8, the largest contribution
// is 1 or more whatever the exponents, and a large V whose key weighs nothing takes
// nothing from the others (a reference of the largest s and the largest e, of
// different keys, did).  f16's 11 bits are three more than bf16's; contributions
// below 2^-24 of the largest are lost.  The sum of the weights, 2^(s - ref), has a
// reference of its own, a score that the row has seen (within 2^16 of the largest): under
// m it would sit at 2^-e, and an e of 120 flushed all but the largest weights, one of
// -100 left the sum little of fp32's range.  O's factor at the end is 2^(m - ref) / l.
// (One reference of largest score and largest exponent for both took 84.1 us for the
// 16 of 32768, a key's own sum 85.0, two references 86.4.)
// Q is brought to f16 by a power of two of its row.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "chunk_plan.cuh"

namespace pcp {

template <int D, bool kFp8>
struct RowsSmem {
  static constexpr int kElt = kFp8 ? 1 : 2;
  // Consumer warps.  bf16, which converts nothing: 8, and the producer, at up to
  // 168 registers.  e4m3: 12, and a warpgroup of its own for the producer, which
  // gives registers up: 384 x 152 + 128 x 56 = 512 x 128 (at 128 they spill).
  static constexpr int kWarps = kFp8 ? 12 : 8;
  static constexpr int kThreads = kFp8 ? 512 : 32 * kWarps + 32;
  static constexpr int kTeam = D / 128;          // warps of a team
  static constexpr int kTeams = kWarps / kTeam;
  static constexpr int kBoxes = D * kElt / 128;             // 128-byte columns of a row
  static constexpr int kStageBytes = 32768;
  static constexpr int kStageKeys = kStageBytes / (256 * kBoxes);  // 32 to 128
  static constexpr int kStages = kFp8 ? 4 : 5;  // bf16, which HBM bounds: 5 127.5 us, 4 128.4
  // Scale bytes of a stage: a copy's K rows, then its V rows, at 128-byte slots.
  static constexpr int kScaleStage = kFp8 ? kStageKeys / 16 * 128 : 0;
  // O exchange: 16 rows of D floats, 4 floats of padding every 32, rows 16
  // banks apart: a lane's 16-byte stores fall on distinct banks.
  static constexpr int kRowFloats = D + D / 8 + (D == 256 ? 16 : 0);
  static constexpr int kBufBytes = 16 * kRowFloats * 4;
  static constexpr int kBufs = kTeams / 2;
  static_assert(kTeams % 2 == 0, "two row tiles share the teams");
  static constexpr int kQOff = kStages * kStageBytes;
  static constexpr int kQBytes = 2 * 16 * D * 2;  // two row tiles in MMA fragment order
  static constexpr int kScaleOff = kQOff + kQBytes;
  static constexpr int kBufOff = kScaleOff + kStages * kScaleStage;
  // The halves of a team's scores, [2 slots][warp][2][lane][4] floats, use the
  // buffers' space before the merge.
  static constexpr int kRowOff = kBufOff + kBufs * kBufBytes;  // float score factor[32], int position[32]
  static constexpr int kMlOff = kRowOff + 2 * kSmallRows * 4;  // float m, l, l's reference: [team][16]
  static constexpr int kInvOff = kMlOff + 3 * kTeams * 16 * 4;  // float factor of O [32]
  static constexpr int kBarOff = kInvOff + kSmallRows * 4;  // full, empty
  static constexpr int kMiscOff = kBarOff + 2 * kStages * 8;
  static constexpr int kPlanOff = kMiscOff + 16;  // ChunkPlanShared
  static constexpr int kBytes = kPlanOff + sizeof(ChunkPlanShared);
  static_assert(kBytes <= 232448, "exceeds the 227 KB of shared memory per CTA");
  static_assert(kBufOff % 16 == 0 && kBarOff % 8 == 0 && kScaleOff % 128 == 0, "alignment");
  static_assert(2 * kWarps * 1024 <= kBufs * kBufBytes, "the score halves fit the buffers");
};

constexpr int kRowsLaunchRegs = 128, kRowsConsumerRegs = 152, kRowsProducerRegs = 56;
static_assert(384 * kRowsConsumerRegs + 128 * kRowsProducerRegs <= 512 * kRowsLaunchRegs, "more than the launch's registers");

template <bool kF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  if (kF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <int D, int kCache>
__global__ void __launch_bounds__(RowsSmem<D, kCache != kCacheBf16>::kThreads, 1)
    chunk_rows_kernel(const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ CUtensorMap tm_scale,
                      const int box_shift, const ChunkParams p) {
  constexpr bool kFp8 = kCache != kCacheBf16, kScaled = kCache == kCacheScaled;
  using L = RowsSmem<D, kFp8>;
  constexpr int kBoxElts = 128 / L::kElt;
  constexpr int kBoxSteps = kBoxElts / 16;  // MMA k steps of a box: 8 or 4
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  ChunkRecord& rec = p.work.small_rec[blockIdx.x];
  if (sbase & 1023u) {
    if (threadIdx.x == 0) {
      clear_record(rec);
      rec.err = kErrSmemAlign;
      rec.failed = 1;
    }
    return;
  }
  const uint32_t sQ = sbase + L::kQOff;
  const uint32_t sScale = sbase + L::kScaleOff;
  float* row_factor = reinterpret_cast<float*>(smem + L::kRowOff);
  int* row_pos = reinterpret_cast<int*>(smem + L::kRowOff) + kSmallRows;
  float* s_m = reinterpret_cast<float*>(smem + L::kMlOff);
  float* s_l = s_m + L::kTeams * 16;
  float* s_ref = kScaled ? s_l + L::kTeams * 16 : s_m;
  float* s_inv = reinterpret_cast<float*>(smem + L::kInvOff);
  auto bar_full = [&](int s) { return sbase + L::kBarOff + 8u * s; };
  auto bar_empty = [&](int s) { return sbase + L::kBarOff + 8u * (L::kStages + s); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff);
  ChunkPlanShared& plan = *reinterpret_cast<ChunkPlanShared*>(smem + L::kPlanOff);
  int* err = &plan.err;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(bar_full(s), 1);
      // Every consumer warp sees every filling of every stage, its keys in it
      // or not: the barrier's parity could not tell two fillings apart otherwise.
      mbar_init(bar_empty(s), L::kWarps);
    }
    *abort_flag = 0;
    *reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4) = 0;
    plan.err = 0;
    fence_mbar_init();
  }
  if (warp == L::kWarps && lane == 0) {
    tma_prefetch_desc(&tm_kv);
    if (kScaled) tma_prefetch_desc(&tm_scale);
  }
  grid_launch_dependents();  // the merge may wait on the SMs
  __syncthreads();
  chunk_plan<false>(p, plan, p.small_ctas, blockIdx.x);
  ChunkWalk<false> walk;
  walk.init(p, plan, err);
  ChunkUnit un;
  int kt0, kt1;
  uint32_t c = 0;  // stages of this CTA so far
  const int box_rows = 1 << box_shift;  // rows (keys) of a copy
  const uint32_t box_bytes = 256 * L::kBoxes * box_rows, scale_slot = max(128, 2 * box_rows);

  if (warp >= L::kWarps) {
    // -------------------------------------------------------- producer --
    if (kFp8) setmaxnreg_dec<kRowsProducerRegs>();
    if (warp > L::kWarps) return;
    // The whole warp walks and waits, one elected lane issues (chunk_tiles.cuh).
    const bool elected = elect_one();
    bool ok = true;
    const int bs = p.pool.block_size;
    while (ok && walk.next(p, err, un, kt0, kt1)) {
      const int k0 = kt0 * kStepKeys, k1 = min(kt1 * kStepKeys, un.kvlen);
      const int* table = p.batch.tables + un.seq * p.batch.table_stride;
      int page = 0, row = 0;  // lane i: where copy i of the current 32 lies
      int i = 32;
      for (int key = k0; key < k1; key += L::kStageKeys) {
        const int st = c % L::kStages;
        const int boxes = (min(L::kStageKeys, k1 - key) + box_rows - 1) >> box_shift;
        ok = __all_sync(0xffffffffu,
                        mbar_wait(bar_empty(st), ((c / L::kStages) & 1u) ^ 1u, abort_flag, err, kErrWaitKvEmpty));
        if (!ok) break;
        if (elected) mbar_arrive_expect_tx(bar_full(st), boxes * (box_bytes + (kScaled ? 2 * box_rows : 0)));
        for (int b = 0; b < boxes; ++b, ++i) {
          if (i == 32) {
            i = 0;
            const int at = key + ((b + lane) << box_shift);
            if (at < k1) {
              page = table[at / bs];
              row = at % bs;
              if (page < 0 || page >= p.pool.blocks) {
                atomicCAS(err, 0, kErrBlockTable);
                page = 0;
              }
            }
          }
          const int pg = 2 * __shfl_sync(0xffffffffu, page, i), at = __shfl_sync(0xffffffffu, row, i);
          if (elected) {
            tma_load_5d(sbase + st * L::kStageBytes + b * box_bytes, &tm_kv, 0, at, 0, un.head, pg, bar_full(st));
            if (kScaled)
              tma_load_3d(sScale + st * L::kScaleStage + b * scale_slot, &tm_scale, at, un.head, pg, bar_full(st));
          }
        }
        ++c;
      }
    }
    if (!ok && elected)  // let the copies in flight land before the CTA ends
      for (uint32_t i = c > L::kStages ? c - L::kStages : 0; i < c; ++i)
        mbar_wait_teardown(bar_full(i % L::kStages), (i / L::kStages) & 1u);
    return;
  }

  // ------------------------------------------------------------ consumers --
  if (kFp8) setmaxnreg_inc<kRowsConsumerRegs>();
  constexpr int kConsumers = 32 * L::kWarps;
  constexpr int kWarpBoxes = L::kElt;        // 128-byte boxes of a warp's 128 columns
  const int gq = lane >> 2, i4 = lane & 3;   // MMA row (and column) group, position in it
  const int part = warp % L::kTeam;          // this warp's 128 columns
  bool ok = true;
  if (threadIdx.x == 0) clear_record(rec);
  // The number of the unit part if V had values taken for zeros (nonfinite8).
  volatile int* patch = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  for (int unit = 1; walk.next(p, err, un, kt0, kt1); ++unit) {
    if (threadIdx.x == 0) note_part(rec, un, kt0, kt1);
    const int k0 = kt0 * kStepKeys, k1 = min(kt1 * kStepKeys, un.kvlen);
    const bool two = un.rows > 16;  // two row tiles
    // Q into fragment order: a warp a row, eight elements a lane.
    for (int r = warp; r < (two ? 32 : 16); r += L::kWarps) {
      const int row = un.row0 + r;
      const bool live = r < un.rows, mine = lane < D / 8;
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (live && mine)
        x = *reinterpret_cast<const uint4*>(
            p.q + static_cast<long long>(un.head * p.group + row % p.group) * p.q_head +
            static_cast<long long>(un.q0 + row / p.group) * p.q_row + 8 * lane);
      float factor = p.scale_log2;
      if (kFp8) {
        float f[8];
        Vec8<__nv_bfloat16>{x}.get(f);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t a = __float_as_uint(f[i]) & 0x7FFFFFFFu;
          if (a < 0x7F800000u) m = max(m, a);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int e = m == 0 ? 0 : max(static_cast<int>(m >> 23) - 127 - 14, -112);
        const float down = exp2_of_int(-e);
        factor = p.scale_log2 * exp2_of_int(e);
        x = make_uint4(pack_f16x2(f[0] * down, f[1] * down), pack_f16x2(f[2] * down, f[3] * down),
                       pack_f16x2(f[4] * down, f[5] * down), pack_f16x2(f[6] * down, f[7] * down));
      }
      if (lane == 0) {
        row_factor[r] = factor;
        row_pos[r] = live ? un.kvlen - un.qlen + row / p.group : -1;
      }
      if (mine) {
        const int d = 8 * lane, box = d / kBoxElts, dd = d % kBoxElts;
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // elements dd + 2 j, + 1
          const int e = dd + 2 * j;
          const int step = box * kBoxSteps + (e % (kBoxElts / 4)) / 4;
          const int at = (r % 8) * 4 + e / (kBoxElts / 4);
          const int reg = ((e & 2) ? 2 : 0) + ((r & 8) ? 1 : 0);
          *reinterpret_cast<uint32_t*>(smem + L::kQOff + (r / 16) * (16 * D * 2) + (step * 32 + at) * 16 + reg * 4) = w[j];
        }
      }
    }
    named_bar_sync(1, kConsumers);
    const int teams = two ? L::kTeams / 2 : L::kTeams;  // of each row tile
    const int team = warp / L::kTeam;
    const int qt = team / teams, turn = team % teams;
    const uint32_t q_frag = sQ + qt * (16 * D * 2) + (part * kWarpBoxes * kBoxSteps * 32 + lane) * 16;
    const float f0 = row_factor[qt * 16 + gq], f1 = row_factor[qt * 16 + gq + 8];
    const int pos0 = row_pos[qt * 16 + gq], pos1 = row_pos[qt * 16 + gq + 8];
    // Keys that every live row of the tile sees: no comparison needed there.
    const int all_see = keys_all_see(un.kvlen, un.qlen, un.row0 + qt * 16, p.group);

    float o[16][4];
#pragma unroll
    for (int t = 0; t < 16; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float ref0 = -INFINITY, ref1 = -INFINITY;  // kScaled: l's reference

    uint32_t swap = 0;     // which of the two score exchange slots
    int next = 16 * turn;  // this team's next keys, from the stage's first
    for (int key0 = k0; key0 < k1; key0 += L::kStageKeys, ++c) {
      const int st = c % L::kStages;
      // (After a failed wait a warp goes on, over whatever the stages hold, so that its
      // team's barriers are met; nothing of it is merged.)
      if (!__all_sync(0xffffffffu, mbar_wait(bar_full(st), (c / L::kStages) & 1u, abort_flag, err, kErrWaitKvFull)))
        ok = false;
      const int here = min(L::kStageKeys, k1 - key0);
      for (; next < here; next += 16 * teams) {
        const int key = key0 + next;
        const int box = next >> box_shift, in_box = next & (box_rows - 1);
        const uint32_t col = box_rows * 128;  // a 128-byte column of K (or V) in its copy
        const uint32_t base = sbase + st * L::kStageBytes + box * box_bytes + in_box * 128 + part * kWarpBoxes * col;
        const uint32_t kV = L::kBoxes * col;
        // S = Q K^T of 16 keys: columns 2 i4, + 1 of two 8-key tiles, in two
        // chains of MMAs each.
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        float s2[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int b = 0; b < kWarpBoxes; ++b) {
          const uint32_t kr = base + b * col + gq * 128;
          const uint32_t ca = ((2 * i4) ^ gq) * 16, cb = ((2 * i4 + 1) ^ gq) * 16;
          const uint4 xa = lds128(kr + ca), ya = lds128(kr + 1024 + ca);
          const uint4 xb = lds128(kr + cb), yb = lds128(kr + 1024 + cb);
          const uint32_t x[8] = {xa.x, xa.y, xa.z, xa.w, xb.x, xb.y, xb.z, xb.w};
          const uint32_t y[8] = {ya.x, ya.y, ya.z, ya.w, yb.x, yb.y, yb.z, yb.w};
#pragma unroll
          for (int j = 0; j < kBoxSteps; ++j) {
            const uint4 a = lds128(q_frag + (b * kBoxSteps + j) * 512);
            float(&sa)[4] = (j & 1) ? s2[0] : s[0];
            float(&sb)[4] = (j & 1) ? s2[1] : s[1];
            if (kFp8) {
              uint32_t b0, b1;
              e4m3x4_to_f16x4(x[j], b0, b1);
              mma16816<true>(sa, a, b0, b1);
              e4m3x4_to_f16x4(y[j], b0, b1);
              mma16816<true>(sb, a, b0, b1);
            } else {
              mma16816<false>(sa, a, x[2 * j], x[2 * j + 1]);
              mma16816<false>(sb, a, y[2 * j], y[2 * j + 1]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] += s2[n][i];
        if (L::kTeam > 1) {  // the other warp's half of the terms
          float4* xch = reinterpret_cast<float4*>(smem + L::kBufOff) + ((swap * L::kWarps + warp) * 2) * 32 + lane;
          xch[0] = make_float4(s[0][0], s[0][1], s[0][2], s[0][3]);
          xch[32] = make_float4(s[1][0], s[1][1], s[1][2], s[1][3]);
          named_bar_sync(2 + team, 32 * L::kTeam);
          const float4* other =
              reinterpret_cast<const float4*>(smem + L::kBufOff) + ((swap * L::kWarps + (warp ^ 1)) * 2) * 32 + lane;
          const float4 u = other[0], v = other[32];
          s[0][0] += u.x, s[0][1] += u.y, s[0][2] += u.z, s[0][3] += u.w;
          s[1][0] += v.x, s[1][1] += v.y, s[1][2] += v.z, s[1][3] += v.w;
          swap ^= 1;
        }
        const int left = k1 - key;  // keys of this group that are there
        // The softmax and P V; `all`: every row sees all 16 keys, as all but the
        // last of a decode step's.
        auto finish = [&](auto all) {
          constexpr bool whole = decltype(all)::value;
          // Scores in log2 units, hidden keys at -inf (their scale bytes may be any);
          // the V exponents of this lane's four keys.
          float ev[4] = {0.f, 0.f, 0.f, 0.f};
          float mx0 = -INFINITY, mx1 = -INFINITY;
          const uint8_t* sc = smem + L::kScaleOff + st * L::kScaleStage + box * scale_slot + in_box + 2 * i4;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            uint32_t kb = 0;
            if (kScaled) {
              kb = *reinterpret_cast<const uint16_t*>(sc + 8 * n);
              const uint32_t vb = *reinterpret_cast<const uint16_t*>(sc + box_rows + 8 * n);
              ev[2 * n] = exponent_of_scale(vb & 0xFFu);
              ev[2 * n + 1] = exponent_of_scale(vb >> 8);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              s[n][j] *= f0;
              s[n][j + 2] *= f1;
              if (kScaled) {
                const float k2 = __uint_as_float((j ? kb >> 8 : kb & 0xFFu) << 23);
                s[n][j] *= k2;
                s[n][j + 2] *= k2;
              }
              if (!whole) {
                const int kk = 8 * n + 2 * i4 + j;
                if (kk >= left || key + kk > pos0) s[n][j] = -INFINITY;
                if (kk >= left || key + kk > pos1) s[n][j + 2] = -INFINITY;
              }
              mx0 = fmaxf(mx0, kScaled ? s[n][j] + ev[2 * n + j] : s[n][j]);
              mx1 = fmaxf(mx1, kScaled ? s[n][j + 2] + ev[2 * n + j] : s[n][j + 2]);
            }
          }
#pragma unroll
          for (int x = 1; x <= 2; x <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
          }
          auto of_row = [](float x) {  // the largest of a row's four lanes
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          };
          // kScaled: l's references up to the scores seen here, of the rows that ask for it.
          auto raise_refs = [&](bool row0, bool row1) {
            const float g0 = of_row(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])));
            const float g1 = of_row(fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])));
            if (row0 && g0 > ref0) l0 *= ex2_approx(ref0 - g0), ref0 = g0;
            if (row1 && g1 > ref1) l1 *= ex2_approx(ref1 - g1), ref1 = g1;
          };
          // The reference moves when the largest weight would pass 2^8 (and
          // from its start); O and l follow.
          const bool up0 = mx0 > m0 + kRescaleThreshold, up1 = mx1 > m1 + kRescaleThreshold;
          if (__any_sync(0xffffffffu, up0 || up1)) {
            float a0 = 1.f, a1 = 1.f;
            if (up0) a0 = ex2_approx(m0 - mx0), m0 = mx0;
            if (up1) a1 = ex2_approx(m1 - mx1), m1 = mx1;
            if (kScaled) {
              raise_refs(up0, up1);
            } else {
              l0 *= a0;
              l1 *= a1;
            }
#pragma unroll
            for (int t = 0; t < 16; ++t) {
              o[t][0] *= a0;
              o[t][1] *= a0;
              o[t][2] *= a1;
              o[t][3] *= a1;
            }
          }
          if (kScaled) {
            float sum0, sum1;
            auto weigh = [&]() {
              const float q0 = ref0 == -INFINITY ? 0.f : ref0, q1 = ref1 == -INFINITY ? 0.f : ref1;
              sum0 = (ex2_approx(s[0][0] - q0) + ex2_approx(s[0][1] - q0)) + (ex2_approx(s[1][0] - q0) + ex2_approx(s[1][1] - q0));
              sum1 = (ex2_approx(s[0][2] - q1) + ex2_approx(s[0][3] - q1)) + (ex2_approx(s[1][2] - q1) + ex2_approx(s[1][3] - q1));
            };
            weigh();
            if (__any_sync(0xffffffffu, fmaxf(sum0, sum1) > 65536.f)) {
              raise_refs(of_row(sum0) > 65536.f, of_row(sum1) > 65536.f);
              weigh();
            }
            l0 += sum0;
            l1 += sum1;
          }
          const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
          uint32_t pk[4];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float ea = kScaled ? ev[2 * n] : 0.f, eb = kScaled ? ev[2 * n + 1] : 0.f;
            const float pa = ex2_approx(kScaled ? s[n][0] + ea - r0 : s[n][0] - r0);
            const float pb = ex2_approx(kScaled ? s[n][1] + eb - r0 : s[n][1] - r0);
            const float pc = ex2_approx(kScaled ? s[n][2] + ea - r1 : s[n][2] - r1);
            const float pd = ex2_approx(kScaled ? s[n][3] + eb - r1 : s[n][3] - r1);
            if (!kScaled) {
              l0 += pa + pb;
              l1 += pc + pd;
            }
            pk[2 * n] = kFp8 ? pack_f16x2(pa, pb) : pack_bf16x2(pa, pb);
            pk[2 * n + 1] = kFp8 ? pack_f16x2(pc, pd) : pack_bf16x2(pc, pd);
          }
          const uint4 pa = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          // O += P V; rows of keys that are not there may hold anything: zeros.
          if (kFp8) {
            const uint32_t vr = base + kV + 2 * i4 * 128;
            const uint32_t ce = (gq ^ (2 * i4)) * 16, co = (gq ^ (2 * i4 + 1)) * 16;
            uint4 v0 = lds128(vr + ce), v1 = lds128(vr + 128 + co);
            uint4 v2 = lds128(vr + 1024 + ce), v3 = lds128(vr + 1024 + 128 + co);
            if (!whole && left < 16) {
              const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
              if (2 * i4 >= left) v0 = zero;
              if (2 * i4 + 1 >= left) v1 = zero;
              if (2 * i4 + 8 >= left) v2 = zero;
              if (2 * i4 + 9 >= left) v3 = zero;
            }
            if (!whole) {  // keys that some rows do not see: nothing that is not finite
              const int look = all_see - key - 2 * i4;
              bool found = false;
              if (look <= 0) found |= drop_nonfinite<true>(v0);
              if (look <= 1) found |= drop_nonfinite<true>(v1);
              if (look <= 8) found |= drop_nonfinite<true>(v2);
              if (look <= 9) found |= drop_nonfinite<true>(v3);
              if (found) *patch = unit;
            }
            const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
            const uint32_t w2[4] = {v2.x, v2.y, v2.z, v2.w}, w3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t a0, a1, b0, b1;
              e4m3x4_to_f16x4(__byte_perm(w0[j], w1[j], 0x5140), a0, a1);
              e4m3x4_to_f16x4(__byte_perm(w2[j], w3[j], 0x5140), b0, b1);
              mma16816<true>(o[4 * j], pa, a0, b0);
              mma16816<true>(o[4 * j + 1], pa, a1, b1);
              e4m3x4_to_f16x4(__byte_perm(w0[j], w1[j], 0x7362), a0, a1);
              e4m3x4_to_f16x4(__byte_perm(w2[j], w3[j], 0x7362), b0, b1);
              mma16816<true>(o[4 * j + 2], pa, a0, b0);
              mma16816<true>(o[4 * j + 3], pa, a1, b1);
            }
          } else {
            const uint32_t z0 = (whole || 2 * i4 < left ? 0xFFFFu : 0u) | (whole || 2 * i4 + 1 < left ? 0xFFFF0000u : 0u);
            const uint32_t z1 = (whole || 2 * i4 + 8 < left ? 0xFFFFu : 0u) | (whole || 2 * i4 + 9 < left ? 0xFFFF0000u : 0u);
            const int look = all_see - key - 2 * i4;
            const uint32_t look0 = (look <= 0 ? 0xFFFFu : 0u) | (look <= 1 ? 0xFFFF0000u : 0u);
            const uint32_t look1 = (look <= 8 ? 0xFFFFu : 0u) | (look <= 9 ? 0xFFFF0000u : 0u);
            const int vrow = lane & 15, vc = lane >> 4;
#pragma unroll
            for (int b = 0; b < kWarpBoxes; ++b) {
              const uint32_t vr = base + kV + b * col + vrow * 128;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t v[4];
                ldmatrix_x4_trans(vr + (((2 * j + vc) ^ (vrow & 7)) * 16), v);
                if (!whole) {  // keys that some rows do not see: nothing that is not finite
                  uint32_t found = 0;
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const uint32_t bad = nonfinite_mask<false>(v[i]) & ((i & 1) ? look1 : look0);
                    v[i] &= ~bad;
                    found |= bad & ((i & 1) ? z1 : z0);
                  }
                  if (found) *patch = unit;
                }
                mma16816<false>(o[b * 8 + 2 * j], pa, v[0] & z0, v[1] & z1);
                mma16816<false>(o[b * 8 + 2 * j + 1], pa, v[2] & z0, v[3] & z1);
              }
            }
          }
        };
        if (left >= 16 && key + 16 <= all_see) finish(std::true_type());
        else finish(std::false_type());
      }
      next -= L::kStageKeys;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_empty(st));
    }

    // ------------------------------------ merge the teams of each row tile --
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    if (i4 == 0 && part == 0) {  // a team's warps hold the same
      s_m[team * 16 + gq] = m0;
      s_m[team * 16 + gq + 8] = m1;
      s_l[team * 16 + gq] = l0;
      s_l[team * 16 + gq + 8] = l1;
      if (kScaled) {
        s_ref[team * 16 + gq] = ref0;
        s_ref[team * 16 + gq + 8] = ref1;
      }
    }
    if (!(ok = named_bar_and(1, kConsumers, ok && *abort_flag == 0))) break;
    float M0 = -INFINITY, M1 = -INFINITY;
    for (int w = qt * teams; w < (qt + 1) * teams; ++w) {
      M0 = fmaxf(M0, s_m[w * 16 + gq]);
      M1 = fmaxf(M1, s_m[w * 16 + gq + 8]);
    }
    const float a0 = ex2_approx(m0 - M0), a1 = ex2_approx(m1 - M1);
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      // A team that saw nothing of a row adds nothing to it.
      o[t][0] = m0 == -INFINITY ? 0.f : o[t][0] * a0;
      o[t][1] = m0 == -INFINITY ? 0.f : o[t][1] * a0;
      o[t][2] = m1 == -INFINITY ? 0.f : o[t][2] * a1;
      o[t][3] = m1 == -INFINITY ? 0.f : o[t][3] * a1;
    }
    // The last teams write their O to the tile's buffers, those before them add
    // theirs, round by round.
    const int bufs = two ? L::kBufs / 2 : L::kBufs;
    float* buf = reinterpret_cast<float*>(smem + L::kBufOff + (qt * bufs + turn % bufs) * L::kBufBytes) + part * 144;
    auto exchange = [&](bool add) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float* row = buf + (gq + 8 * r) * L::kRowFloats;
        if (kFp8) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // columns 32 i4 + 16 h + 4 j ..
              float4* at = reinterpret_cast<float4*>(row + 36 * i4 + 16 * h + 4 * j);
              float4 v = make_float4(o[4 * j][2 * r + h], o[4 * j + 1][2 * r + h], o[4 * j + 2][2 * r + h],
                                     o[4 * j + 3][2 * r + h]);
              if (add) {
                const float4 x = *at;
                v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
              }
              *at = v;
            }
        } else {
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            const int d = 8 * t + 2 * i4;
            float2* at = reinterpret_cast<float2*>(row + d + 4 * (d / 32));
            float2 v = make_float2(o[t][2 * r], o[t][2 * r + 1]);
            if (add) {
              const float2 x = *at;
              v = make_float2(v.x + x.x, v.y + x.y);
            }
            *at = v;
          }
        }
      }
    };
    // Each row's sum over its teams (the rounds' barriers pass it on).
    const int slot = part_slot(un, kt0, kt1, blockIdx.x);
    if (threadIdx.x < (two ? 32 : 16)) {
      const int r = threadIdx.x, t0 = r / 16 * teams;
      float M = -INFINITY, ref = -INFINITY, lsum = 0.f;
      for (int w = t0; w < t0 + teams; ++w) {
        M = fmaxf(M, s_m[w * 16 + r % 16]);
        ref = fmaxf(ref, s_ref[w * 16 + r % 16]);
      }
      for (int w = t0; w < t0 + teams; ++w) {
        const float rw = s_ref[w * 16 + r % 16];
        // Without a maximum the sum is 0, or NaN where every score was NaN.
        lsum += rw == -INFINITY ? s_l[w * 16 + r % 16] : s_l[w * 16 + r % 16] * ex2_approx(rw - ref);
      }
      s_inv[r] = lsum == 0.f ? 0.f : kScaled ? output_factor(M, ref, lsum) : 1.f / lsum;  // no key seen: zeros
      if (slot >= 0 && r < un.rows)
        p.work.small_lse[static_cast<long long>(slot) * kSmallRows + r] = lsum == 0.f ? -INFINITY : ref + __log2f(lsum);
    }
    for (int round = (teams - 1) / bufs; round >= 0; --round) {
      if (turn / bufs == round) exchange(turn + bufs < teams);
      named_bar_sync(1, kConsumers);
    }
    // Every thread eight elements of a row: sum the buffers, divide, write.
    for (int x = threadIdx.x; x < un.rows * (D / 8); x += kConsumers) {
      const int r = x / (D / 8), d = (x % (D / 8)) * 8;
      const int t = r / 16;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const float* src = reinterpret_cast<const float*>(smem + L::kBufOff) + (r % 16) * L::kRowFloats + d + 4 * (d / 32);
      for (int k = 0; k < bufs; ++k) {
        const float4* at = reinterpret_cast<const float4*>(src + (t * bufs + k) * (L::kBufBytes / 4));
        const float4 u = at[0], v = at[1];
        f[0] += u.x, f[1] += u.y, f[2] += u.z, f[3] += u.w, f[4] += v.x, f[5] += v.y, f[6] += v.z, f[7] += v.w;
      }
      const float inv = s_inv[r];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= inv;
      if (*patch == unit) {  // rare: see nonfinite8
        const int first = keys_all_see(un.kvlen, un.qlen, un.row0 + 16 * t, p.group);
        uint32_t bad = 0;
        for (int key = max(first, k0); key < min(un.kvlen - un.qlen + (un.row0 + r) / p.group + 1, k1); ++key)
          bad |= nonfinite8<D>(p, un.seq, un.head, key, d);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if ((bad >> i) & 1u) f[i] = NAN;
      }
      if (slot < 0) {
        const int row = un.row0 + r;
        Vec8<__nv_bfloat16>::store(p.out + static_cast<long long>(un.head * p.group + row % p.group) * p.out_head +
                                       static_cast<long long>(un.q0 + row / p.group) * p.out_row + d,
                                   f);
      } else {
        const long long at = static_cast<long long>(slot) * kSmallRows + r;
        Vec8<float>::store(p.work.small_o + at * D + d, f);
      }
    }
  }
  if (threadIdx.x == 0) {
    // After a failure nothing of the range is merged: its partials may be unwritten.
    rec.failed = !ok || *abort_flag;
    rec.err = *static_cast<volatile int*>(err);
  }
}

}  // namespace pcp
