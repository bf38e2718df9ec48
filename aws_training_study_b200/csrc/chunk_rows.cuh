// Attention of a few query rows (a KV head's group of queries of one token, or
// of a few drafted ones: at most kSmallRows) over a long paged cache.
//
// Bound by reading the cache: 4 rows' flops a byte are far below what the
// tensor cores need, so the cache must stream at HBM's rate and everything else
// hide behind it.  A 128-row tcgen05 tile would spend its time on empty rows
// (the tile kernel reads 2.4 TB/s on such a unit); here a warp's mma.sync tile is
// 16 rows, which one token's group of heads fills, and warps split the KEYS:
//   * A producer warp streams stages of kStageKeys keys (K and V of one head, 8
//     KB of e4m3 or 16 KB of bf16) through a 128 KB shared-memory ring with TMA
//     (16-row boxes, so pages of any multiple of 16 tokens; 128-byte swizzle).
//   * Stage c goes to warp c % 8, which scores its keys against all rows and
//     adds P V into its own 16 x D accumulators, with its own running maximum:
//     nothing is exchanged between warps until the unit ends.  A unit of 17 to
//     32 rows uses warps w and w + 4 as its two row tiles on the same stage.
//   * The warps' (m, l, O) are merged through shared memory when the unit's part
//     ends, into bf16 rows or an fp32 partial.
//
// e4m3 codes become f16 in registers (exact) on their way into the MMA.  No
// ldmatrix: the order of an MMA's k index is free as long as both operands
// agree, so a lane takes 16 consecutive bytes of a K row as four k steps (Q's
// fragments are laid out to match), and of a V row as 16 output columns (pairs
// of keys are zipped with byte permutes).  All accesses hit distinct banks.
// Scales: K's 2^e multiplies its key's score, V's 2^e its key's weight p.  The
// softmax's reference m is kept above (score + V exponent) instead of the score
// alone, so that p 2^e stays in f16's range whatever the exponents; m cancels
// between O and l as ever.  f16's 11 bits for p 2^e are three more than bf16's.
// Q is brought to f16 by a power of two of its row.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "chunk_plan.cuh"

namespace pcp {

constexpr int kRowsWarps = 8;
constexpr int kRowsThreads = 32 * kRowsWarps + 32;  // + the producer warp

template <int D, bool kFp8>
struct RowsSmem {
  static constexpr int kElt = kFp8 ? 1 : 2;
  static constexpr int kStageKeys = 4096 / D;             // 16 or 32
  static constexpr int kGroups = kStageKeys / 16;          // 16-row boxes down a stage
  static constexpr int kBoxes = D * kElt / 128;            // 128-byte boxes across a row
  static constexpr int kBoxPair = 2 * 16 * 128;            // a box's K rows, then its V rows
  static constexpr int kStageBytes = kGroups * kBoxes * kBoxPair;
  static constexpr int kStages = 131072 / kStageBytes;
  static constexpr int kScaleBytes = kFp8 ? kStageKeys * 2 : 0;  // [group][K, V][16]
  // O exchange: 16 rows of D floats, 4 floats of padding every 32, rows 16
  // banks apart: a lane's 16-byte stores fall on distinct banks.
  static constexpr int kRowFloats = D + D / 8 + (D == 256 ? 16 : 0);
  static constexpr int kBufBytes = 16 * kRowFloats * 4;
  static constexpr int kBufs = 4;
  static constexpr int kQOff = kStages * kStageBytes;
  static constexpr int kQBytes = 2 * 16 * D * 2;  // two row tiles in MMA fragment order
  static constexpr int kScaleOff = kQOff + kQBytes;
  static constexpr int kBufOff = kScaleOff + kStages * kScaleBytes;
  static constexpr int kRowOff = kBufOff + kBufs * kBufBytes;       // float score factor[32], int position[32]
  static constexpr int kMlOff = kRowOff + 2 * kSmallRows * 4;       // float m[8][16], l[8][16]
  static constexpr int kBarOff = kMlOff + 2 * kRowsWarps * 16 * 4;  // full, empty
  static constexpr int kMiscOff = kBarOff + 2 * kStages * 8;
  static constexpr int kBytes = kMiscOff + 16;
  static_assert(kBytes <= 232448, "exceeds the 227 KB of shared memory per CTA");
  static_assert(kBufOff % 16 == 0 && kBarOff % 8 == 0 && kScaleOff % 16 == 0, "alignment");
};

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

// Untiled copy of `bytes` (a multiple of 16) from global memory into THIS
// CTA's shared memory, completion on `bar`.  No multicast.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, uint32_t n) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}

template <int D, bool kFp8>
__global__ void __launch_bounds__(kRowsThreads, 1)
    chunk_rows_kernel(const __grid_constant__ CUtensorMap tm_kv, const ChunkParams p) {
  using L = RowsSmem<D, kFp8>;
  constexpr int NST = L::kStages;
  constexpr int kBoxElts = 128 / L::kElt;
  constexpr int kBoxSteps = kBoxElts / 16;  // MMA k steps of a box: 8 or 4
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  if (sbase & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, kErrSmemAlign);
    return;
  }
  const uint32_t sQ = sbase + L::kQOff;
  const uint32_t sScale = sbase + L::kScaleOff;
  float* row_factor = reinterpret_cast<float*>(smem + L::kRowOff);
  int* row_pos = reinterpret_cast<int*>(smem + L::kRowOff) + kSmallRows;
  float* s_m = reinterpret_cast<float*>(smem + L::kMlOff);
  float* s_l = s_m + kRowsWarps * 16;
  auto bar_full = [&](int s) { return sbase + L::kBarOff + 8u * s; };
  auto bar_empty = [&](int s) { return sbase + L::kBarOff + 8u * (NST + s); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 2);  // both row tiles' warps, or one warp twice
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  ChunkWalk walk;
  walk.init(p.work.small, p.work.small_start, p.work.plan->small_units, p.work.plan->small_steps, p.small_ctas,
            blockIdx.x);
  ChunkUnit un;
  int kt0, kt1, slot;
  uint32_t c = 0;  // stages of this CTA so far

  if (warp == kRowsWarps) {
    // -------------------------------------------------------- producer --
    bool ok = true;
    while (ok && walk.next(un, kt0, kt1, slot)) {
      const int k0 = kt0 * kStepKeys, k1 = min(kt1 * kStepKeys, un.kvlen);
      const int* table = p.batch.tables + un.seq * p.batch.table_stride;
      int page = 0;  // lane i: the page of 16-key group i of the current 32
      for (int key = k0; key < k1; key += L::kStageKeys) {
        const int g0 = (key - k0) / 16;
        if (g0 % 32 == 0) {
          const int at = key + 16 * lane;
          if (at < k1) {
            page = table[at / p.pool.block_size];
            if (page < 0 || page >= p.pool.blocks) {
              atomicCAS(p.err, 0, kErrBlockTable);
              page = 0;
            }
          }
        }
        const int st = c % NST;
        ok = __all_sync(0xffffffffu,
                        mbar_wait(bar_empty(st), ((c / NST) & 1u) ^ 1u, abort_flag, p.err, kErrWaitKvEmpty));
        if (!ok) break;
        const int groups = min(L::kGroups, (k1 - key + 15) / 16);
        const bool scaled = kFp8 && p.pool.scales;
        if (lane == 0)
          mbar_arrive_expect_tx(bar_full(st), groups * (L::kBoxes * L::kBoxPair + (scaled ? 32 : 0)));
        __syncwarp();
        // Lane (group, box) loads a box of K and V; the lanes behind them the scales.
        const int g = lane / L::kBoxes;
        const int pg = __shfl_sync(0xffffffffu, page, (g0 + min(g, L::kGroups - 1)) % 32);
        if (g < groups)
          tma_load_5d(sbase + st * L::kStageBytes + lane * L::kBoxPair, &tm_kv, (lane % L::kBoxes) * kBoxElts,
                      (key + 16 * g) % p.pool.block_size, un.head, 0, pg, bar_full(st));
        if (kFp8) {
          const int j = lane - 16;  // group, K or V
          const int ps = __shfl_sync(0xffffffffu, page, (g0 + min(max(j, 0) / 2, L::kGroups - 1)) % 32);
          if (scaled && j >= 0 && j < 2 * groups) {
            const long long row = (static_cast<long long>(ps) * 2 + (j & 1)) * p.pool.heads + un.head;
            bulk_load(sScale + st * L::kScaleBytes + j * 16,
                      p.pool.scales + row * p.pool.block_size + (key + 16 * (j / 2)) % p.pool.block_size, 16,
                      bar_full(st));
          }
        }
        ++c;
      }
    }
    if (!ok)  // let the copies in flight land before the CTA ends
      for (uint32_t i = c > NST ? c - NST : 0; i < c; ++i) mbar_wait_teardown(bar_full(i % NST), (i / NST) & 1u);
    return;
  }

  // ------------------------------------------------------------ consumers --
  const int gq = lane >> 2, i4 = lane & 3;  // MMA row (and column) group, position in it
  bool ok = true;
  while (walk.next(un, kt0, kt1, slot)) {
    const int k0 = kt0 * kStepKeys, k1 = min(kt1 * kStepKeys, un.kvlen);
    const int two = un.rows > 16;  // two row tiles
    // Q into fragment order: a warp a row, eight elements a lane.
    for (int r = warp; r < (two ? 32 : 16); r += kRowsWarps) {
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
    named_bar_sync(1, 32 * kRowsWarps);
    const int tile = two ? warp >> 2 : 0;
    const uint32_t q_frag = sQ + tile * (16 * D * 2) + lane * 16;
    const float f0 = row_factor[tile * 16 + gq], f1 = row_factor[tile * 16 + gq + 8];
    const int pos0 = row_pos[tile * 16 + gq], pos1 = row_pos[tile * 16 + gq + 8];
    const bool scaled = kFp8 && p.pool.scales;

    float o[D / 8][4];
#pragma unroll
    for (int t = 0; t < D / 8; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    const uint32_t c0 = c;
    c += (max(k1 - k0, 0) + L::kStageKeys - 1) / L::kStageKeys;
    const uint32_t step = two ? 4 : 8, first = two ? (warp & 3) : warp;
    for (uint32_t cc = c0 + ((first - c0) & (step - 1)); ok && cc < c; cc += step) {
      const int st = cc % NST;
      ok = __all_sync(0xffffffffu, mbar_wait(bar_full(st), (cc / NST) & 1u, abort_flag, p.err, kErrWaitKvFull));
      if (!ok) break;
      const int key0 = k0 + static_cast<int>(cc - c0) * L::kStageKeys;
#pragma unroll 1
      for (int gr = 0; gr < L::kGroups; ++gr) {
        const int key = key0 + 16 * gr;
        if (key >= k1) break;
        const uint32_t base = sbase + st * L::kStageBytes + gr * (L::kBoxes * L::kBoxPair);
        // S = Q K^T of 16 keys: columns 2 i4, + 1 of two 8-key tiles.
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int b = 0; b < L::kBoxes; ++b) {
          const uint32_t kr = base + b * L::kBoxPair + gq * 128;
          const uint32_t ca = ((2 * i4) ^ gq) * 16, cb = ((2 * i4 + 1) ^ gq) * 16;
          const uint4 xa = lds128(kr + ca), xb = lds128(kr + cb);
          const uint4 ya = lds128(kr + 1024 + ca), yb = lds128(kr + 1024 + cb);
          const uint32_t x[8] = {xa.x, xa.y, xa.z, xa.w, xb.x, xb.y, xb.z, xb.w};
          const uint32_t y[8] = {ya.x, ya.y, ya.z, ya.w, yb.x, yb.y, yb.z, yb.w};
#pragma unroll
          for (int j = 0; j < kBoxSteps; ++j) {
            const uint4 a = lds128(q_frag + (b * kBoxSteps + j) * 512);
            if (kFp8) {
              uint32_t b0, b1;
              e4m3x4_to_f16x4(x[j], b0, b1);
              mma16816<true>(s[0], a, b0, b1);
              e4m3x4_to_f16x4(y[j], b0, b1);
              mma16816<true>(s[1], a, b0, b1);
            } else {
              mma16816<false>(s[0], a, x[2 * j], x[2 * j + 1]);
              mma16816<false>(s[1], a, y[2 * j], y[2 * j + 1]);
            }
          }
        }
        // Scores in log2 units, hidden keys at -inf.
        float vs[4] = {1.f, 1.f, 1.f, 1.f};  // V scales of this lane's four keys
        int vb[4] = {127, 127, 127, 127};    // their exponents, biased
        if (scaled) {
          const uint8_t* sc = smem + L::kScaleOff + st * L::kScaleBytes + gr * 32 + 2 * i4;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint32_t kb = *reinterpret_cast<const uint16_t*>(sc + 8 * n);
            const uint32_t vv = *reinterpret_cast<const uint16_t*>(sc + 16 + 8 * n);
            const float ka = __uint_as_float((kb & 0xFFu) << 23), kc = __uint_as_float((kb >> 8) << 23);
            s[n][0] *= ka;
            s[n][1] *= kc;
            s[n][2] *= ka;
            s[n][3] *= kc;
            vb[2 * n] = vv & 0xFF;
            vb[2 * n + 1] = vv >> 8;
          }
        }
        const int left = k1 - key;  // keys of this group that are there
        float mx0 = -INFINITY, mx1 = -INFINITY;
        int ev = 0;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int kk = 8 * n + 2 * i4 + j;
            s[n][j] = kk < left && key + kk <= pos0 ? s[n][j] * f0 : -INFINITY;
            s[n][j + 2] = kk < left && key + kk <= pos1 ? s[n][j + 2] * f1 : -INFINITY;
            mx0 = fmaxf(mx0, s[n][j]);
            mx1 = fmaxf(mx1, s[n][j + 2]);
            if (scaled) {
              vs[2 * n + j] = kk < left ? __uint_as_float(static_cast<uint32_t>(vb[2 * n + j]) << 23) : 0.f;
              ev = kk < left ? max(ev, vb[2 * n + j]) : ev;
            }
          }
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
          if (scaled) ev = max(ev, __shfl_xor_sync(0xffffffffu, ev, x));
        }
        if (scaled) {
          mx0 += static_cast<float>(ev - 127);
          mx1 += static_cast<float>(ev - 127);
        }
        // The reference moves when the largest weight would pass 2^8 (and
        // from its start); O and l follow.
        const bool up0 = mx0 > m0 + kRescaleThreshold, up1 = mx1 > m1 + kRescaleThreshold;
        if (__any_sync(0xffffffffu, up0 || up1)) {
          float a0 = 1.f, a1 = 1.f;
          if (up0) a0 = ex2_approx(m0 - mx0), m0 = mx0;
          if (up1) a1 = ex2_approx(m1 - mx1), m1 = mx1;
          l0 *= a0;
          l1 *= a1;
#pragma unroll
          for (int t = 0; t < D / 8; ++t) {
            o[t][0] *= a0;
            o[t][1] *= a0;
            o[t][2] *= a1;
            o[t][3] *= a1;
          }
        }
        const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
        uint32_t pk[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          float pa = ex2_approx(s[n][0] - r0), pb = ex2_approx(s[n][1] - r0);
          float pc = ex2_approx(s[n][2] - r1), pd = ex2_approx(s[n][3] - r1);
          l0 += pa + pb;
          l1 += pc + pd;
          if (scaled) {
            pa *= vs[2 * n];
            pb *= vs[2 * n + 1];
            pc *= vs[2 * n];
            pd *= vs[2 * n + 1];
          }
          pk[2 * n] = kFp8 ? pack_f16x2(pa, pb) : pack_bf16x2(pa, pb);
          pk[2 * n + 1] = kFp8 ? pack_f16x2(pc, pd) : pack_bf16x2(pc, pd);
        }
        const uint4 pa = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        // O += P V; rows of keys that are not there may hold anything: zeros.
        if (kFp8) {
          const uint32_t z0 = 2 * i4 < left ? ~0u : 0u, z1 = 2 * i4 + 1 < left ? ~0u : 0u;
          const uint32_t z2 = 2 * i4 + 8 < left ? ~0u : 0u, z3 = 2 * i4 + 9 < left ? ~0u : 0u;
#pragma unroll
          for (int b = 0; b < L::kBoxes; ++b) {
            const uint32_t vr = base + b * L::kBoxPair + 2048 + 2 * i4 * 128;
            const uint32_t ce = (gq ^ (2 * i4)) * 16, co = (gq ^ (2 * i4 + 1)) * 16;
            const uint4 v0 = lds128(vr + ce), v1 = lds128(vr + 128 + co);
            const uint4 v2 = lds128(vr + 1024 + ce), v3 = lds128(vr + 1024 + 128 + co);
            const uint32_t w0[4] = {v0.x & z0, v0.y & z0, v0.z & z0, v0.w & z0};
            const uint32_t w1[4] = {v1.x & z1, v1.y & z1, v1.z & z1, v1.w & z1};
            const uint32_t w2[4] = {v2.x & z2, v2.y & z2, v2.z & z2, v2.w & z2};
            const uint32_t w3[4] = {v3.x & z3, v3.y & z3, v3.z & z3, v3.w & z3};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t a0, a1, b0, b1;
              e4m3x4_to_f16x4(__byte_perm(w0[j], w1[j], 0x5140), a0, a1);
              e4m3x4_to_f16x4(__byte_perm(w2[j], w3[j], 0x5140), b0, b1);
              mma16816<true>(o[b * 16 + 4 * j], pa, a0, b0);
              mma16816<true>(o[b * 16 + 4 * j + 1], pa, a1, b1);
              e4m3x4_to_f16x4(__byte_perm(w0[j], w1[j], 0x7362), a0, a1);
              e4m3x4_to_f16x4(__byte_perm(w2[j], w3[j], 0x7362), b0, b1);
              mma16816<true>(o[b * 16 + 4 * j + 2], pa, a0, b0);
              mma16816<true>(o[b * 16 + 4 * j + 3], pa, a1, b1);
            }
          }
        } else {
          const uint32_t z0 = (2 * i4 < left ? 0xFFFFu : 0u) | (2 * i4 + 1 < left ? 0xFFFF0000u : 0u);
          const uint32_t z1 = (2 * i4 + 8 < left ? 0xFFFFu : 0u) | (2 * i4 + 9 < left ? 0xFFFF0000u : 0u);
          const int vrow = lane & 15, vc = lane >> 4;
#pragma unroll
          for (int b = 0; b < L::kBoxes; ++b) {
            const uint32_t vr = base + b * L::kBoxPair + 2048 + vrow * 128;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t v[4];
              ldmatrix_x4_trans(vr + (((2 * j + vc) ^ (vrow & 7)) * 16), v);
              mma16816<false>(o[b * 8 + 2 * j], pa, v[0] & z0, v[1] & z1);
              mma16816<false>(o[b * 8 + 2 * j + 1], pa, v[2] & z0, v[3] & z1);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_n(bar_empty(st), two ? 1 : 2);
    }

    // ------------------------------------ merge the warps of each row tile --
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    if (i4 == 0) {
      s_m[warp * 16 + gq] = m0;
      s_m[warp * 16 + gq + 8] = m1;
      s_l[warp * 16 + gq] = l0;
      s_l[warp * 16 + gq + 8] = l1;
    }
    if (!named_bar_and(1, 32 * kRowsWarps, ok && *abort_flag == 0)) return;
    const int w0 = two ? tile * 4 : 0, wn = two ? 4 : 8;
    float M0 = -INFINITY, M1 = -INFINITY;
    for (int w = w0; w < w0 + wn; ++w) {
      M0 = fmaxf(M0, s_m[w * 16 + gq]);
      M1 = fmaxf(M1, s_m[w * 16 + gq + 8]);
    }
    const float a0 = m0 == -INFINITY ? 0.f : ex2_approx(m0 - M0);
    const float a1 = m1 == -INFINITY ? 0.f : ex2_approx(m1 - M1);
#pragma unroll
    for (int t = 0; t < D / 8; ++t) {
      // A warp that saw nothing of a row adds nothing to it.
      o[t][0] = m0 == -INFINITY ? 0.f : o[t][0] * a0;
      o[t][1] = m0 == -INFINITY ? 0.f : o[t][1] * a0;
      o[t][2] = m1 == -INFINITY ? 0.f : o[t][2] * a1;
      o[t][3] = m1 == -INFINITY ? 0.f : o[t][3] * a1;
    }
    const int half = wn / 2, wi = warp - w0;
    float* buf = reinterpret_cast<float*>(smem + L::kBufOff + ((two ? tile * 2 : 0) + wi % half) * L::kBufBytes);
    // This lane's elements of a row, four (e4m3) or two (bf16) at a time.
    auto exchange = [&](bool add) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float* row = buf + (gq + 8 * r) * L::kRowFloats;
        if (kFp8) {
#pragma unroll
          for (int b = 0; b < L::kBoxes; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int d = b * 128 + 32 * i4 + 16 * h + 4 * j;
                float4* at = reinterpret_cast<float4*>(row + d + 4 * (d / 32));
                float4 v = make_float4(o[b * 16 + 4 * j][2 * r + h], o[b * 16 + 4 * j + 1][2 * r + h],
                                       o[b * 16 + 4 * j + 2][2 * r + h], o[b * 16 + 4 * j + 3][2 * r + h]);
                if (add) {
                  const float4 x = *at;
                  v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
                }
                *at = v;
              }
        } else {
#pragma unroll
          for (int t = 0; t < D / 8; ++t) {
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
    if (wi >= half) exchange(false);
    named_bar_sync(1, 32 * kRowsWarps);
    if (wi < half) exchange(true);
    named_bar_sync(1, 32 * kRowsWarps);
    // Every thread eight elements of a row: sum the buffers, divide, write.
    for (int x = threadIdx.x; x < un.rows * (D / 8); x += 32 * kRowsWarps) {
      const int r = x / (D / 8), d = (x % (D / 8)) * 8;
      const int t = r / 16, tw0 = two ? t * 4 : 0;
      float M = -INFINITY, lsum = 0.f;
      for (int w = tw0; w < tw0 + wn; ++w) M = fmaxf(M, s_m[w * 16 + r % 16]);
      for (int w = tw0; w < tw0 + wn; ++w) {
        const float mw = s_m[w * 16 + r % 16];
        // Without a maximum the sum is 0, or NaN where every score was NaN.
        lsum += mw == -INFINITY ? s_l[w * 16 + r % 16] : s_l[w * 16 + r % 16] * ex2_approx(mw - M);
      }
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const float* src = reinterpret_cast<const float*>(smem + L::kBufOff) + (r % 16) * L::kRowFloats + d + 4 * (d / 32);
      for (int k = 0; k < half; ++k) {
        const float4* at = reinterpret_cast<const float4*>(src + ((two ? t * 2 : 0) + k) * (L::kBufBytes / 4));
        const float4 u = at[0], v = at[1];
        f[0] += u.x, f[1] += u.y, f[2] += u.z, f[3] += u.w, f[4] += v.x, f[5] += v.y, f[6] += v.z, f[7] += v.w;
      }
      const float inv = lsum == 0.f ? 0.f : 1.f / lsum;  // no key seen: zeros
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= inv;
      if (slot < 0) {
        const int row = un.row0 + r;
        Vec8<__nv_bfloat16>::store(p.out + static_cast<long long>(un.head * p.group + row % p.group) * p.out_head +
                                       static_cast<long long>(un.q0 + row / p.group) * p.out_row + d,
                                   f);
      } else {
        const long long at = static_cast<long long>(slot) * kSmallRows + r;
        Vec8<float>::store(p.work.small_o + at * D + d, f);
        if (d == 0) p.work.small_lse[at] = lsum == 0.f ? -INFINITY : M + __log2f(lsum);
      }
    }
  }
}

}  // namespace pcp
