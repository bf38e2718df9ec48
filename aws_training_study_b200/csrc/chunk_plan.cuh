// Attention of each sequence's new tokens over its paged cache: the work
// units, their plan, and the merge of split units (include/pcp_serve.h,
// pcp_chunk_attention).
//
// With G query heads a KV head, the rows of (sequence, KV head) are its tokens'
// G queries each, token by token: row i is query head i % G of token i / G, so
// that neighbouring rows see nearly the same keys.  A unit is a run of them:
//   small: all rows of a (sequence, KV head) that has at most kSmallRows of them
//          (single tokens, drafts): bound by reading the cache, chunk_rows.cuh;
//   tile:  kPairRows rows of a longer chunk: bound by the tensor cores,
//          chunk_tiles.cuh.
// A unit's steps are the 128-key tiles that its last row sees (at least one, so
// that rows without keys are written too).  Each kernel cuts the list of its
// units' steps into equal contiguous ranges, one per CTA (or CTA pair): every
// one gets the same work whatever the lengths.  Every CTA finds its range by
// itself, summing the steps of all sequences in its prologue (a first kernel
// that listed the units took 16 to 26 us; the sums of a batch take about 2).  A
// unit that a range boundary cuts leaves fp32 partials, which
// chunk_combine_kernel merges; a range leaves a record of what it cut.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "attn_common.cuh"
#include "ptx.cuh"
#include "serve_ops.cuh"

namespace pcp {

enum : int { kCacheBf16 = 0, kCacheE4m3 = 1, kCacheScaled = 2 };

constexpr int kSmallRows = 32;
constexpr int kUnitRows = 256;  // rows of a tile unit: a CTA pair's
constexpr int kStepKeys = 128;

struct ChunkUnit {
  int seq, head;
  int row0, rows;  // first row within the (sequence, head), rows of the unit
  int q0, qlen;    // first packed row (token) and tokens of the sequence
  int kvlen;       // its tokens, the new ones included
  int steps;
};

// What a range cut: the unit it starts in the middle of (slot 2 g), and the one
// it leaves unfinished (slot 2 g + 1).
struct ChunkRecord {
  ChunkUnit last;   // the unfinished unit, when `last_cut`
  int last_cut;
  int first_state;  // 0: no partial, 1: does not end its unit, 2: ends it
  int err;          // the CTA's device error
  int failed;       // a wait of the CTA ran out: what it left may be unwritten
  int patch;        // tile units: V had values that were taken for zeros (nonfinite8)
};

struct ChunkWork {
  ChunkRecord* small_rec;  // [small CTAs]
  ChunkRecord* tile_rec;   // [2 pairs] (err, failed and patch of each CTA; the rest by pair)
  float* small_o;          // [2 small CTAs][kSmallRows][D] partials, normalised
  float* small_lse;        // [2 small CTAs][kSmallRows], log2
  float* tile_o;           // [2 pairs][kUnitRows][D]
  float* tile_lse;
};

struct ChunkParams {
  BatchView batch;
  PoolView pool;
  ChunkWork work;
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  long long q_head, q_row, out_head, out_row;
  int group;       // query heads per KV head
  long long capacity;  // tokens a sequence's table holds
  int max_chunk;
  float scale_log2;
  float v_factor;  // what V of a bf16 cache is to be multiplied with (kCopyShift)
  int small_ctas, tile_pairs;  // grids of the two kernels (0 pairs: not launched)
  int small_y, tile_y;         // blocks that merge a unit of either kind
  int* status;
};

__device__ __forceinline__ float exp2_of_int(int e) {  // 2^e, 0 below the normal range
  return __uint_as_float(static_cast<uint32_t>(min(max(e + 127, 0), 254)) << 23);
}

// A scale byte's exponent, b - 127: b as the low bits of 1.5 * 2^23.
__device__ __forceinline__ float exponent_of_scale(uint32_t b) { return __uint_as_float(0x4B400000u | b) - 12583039.f; }

// What O, weights of 2^(s + e - m), is to be multiplied with when the sum of the
// weights alone, 2^(s - ref), is l: 2^(m - ref) / l.  In two halves: it is in fp32's
// range, 2^(m - ref) need not be.
__device__ __forceinline__ float output_factor(float m, float ref, float l) {
  const float h = ex2_approx(0.5f * (m - ref));
  return h / l * h;
}

// 5-D tiled TMA load into THIS CTA's shared memory whose bytes count on
// `cluster_bar`, an mbarrier of either CTA of the pair.  Local-GPU memory; no
// multicast.
__device__ __forceinline__ void tma_load_5d_pair(uint32_t dst, const void* tmap, int32_t c0, int32_t c1, int32_t c2,
                                                 int32_t c3, int32_t c4, uint32_t cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(cluster_bar)
      : "memory");
}

// One lane of the (converged) warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// CTAs (or pairs) that a list of `steps` is cut for: at least one step each (at
// least 2 or 4 took the same times, 16 to 256 tokens over 500 to 32768).
__device__ __forceinline__ long long chunk_ranges(long long steps, int grid) {
  return min(max(steps, 1LL), static_cast<long long>(grid));
}

// Steps of rows [row0, row0 + rows) of a sequence: tiles up to the last row's
// position.
__device__ __forceinline__ int unit_steps(int kvlen, int qlen, int last_row, int group) {
  const int visible = kvlen - qlen + last_row / group + 1;
  return max(1, (visible + kStepKeys - 1) / kStepKeys);
}

// Keys that every row from `row0` on sees (not positive: some row sees none).
__device__ __forceinline__ int keys_all_see(int kvlen, int qlen, int row0, int group) {
  return kvlen - qlen + row0 / group + 1;
}

// The elements of a 32-bit word of two bf16 or four e4m3 codes that are not finite.
template <bool kFp8>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w) {
  return kFp8 ? __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu) : __vcmpeq2(w & 0x7F807F80u, 0x7F807F80u);
}

// Zeros in place of what is not finite; true if there was any.
template <bool kFp8>
__device__ __forceinline__ bool drop_nonfinite(uint4& x) {
  const uint4 m = make_uint4(nonfinite_mask<kFp8>(x.x), nonfinite_mask<kFp8>(x.y), nonfinite_mask<kFp8>(x.z),
                             nonfinite_mask<kFp8>(x.w));
  x = make_uint4(x.x & ~m.x, x.y & ~m.y, x.z & ~m.z, x.w & ~m.w);
  return (m.x | m.y | m.z | m.w) != 0;
}

// Non-finite values of V at a key that some rows of a unit see and others do
// not: 0 * NaN would reach the others, so the kernels take zeros in their place,
// note that they did, and the output is patched afterwards.  Of the elements d ..
// d + 7 of V at `key`, those that are not finite (a bit each).
template <int D>
__device__ __forceinline__ uint32_t nonfinite8(const ChunkParams& p, int seq, int head, int key, int d) {
  const int bs = p.pool.block_size, lb = key / bs;
  if (lb >= p.batch.table_width) return 0;
  const int pg = p.batch.tables ? p.batch.tables[seq * p.batch.table_stride + lb] : seq;
  if (pg < 0 || pg >= p.pool.blocks) return 0;
  const long long at = (((pg * 2LL + 1) * p.pool.heads + head) * bs + key % bs) * D + d;
  uint32_t bad = 0;
  if (p.pool.bf16) {
    const uint4 x = *reinterpret_cast<const uint4*>(p.pool.data + 2 * at);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = nonfinite_mask<false>(w[i]);
      bad |= ((m & 1u) | ((m >> 16) & 1u) << 1) << (2 * i);
    }
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(p.pool.data + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) bad |= ((nonfinite_mask<true>(i < 4 ? x.x : x.y) >> (8 * (i & 3))) & 1u) << i;
  }
  return bad;
}

// A sequence as a kernel sees it; `tiles` 0 unless it has units of that kind.
struct ChunkSeq {
  int q0, qlen, kvlen;
  int tiles;  // units of one KV head (small: one)
};

template <bool kTile>
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams& p, int s, int* err) {
  ChunkSeq q;
  q.q0 = p.batch.offsets[s];
  q.qlen = p.batch.offsets[s + 1] - q.q0;
  q.kvlen = p.batch.kv_len[s];
  if (q.kvlen < 0) {
    atomicCAS(err, 0, kErrSequence);
    q.kvlen = 0;
  }
  if (q.kvlen > p.capacity) {
    atomicCAS(err, 0, kErrBlockTable);
    q.kvlen = static_cast<int>(p.capacity);
  }
  if (q.qlen > p.max_chunk) {
    atomicCAS(err, 0, kErrSequence);
    q.qlen = 0;
  }
  const long long rows = static_cast<long long>(q.qlen) * p.group;
  q.tiles = q.qlen <= 0 || kTile == (rows <= kSmallRows) ? 0
            : kTile                                      ? static_cast<int>((rows + kUnitRows - 1) / kUnitRows)
                                                         : 1;
  return q;
}

// Unit i of a sequence's head: the last rows first, so that long units start.
template <bool kTile>
__device__ __forceinline__ ChunkUnit chunk_unit(const ChunkParams& p, const ChunkSeq& q, int s, int head, int i) {
  ChunkUnit u;
  u.seq = s;
  u.head = head;
  u.row0 = kTile ? (q.tiles - 1 - i) * kUnitRows : 0;
  const int rows = q.qlen * p.group;
  u.rows = kTile ? min(kUnitRows, rows - u.row0) : rows;
  u.q0 = q.q0;
  u.qlen = q.qlen;
  u.kvlen = q.kvlen;
  u.steps = unit_steps(q.kvlen, q.qlen, u.row0 + u.rows - 1, p.group);
  return u;
}

// Shared memory of a range's planning.
struct ChunkPlanShared {
  long long sums[16];  // steps (of one KV head) of each warp's sequences
  long long x, end;    // this range
  int seq, head, unit, kt;
  int err;             // the CTA's error word
};

__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ long long warp_scan(long long v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// a / b of numbers that are not negative; the short way where 32 bits hold them.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// The whole block (at most 16 warps): finds range g of `grid` in the list of
// units, in the order sequence, KV head, unit.  Warps sum runs of sequences;
// the one whose run holds the range's first step looks it up.  A batch whose
// offsets decrease or leave the packed rows is not run at all: its ranges are
// empty.  sh.err must be set before.
template <bool kTile>
__device__ __forceinline__ void chunk_plan(const ChunkParams& p, ChunkPlanShared& sh, int grid, int g) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int per = (p.batch.seqs + warps - 1) / warps;
  const int s0 = min(warp * per, p.batch.seqs), s1 = min(s0 + per, p.batch.seqs);
  // Steps of one head of sequence s; with kTile by the whole warp.
  auto steps_of = [&](int s) {
    const ChunkSeq q = chunk_seq<kTile>(p, s, &sh.err);
    if (!kTile) return static_cast<long long>(q.tiles ? chunk_unit<kTile>(p, q, s, 0, 0).steps : 0);
    long long n = 0;
    for (int i = lane; i < q.tiles; i += 32) n += chunk_unit<kTile>(p, q, s, 0, i).steps;
    return warp_sum(n);
  };
  bool bad = false;
  auto check = [&](int s) {
    const int o0 = p.batch.offsets[s], o1 = p.batch.offsets[s + 1];
    bad |= o0 < 0 || o1 < o0 || o1 > p.batch.rows;
  };
  long long sum = 0;
  if (kTile) {
    for (int s = s0; s < s1; ++s) {
      check(s);
      sum += steps_of(s);
    }
  } else {
    for (int s = s0 + lane; s < s1; s += 32) {
      check(s);
      sum += steps_of(s);
    }
    sum = warp_sum(sum);
  }
  if (lane == 0) sh.sums[warp] = sum;
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0) atomicCAS(&sh.err, 0, kErrSequence);
  const long long of_lane = lane < warps && !bad ? sh.sums[lane] : 0;
  const long long before = warp_sum(lane < warp ? of_lane : 0), total = warp_sum(of_lane);
  const int heads = p.pool.heads;
  const long long steps = total * heads, ranges = chunk_ranges(steps, grid);
  const bool none = total == 0 || g >= ranges;
  // The first `more` ranges have a step more than the others.
  const long long each = quotient(steps, ranges), more = steps - each * ranges;
  const long long x = none ? 0 : g * each + min(static_cast<long long>(g), more);
  const long long end = none ? 0 : x + each + (g < more ? 1 : 0);
  if (threadIdx.x == 0) {
    sh.x = x;
    sh.end = end;
  }
  if (!none && before * heads <= x && x < (before + sum) * heads) {  // this warp's run
    int seq = -1;
    long long at = before, in_seq = 0;
    if (kTile) {
      for (int s = s0; s < s1 && seq < 0; ++s) {
        in_seq = steps_of(s);
        if (x < (at + in_seq) * heads) seq = s;
        else at += in_seq;
      }
    } else {
      for (int b = s0; b < s1 && seq < 0; b += 32) {
        const long long n = b + lane < s1 ? steps_of(b + lane) : 0;
        const long long upto = at + warp_scan(n);
        const uint32_t past = __ballot_sync(0xffffffffu, x < upto * heads);
        if (past) {
          const int i = __ffs(past) - 1;
          seq = b + i;
          in_seq = __shfl_sync(0xffffffffu, n, i);
          at = __shfl_sync(0xffffffffu, upto, i) - in_seq;
        } else {
          at = __shfl_sync(0xffffffffu, upto, 31);
        }
      }
    }
    const long long rest = x - at * heads;
    const int head = static_cast<int>(quotient(rest, in_seq));
    long long kt = rest - head * in_seq;
    int unit = 0;
    if (kTile) {
      const ChunkSeq q = chunk_seq<kTile>(p, seq, &sh.err);
      for (int b = 0; b < q.tiles; b += 32) {
        const long long n = b + lane < q.tiles ? chunk_unit<kTile>(p, q, seq, 0, b + lane).steps : 0;
        const long long upto = warp_scan(n);
        const uint32_t past = __ballot_sync(0xffffffffu, kt < upto);
        if (past) {
          const int i = __ffs(past) - 1;
          unit = b + i;
          kt -= __shfl_sync(0xffffffffu, upto - n, i);
          break;
        }
        kt -= __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (lane == 0) {
      sh.seq = seq;
      sh.head = head;
      sh.unit = unit;
      sh.kt = static_cast<int>(kt);
    }
  }
  __syncthreads();
}

// A range's walk over its units: the part [kt0, kt1) of each one's steps.
//
// Tile units of a sequence share its K/V, and a long cache does not fit the L2:
// ranges should be at the same keys at the same time.  So a range that starts in
// the middle of a unit leaves that part for last: whole units first, from key 0
// on in every range, then the unit it leaves unfinished, likewise, then the
// part it started with.  (Ranges are equally long, so those last parts keep a
// constant distance in keys to the others too.)
template <bool kTile>
struct ChunkWalk {
  int left;  // steps of the range still to come, but for a part left for last
  int seq, head, unit, kt;
  ChunkSeq q;                                              // of seq
  int later_seq, later_head, later_unit, later_kt, later;  // that part and its steps

  __device__ __forceinline__ void init(const ChunkParams& p, const ChunkPlanShared& sh, int* err) {
    left = static_cast<int>(sh.end - sh.x);
    seq = sh.seq;
    head = sh.head;
    unit = sh.unit;
    kt = sh.kt;
    later = 0;
    if (left <= 0) return;
    q = chunk_seq<kTile>(p, seq, err);
    if (kTile && kt > 0) {
      const int rest = chunk_unit<kTile>(p, q, seq, head, unit).steps - kt;
      if (rest < left) {
        later = rest;
        later_seq = seq;
        later_head = head;
        later_unit = unit;
        later_kt = kt;
        left -= rest;
        advance(p, err);
      }
    }
  }
  __device__ __forceinline__ void advance(const ChunkParams& p, int* err) {
    kt = 0;
    if (left > 0 && ++unit == q.tiles) {
      unit = 0;
      if (++head == p.pool.heads) {
        head = 0;
        do {
          q = chunk_seq<kTile>(p, ++seq, err);
        } while (q.tiles == 0);
      }
    }
  }
  __device__ __forceinline__ bool next(const ChunkParams& p, int* err, ChunkUnit& u, int& kt0, int& kt1) {
    if (left <= 0) {
      if (!kTile || later == 0) return false;
      left = later;
      seq = later_seq;
      head = later_head;
      unit = later_unit;
      kt = later_kt;
      later = 0;
      q = chunk_seq<kTile>(p, seq, err);
    }
    u = chunk_unit<kTile>(p, q, seq, head, unit);
    kt0 = kt;
    kt1 = min(u.steps, kt + left);
    left -= kt1 - kt0;
    advance(p, err);
    return true;
  }
};

// Partial slot of a part of range g (-1: the whole unit).  A part that starts
// its unit without ending it is the range's last; every other partial part is
// the range's first.
__device__ __forceinline__ int part_slot(const ChunkUnit& u, int kt0, int kt1, int g) {
  return kt0 > 0 ? 2 * g : kt1 < u.steps ? 2 * g + 1 : -1;
}

// One thread of a CTA (pair) keeps its range's record.
__device__ __forceinline__ void clear_record(ChunkRecord& r) { r.last_cut = r.first_state = 0; }
__device__ __forceinline__ void note_part(ChunkRecord& r, const ChunkUnit& u, int kt0, int kt1) {
  if (kt0 > 0) {
    r.first_state = kt1 == u.steps ? 2 : 1;
  } else if (kt1 < u.steps) {
    r.last = u;
    r.last_cut = 1;
  }
}

__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Parts of the unit that range g of `grid` leaves unfinished: that range's, then the
// first parts of the ranges behind it up to the one that ends the unit.  0 if it
// cannot be merged: a range among them failed, or left no part of it.
// masks(b, stop, end): bits of the ranges b .. b + 31 whose first part is not one that
// goes on (or that failed, or do not exist), and of those whose part ends its unit.
template <typename Masks>
__host__ __device__ __forceinline__ int cut_parts(int g, int grid, bool failed, Masks masks) {
  if (failed) return 0;
  for (int b = g + 1; b < grid; b += 32) {
    uint32_t stop, end;
    masks(b, stop, end);
    if (stop == 0) continue;
    const uint32_t first = stop & (0u - stop);
    if ((end & first) == 0) return 0;
    int parts = b - g;  // g .. b - 1
    for (uint32_t i = first; i != 0; i >>= 1) ++parts;
    return parts;
  }
  return 0;
}

// Merges the parts of cut units: O = sum_i 2^(lse_i - M) O_i / sum_i 2^(lse_i -
// M); rows that saw no key are zeros.  Block (g, y) takes the rows [8 / kW y, ...)
// of the unit that range g left unfinished, if any: kW warps a row, each every
// kW-th part (few rows of many parts, as a long cache leaves them, or many of few).
// For tile units one: four gained 4 us with 37 parts a unit and lost 4 to 6 with 4
// to 8; four rows a warp, their loads side by side, lost up to 30.
template <int D, int kW, bool kTile>
__device__ __forceinline__ void combine_rows(const ChunkParams& p, const ChunkRecord* rec, int grid, int unit_rows,
                                             const float* part_o, const float* part_lse, int g, int y) {
  constexpr int kPer = D / 32;
  __shared__ float s_acc[kW > 1 ? 8 : 1][D];
  __shared__ float s_w[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (!rec[g].last_cut) return;
  const ChunkUnit unit = rec[g].last;
  const int r = y * (8 / kW) + warp / kW;
  if (y * (8 / kW) >= unit.rows) return;
  // Slot 2 g + 1, then the first parts of the ranges behind it.
  auto failed_range = [&](int i) { return (kTile ? p.work.tile_rec[2 * i].failed | p.work.tile_rec[2 * i + 1].failed
                                                 : p.work.small_rec[i].failed) != 0; };
  const int parts = cut_parts(g, grid, failed_range(g), [&](int b, uint32_t& stop, uint32_t& end) {
    const bool there = b + lane < grid && !failed_range(b + lane);
    const int state = there ? rec[b + lane].first_state : 0;
    stop = __ballot_sync(0xffffffffu, state != 1);
    end = __ballot_sync(0xffffffffu, state == 2);
  });
  if (parts == 0) return;
  // (Warps behind the unit's last row go along with it and write nothing.)
  auto row_of = [&](int i) {
    return static_cast<long long>(i == 0 ? 2 * g + 1 : 2 * (g + i)) * unit_rows + min(r, unit.rows - 1);
  };
  float m = -INFINITY, acc[kPer], wsum = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
  for (int b = lane; b < parts; b += 32) m = fmaxf(m, part_lse[row_of(b)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m == -INFINITY) m = 0.f;
#pragma unroll 4
  for (int i = warp % kW; i < parts; i += kW) {
    const long long row = row_of(i);
    const float lse = part_lse[row];
    float4 v[kPer / 4];
#pragma unroll
    for (int c = 0; c < kPer / 4; ++c) v[c] = reinterpret_cast<const float4*>(part_o + row * D + lane * kPer)[c];
    // A part whose row saw nothing weighs nothing, whatever its O holds; a NaN (a
    // NaN score somewhere) passes on.
    const float w = lse == -INFINITY ? 0.f : ex2_approx(lse - m);
    wsum += w;
#pragma unroll
    for (int c = 0; c < kPer / 4; ++c) {
      acc[4 * c] = w == 0.f ? acc[4 * c] : fmaf(w, v[c].x, acc[4 * c]);
      acc[4 * c + 1] = w == 0.f ? acc[4 * c + 1] : fmaf(w, v[c].y, acc[4 * c + 1]);
      acc[4 * c + 2] = w == 0.f ? acc[4 * c + 2] : fmaf(w, v[c].z, acc[4 * c + 2]);
      acc[4 * c + 3] = w == 0.f ? acc[4 * c + 3] : fmaf(w, v[c].w, acc[4 * c + 3]);
    }
  }
  if (kW > 1) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) s_acc[warp][lane * kPer + k] = acc[k];
    if (lane == 0) s_w[warp] = wsum;
    __syncthreads();
    if (warp % kW) return;
    for (int w = 1; w < kW; ++w) {
      wsum += s_w[warp + w];
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] += s_acc[warp + w][lane * kPer + k];
    }
  }
  if (r >= unit.rows) return;
  const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
  const int row = unit.row0 + r;
  if (kTile) {
    bool patch = false;
    for (int i = lane; i < 2 * parts; i += 32) patch |= rec[2 * g + i].patch != 0;
    if (__any_sync(0xffffffffu, patch)) {
      uint32_t bad = 0;
      const int pos = unit.kvlen - unit.qlen + row / p.group;
      for (int key = max(0, keys_all_see(unit.kvlen, unit.qlen, unit.row0, p.group)); key <= pos; ++key)
        bad |= nonfinite8<D>(p, unit.seq, unit.head, key, lane * kPer & ~7) >> (lane * kPer & 7);
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        if ((bad >> k) & 1u) acc[k] = NAN;
    }
  }
  __nv_bfloat16* dst = p.out + static_cast<long long>(unit.head * p.group + row % p.group) * p.out_head +
                       static_cast<long long>(unit.q0 + row / p.group) * p.out_row + lane * kPer;
#pragma unroll
  for (int k = 0; k < kPer; k += 4)
    *reinterpret_cast<uint2*>(dst + k) =
        make_uint2(pack_bf16x2(acc[k] * inv, acc[k + 1] * inv), pack_bf16x2(acc[k + 2] * inv, acc[k + 3] * inv));
}

constexpr int kCombineSmallW = 4, kCombineTileW = 1;  // warps a row

// The whole units of tile range g, if it took any values of V for zeros: NaN into
// the output of the rows that see them, in their columns.  A warp a unit, eight
// columns a lane.
template <int D>
__device__ __forceinline__ void patch_range(const ChunkParams& p, int g) {
  if (!p.work.tile_rec[2 * g].patch && !p.work.tile_rec[2 * g + 1].patch) return;
  __shared__ ChunkPlanShared sh;
  if (threadIdx.x == 0) sh.err = 0;  // (reported already)
  __syncthreads();
  chunk_plan<true>(p, sh, p.tile_pairs, g);
  ChunkWalk<true> walk;
  walk.init(p, sh, &sh.err);
  ChunkUnit u;
  int kt0, kt1;
  for (int n = 0; walk.next(p, &sh.err, u, kt0, kt1); ++n) {
    if (n % 8 != threadIdx.x / 32 || part_slot(u, kt0, kt1, g) >= 0) continue;  // (a cut one: combine_rows)
    const int before = u.kvlen - u.qlen;
    for (int d = 8 * (threadIdx.x & 31); d < D; d += 256) {
      uint32_t bad = 0;
      const int end = before + (u.row0 + u.rows - 1) / p.group;
      for (int key = max(0, keys_all_see(u.kvlen, u.qlen, u.row0, p.group)); key <= end; ++key) {
        bad |= nonfinite8<D>(p, u.seq, u.head, key, d);
        if (bad == 0) continue;
        const int token = key - before;
        for (int h = 0; h < p.group; ++h) {
          const int row = token * p.group + h;
          if (row < u.row0 || row >= u.row0 + u.rows) continue;
          __nv_bfloat16* dst = p.out + static_cast<long long>(u.head * p.group + h) * p.out_head +
                               static_cast<long long>(u.q0 + token) * p.out_row + d;
          for (int i = 0; i < 8; ++i)
            if ((bad >> i) & 1u) dst[i] = __float2bfloat16(NAN);
        }
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(256) chunk_combine_kernel(const ChunkParams p) {
  grid_dependency_wait();
  const int small_blocks = p.small_ctas * p.small_y;
  if (blockIdx.x == 0) {
    int err = 0;
    for (int i = threadIdx.x; i < p.small_ctas + 2 * p.tile_pairs; i += 256) {
      const int e = i < p.small_ctas ? p.work.small_rec[i].err : p.work.tile_rec[i - p.small_ctas].err;
      err = max(err, e);
    }
    for (int o = 16; o > 0; o >>= 1) err = max(err, __shfl_xor_sync(0xffffffffu, err, o));
    __shared__ int s_err[8];
    if ((threadIdx.x & 31) == 0) s_err[threadIdx.x >> 5] = err;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) err = max(err, s_err[w]);
      if (err) atomicCAS(p.status, 0, err);
    }
  }
  if (blockIdx.x < small_blocks) {
    combine_rows<D, kCombineSmallW, false>(p, p.work.small_rec, p.small_ctas, kSmallRows, p.work.small_o, p.work.small_lse,
                       blockIdx.x / p.small_y, blockIdx.x % p.small_y);
  } else {
    const int b = blockIdx.x - small_blocks;
    if (b >= p.tile_pairs * p.tile_y) {
      patch_range<D>(p, b - p.tile_pairs * p.tile_y);
      return;
    }
    combine_rows<D, kCombineTileW, true>(p, p.work.tile_rec, p.tile_pairs, kUnitRows, p.work.tile_o, p.work.tile_lse,
                                         b / p.tile_y, b % p.tile_y);
  }
}

}  // namespace pcp
