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
// one gets the same work whatever the lengths.  A unit that a range boundary
// cuts leaves fp32 partials, which chunk_combine_kernel merges.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "attn_common.cuh"
#include "ptx.cuh"
#include "serve_ops.cuh"

namespace pcp {

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

struct ChunkPlan {
  int small_units, tile_units;
  long long small_steps, tile_steps;
};

// Where a launch's scratch lies.
struct ChunkWork {
  ChunkPlan* plan;
  ChunkUnit* small;
  long long* small_start;  // first step of each unit, and the total
  ChunkUnit* tile;
  long long* tile_start;
  int* seq_tile;           // [seqs + 1]: query tiles (per head) before each sequence
  long long* tile_prefix;  // [query tiles + 1]: their steps
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
  int max_chunk;
  float scale_log2;
  int small_ctas, tile_pairs;  // grids of the two kernels
  int* err;
};

__device__ __forceinline__ float exp2_of_int(int e) {  // 2^e, 0 below the normal range
  return __uint_as_float(static_cast<uint32_t>(min(max(e + 127, 0), 254)) << 23);
}

// CTAs (or pairs) that a list of `steps` is cut for: at least one step each.
__host__ __device__ __forceinline__ long long chunk_ranges(long long steps, int grid) {
  return steps < grid ? (steps > 1 ? steps : 1) : grid;
}

// Exclusive block scan over 1024 threads; `total` gets the sum.
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the sums of an earlier scan are read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  long long before = 0, all = 0;
  const long long w = warp_sums[lane];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const long long s = __shfl_sync(0xffffffffu, w, i);
    if (i < warp) before += s;
    all += s;
  }
  total = all;
  return before + x - v;
}

// Steps of rows [row0, row0 + rows) of a sequence: tiles up to the last row's
// position.
__device__ __forceinline__ int unit_steps(int kvlen, int qlen, int last_row, int group) {
  const int visible = kvlen - qlen + last_row / group + 1;
  return max(1, (visible + kStepKeys - 1) / kStepKeys);
}

// One block of 1024 threads: checks the batch, then lists the units and their
// steps.  A batch whose offsets decrease or leave the packed rows is not run
// at all (its units could overlap or pass the scratch).
__global__ void __launch_bounds__(1024, 1) chunk_plan_kernel(const ChunkParams p) {
  __shared__ long long sums[32];
  const BatchView& b = p.batch;
  const int tid = threadIdx.x;
  const int Hkv = p.pool.heads;
  const long long capacity = static_cast<long long>(b.table_width) * p.pool.block_size;
  if (tid == 0) *p.err = 0;
  bool bad = false;
  for (int s = tid; s < b.seqs; s += 1024) {
    const int o0 = b.offsets[s], o1 = b.offsets[s + 1];
    bad |= o0 < 0 || o1 < o0 || o1 > b.rows;
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) {
      atomicCAS(p.err, 0, kErrSequence);
      *p.work.plan = {0, 0, 0, 0};
    }
    return;
  }
  long long small0 = 0, steps0 = 0, tile0 = 0;  // totals of the sequences before this block of 1024
  for (int base = 0; base < b.seqs; base += 1024) {
    const int s = base + tid;
    int qlen = 0, kvlen = 0, q0 = 0;
    if (s < b.seqs) {
      q0 = b.offsets[s];
      qlen = b.offsets[s + 1] - q0;
      kvlen = b.kv_len[s];
      if (kvlen < 0 || qlen > p.max_chunk) {
        atomicCAS(p.err, 0, kErrSequence);
        if (qlen > p.max_chunk) qlen = 0;
        kvlen = max(kvlen, 0);
      }
      if (kvlen > capacity) {
        atomicCAS(p.err, 0, kErrBlockTable);
        kvlen = static_cast<int>(capacity);
      }
    }
    const long long rows = static_cast<long long>(qlen) * p.group;
    const bool small = qlen > 0 && rows <= kSmallRows;
    const int tiles = qlen > 0 && !small ? static_cast<int>((rows + kUnitRows - 1) / kUnitRows) : 0;
    const int steps = small ? unit_steps(kvlen, qlen, static_cast<int>(rows) - 1, p.group) : 0;
    long long n_small, n_steps, n_tiles;
    const long long u = small0 + block_scan(small ? 1 : 0, sums, n_small);
    const long long st = steps0 + block_scan(steps, sums, n_steps);
    const long long t = tile0 + block_scan(tiles, sums, n_tiles);
    if (small)
      for (int h = 0; h < Hkv; ++h) {
        p.work.small[u * Hkv + h] = {s, h, 0, static_cast<int>(rows), q0, qlen, kvlen, steps};
        p.work.small_start[u * Hkv + h] = st * Hkv + static_cast<long long>(h) * steps;
      }
    if (s < b.seqs) p.work.seq_tile[s] = static_cast<int>(t);
    small0 += n_small;
    steps0 += n_steps;
    tile0 += n_tiles;
  }
  if (tid == 0) {
    p.work.small_start[small0 * Hkv] = steps0 * Hkv;
    p.work.seq_tile[b.seqs] = static_cast<int>(tile0);
    *p.work.plan = {static_cast<int>(small0 * Hkv), static_cast<int>(tile0 * Hkv), steps0 * Hkv, 0};
  }
  if (tile0 == 0) return;
  __syncthreads();
  // Steps before each query tile (of one head).  Tiles of a sequence are
  // listed last first: the longest ones start.
  auto find = [&](int t) {
    int lo = 0, n = b.seqs;
    while (n > 1) {
      const int h = n >> 1;
      if (p.work.seq_tile[lo + h] <= t) lo += h, n -= h;
      else n = h;
    }
    return lo;
  };
  auto unit_of = [&](int t, int s) {
    const int tiles = p.work.seq_tile[s + 1] - p.work.seq_tile[s];
    const int q0 = b.offsets[s], qlen = b.offsets[s + 1] - q0;
    const int kvlen = static_cast<int>(min(static_cast<long long>(max(b.kv_len[s], 0)), capacity));
    const int row0 = (tiles - 1 - (t - p.work.seq_tile[s])) * kUnitRows;
    const int rows = static_cast<int>(min(static_cast<long long>(kUnitRows), static_cast<long long>(qlen) * p.group - row0));
    return ChunkUnit{s, 0, row0, rows, q0, qlen, kvlen, unit_steps(kvlen, qlen, row0 + rows - 1, p.group)};
  };
  long long done = 0;
  for (int base = 0; base < tile0; base += 1024) {
    const int t = base + tid;
    const int steps = t < tile0 ? unit_of(t, find(t)).steps : 0;
    long long n;
    const long long before = block_scan(steps, sums, n);
    if (t < tile0) p.work.tile_prefix[t] = done + before;
    done += n;
  }
  if (tid == 0) {
    p.work.tile_prefix[tile0] = done;
    p.work.tile_start[tile0 * Hkv] = done * Hkv;
    p.work.plan->tile_steps = done * Hkv;
  }
  __syncthreads();
  // Units in the order sequence, KV head, tile: a pair's neighbours share K/V.
  for (long long i = tid; i < tile0 * Hkv; i += 1024) {
    const int t = static_cast<int>(i / Hkv), h = static_cast<int>(i % Hkv);
    const int s = find(t);
    ChunkUnit u = unit_of(t, s);
    u.head = h;
    const int first = p.work.seq_tile[s], tiles = p.work.seq_tile[s + 1] - first;
    const long long at0 = p.work.tile_prefix[first];
    const long long idx = static_cast<long long>(first) * Hkv + static_cast<long long>(h) * tiles + (t - first);
    p.work.tile[idx] = u;
    p.work.tile_start[idx] =
        at0 * Hkv + h * (p.work.tile_prefix[first + tiles] - at0) + (p.work.tile_prefix[t] - at0);
  }
}

// A range's walk over its units: the part [kt0, kt1) of each one's steps.
struct ChunkWalk {
  const ChunkUnit* units;
  const long long* start;
  long long x, end;
  int u;
  int range;

  __device__ __forceinline__ void init(const ChunkUnit* list, const long long* starts, int n, long long steps, int grid,
                                       int g) {
    units = list;
    start = starts;
    range = g;
    const long long ranges = chunk_ranges(steps, grid);
    x = end = 0;
    u = 0;
    if (n == 0 || g >= ranges) return;
    x = steps * g / ranges;
    end = steps * (g + 1) / ranges;
    int k = n;  // the unit that holds step x
    while (k > 1) {
      const int h = k >> 1;
      if (start[u + h] <= x) u += h, k -= h;
      else k = h;
    }
  }
  // The next part: its unit, steps [kt0, kt1) and partial slot (-1: the whole
  // unit).  A part that starts its unit is the range's last (slot 2 range + 1)
  // if it does not end it; every other partial part is the range's first.
  __device__ __forceinline__ bool next(ChunkUnit& unit, int& kt0, int& kt1, int& slot) {
    if (x >= end) return false;
    unit = units[u];
    const long long s0 = start[u], s1 = s0 + unit.steps;
    const long long to = s1 < end ? s1 : end;
    kt0 = static_cast<int>(x - s0);
    kt1 = static_cast<int>(to - s0);
    slot = kt0 == 0 ? (to == s1 ? -1 : 2 * range + 1) : 2 * range;
    x = to;
    ++u;
    return true;
  }
};

// Merges the parts of split units: O = sum_i 2^(lse_i - M) O_i / sum_i 2^(lse_i
// - M).  A block takes kSmallRows rows of a unit, a warp a row at a time; rows
// that saw no key are zeros.  Blocks of whole units leave at once.
template <int D>
__global__ void __launch_bounds__(256) chunk_combine_kernel(const ChunkParams p) {
  constexpr int kPer = D / 32;
  constexpr int kParts = kUnitRows / kSmallRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const ChunkPlan plan = *p.work.plan;
  const long long items = plan.small_units + static_cast<long long>(plan.tile_units) * kParts;
  for (long long it = blockIdx.x; it < items; it += gridDim.x) {
    const bool small = it < plan.small_units;
    const long long u = small ? it : (it - plan.small_units) / kParts;
    const int r0 = small ? 0 : static_cast<int>((it - plan.small_units) % kParts) * kSmallRows;
    const long long steps = small ? plan.small_steps : plan.tile_steps;
    const long long ranges = chunk_ranges(steps, small ? p.small_ctas : p.tile_pairs);
    const ChunkUnit unit = (small ? p.work.small : p.work.tile)[u];
    const long long s0 = (small ? p.work.small_start : p.work.tile_start)[u];
    const long long g0 = stream_k_pair_of(s0, steps, ranges);
    const long long g1 = stream_k_pair_of(s0 + unit.steps - 1, steps, ranges);
    if (g0 == g1) continue;
    const int unit_rows = small ? kSmallRows : kUnitRows;
    const float* part_o = small ? p.work.small_o : p.work.tile_o;
    const float* part_lse = small ? p.work.small_lse : p.work.tile_lse;
    for (int r = r0 + warp; r < min(r0 + kSmallRows, unit.rows); r += 8) {
      // Lane i follows part i of each 32.
      float m = -INFINITY, acc[kPer], wsum = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
      for (long long gb = g0; gb <= g1; gb += 32) {
        const long long g = gb + lane;
        const long long slot = g == g0 ? 2 * g + 1 : 2 * g;
        const float lse = g <= g1 ? part_lse[slot * unit_rows + r] : -INFINITY;
        float mx = lse;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float nm = fmaxf(m, mx);
        // A NaN lse (a NaN score somewhere) passes into its weight.
        const float w = lse == -INFINITY ? 0.f : ex2_approx(lse - (nm == -INFINITY ? 0.f : nm));
        const float keep = m == -INFINITY ? 0.f : ex2_approx(m - nm);
        m = nm;
        wsum *= keep;
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] *= keep;
        const int n = static_cast<int>(min(32LL, g1 - gb + 1));
        for (int i = 0; i < n; ++i) {
          const float wi = __shfl_sync(0xffffffffu, w, i);
          if (wi == 0.f) continue;  // a part whose rows saw nothing wrote no O
          wsum += wi;
          const long long gi = gb + i;
          const long long si = gi == g0 ? 2 * gi + 1 : 2 * gi;
          const float* src = part_o + (si * unit_rows + r) * D + lane * kPer;
#pragma unroll
          for (int k = 0; k < kPer; k += 4) {
            const float4 v = *reinterpret_cast<const float4*>(src + k);
            acc[k] = fmaf(wi, v.x, acc[k]);
            acc[k + 1] = fmaf(wi, v.y, acc[k + 1]);
            acc[k + 2] = fmaf(wi, v.z, acc[k + 2]);
            acc[k + 3] = fmaf(wi, v.w, acc[k + 3]);
          }
        }
      }
      const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
      const int row = unit.row0 + r;
      __nv_bfloat16* dst = p.out + static_cast<long long>(unit.head * p.group + row % p.group) * p.out_head +
                           static_cast<long long>(unit.q0 + row / p.group) * p.out_row + lane * kPer;
#pragma unroll
      for (int k = 0; k < kPer; k += 4)
        *reinterpret_cast<uint2*>(dst + k) = make_uint2(pack_bf16x2(acc[k] * inv, acc[k + 1] * inv),
                                                        pack_bf16x2(acc[k + 2] * inv, acc[k + 3] * inv));
    }
  }
}

}  // namespace pcp
