// Memory-bound serving kernels: norm and rotation of query and key heads,
// and the scaled paged cache's append and read-back (include/pcp_serve.h).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "attn_common.cuh"
#include "e4m3.cuh"
#include "ptx.cuh"

namespace pcp {

constexpr int kErrSequence = 112;  // a sequence the call does not take (include/pcp_serve.h)

// ------------------------------------------------- eight elements a lane --
template <typename T>
struct Vec8;  // raw: what is loaded and stored at once

template <>
struct Vec8<__nv_bfloat16> {
  uint4 r;
  __device__ __forceinline__ void load(const void* p) { r = *static_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* f) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ void store(void* p, const float* f) {
    *static_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                                         pack_bf16x2(f[6], f[7]));
  }
};

template <>
struct Vec8<__half> {
  uint4 r;
  __device__ __forceinline__ void load(const void* p) { r = *static_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* f) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
  static __device__ __forceinline__ void store(void* p, const float* f) {
    *static_cast<uint4*>(p) = make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]),
                                         pack_f16x2(f[6], f[7]));
  }
};

template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* p) {
    a = static_cast<const float4*>(p)[0];
    b = static_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
  static __device__ __forceinline__ void store(void* p, const float* f) {
    static_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    static_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};

// ------------------------------------------------------- norm and rotation --
struct HeadRows {  // [heads][rows][head_dim] at any head and row stride (elements)
  const void* in;
  void* out;
  long long in_head, in_row, out_head, out_row;
  int heads;
  const void* weight;  // NULL: no norm
};

struct NormRopeParams {
  HeadRows q, k;
  int rows;
  int head_dim, rotary_dim;
  int lanes;          // lanes a head takes: head_dim / 16 rounded up to a power of two
  int passes;         // passes of 32 / lanes heads: of q's, then of k's
  int passes_q;
  int per_warp;       // passes of one row that a warp takes
  int interleaved;
  const void* positions;
  int positions_64;
  const unsigned long long* turns;  // turns per position of each pair, as a 64-bit fraction
  float magnitude;
  float eps;
};

// A warp takes one row (token) and some of its heads, 16 elements of a head a
// lane: the mean of squares is one shuffle reduction, and a rotated pair's two
// halves sit in one lane -- half layout: eight elements at 8 l and the eight at
// 8 l + rotary_dim / 2; interleaved: sixteen in a row -- so nothing else moves
// between lanes.  cos and sin are made once per row and lane, from the position
// times the pair's turns in 64-bit integers (whole turns overflow away, so
// there is no table to read and no error that grows with the position), and
// used for every head of the warp.  Bound by HBM: each element is read and
// written once; kUnroll passes' loads are in flight together.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const NormRopeParams p) {
  constexpr int kUnroll = sizeof(T) == 4 ? 2 : 4;
  const int lane = threadIdx.x & 31;
  const int parts = (p.passes + p.per_warp - 1) / p.per_warp;
  const long long items = static_cast<long long>(p.rows) * parts;
  const int l = lane & (p.lanes - 1);
  const int sub = lane / p.lanes;       // which of the pass's heads
  const int per_pass = 32 / p.lanes;
  const int half = p.rotary_dim / 2;
  const bool live_lane = 16 * l < p.head_dim;
  // First elements of this lane's two runs of eight, and whether they turn.
  bool turned = 16 * l < p.rotary_dim;
  int e0 = 16 * l, e1 = 16 * l + 8;
  if (turned && !p.interleaved) e0 = 8 * l, e1 = 8 * l + half;
  const float inv_d = 1.f / static_cast<float>(p.head_dim);

  for (long long item = blockIdx.x * 8LL + (threadIdx.x >> 5); item < items; item += gridDim.x * 8LL) {
    const int row = static_cast<int>(item / parts);
    const int p0 = static_cast<int>(item % parts) * p.per_warp;
    const int p1 = min(p0 + p.per_warp, p.passes);
    float co[8], si[8];
    bool have_angles = false;
    float w0[8], w1[8];
    for (int pb = p0; pb < p1; pb += kUnroll) {
      Vec8<T> x0[kUnroll], x1[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int pass = pb + u;
        if (pass >= p1 || !live_lane) continue;
        const bool is_k = pass >= p.passes_q;
        const HeadRows& h = is_k ? p.k : p.q;
        const int head = (is_k ? pass - p.passes_q : pass) * per_pass + sub;
        if (head >= h.heads) continue;
        const T* in = static_cast<const T*>(h.in) + head * h.in_head + row * h.in_row;
        x0[u].load(in + e0);
        x1[u].load(in + e1);
      }
      if (!have_angles) {  // behind the first loads
        have_angles = true;
        if (turned) {
          const long long pos = p.positions_64 ? static_cast<const long long*>(p.positions)[row]
                                               : static_cast<const int*>(p.positions)[row];
          const int pair0 = 8 * l;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const unsigned long long t = static_cast<unsigned long long>(pos) * p.turns[pair0 + i];
            // the top 32 bits as half turns in [-1, 1)
            const float a = static_cast<float>(static_cast<int>(t >> 32)) * 4.656612873077393e-10f;
            sincospif(a, &si[i], &co[i]);
            si[i] *= p.magnitude;
            co[i] *= p.magnitude;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int pass = pb + u;
        if (pass >= p1) continue;  // the same for the whole warp
        const bool is_k = pass >= p.passes_q;
        const HeadRows& h = is_k ? p.k : p.q;
        const int head = (is_k ? pass - p.passes_q : pass) * per_pass + sub;
        const bool live = live_lane && head < h.heads;
        float f0[8], f1[8];
        if (live) {
          x0[u].get(f0);
          x1[u].get(f1);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) f0[i] = f1[i] = 0.f;
        }
        if (h.weight) {
          if ((pass == p0 || pass == p.passes_q) && live_lane) {
            Vec8<T> a, b;
            a.load(static_cast<const T*>(h.weight) + e0);
            b.load(static_cast<const T*>(h.weight) + e1);
            a.get(w0);
            b.get(w1);
          }
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = fmaf(f0[i], f0[i], fmaf(f1[i], f1[i], ss));
          for (int o = p.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float r = rsqrtf(ss * inv_d + p.eps);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            f0[i] = f0[i] * r * w0[i];
            f1[i] = f1[i] * r * w1[i];
          }
        }
        if (turned) {
          if (p.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float a = f0[2 * i], b = f0[2 * i + 1], c = f1[2 * i], d = f1[2 * i + 1];
              f0[2 * i] = a * co[i] - b * si[i];
              f0[2 * i + 1] = b * co[i] + a * si[i];
              f1[2 * i] = c * co[i + 4] - d * si[i + 4];
              f1[2 * i + 1] = d * co[i + 4] + c * si[i + 4];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float a = f0[i], b = f1[i];
              f0[i] = a * co[i] - b * si[i];
              f1[i] = b * co[i] + a * si[i];
            }
          }
        }
        if (live) {
          T* out = static_cast<T*>(h.out) + head * h.out_head + row * h.out_row;
          Vec8<T>::store(out + e0, f0);
          Vec8<T>::store(out + e1, f1);
        }
      }
    }
  }
}

// ------------------------------------------- paged cache: append and read --
struct BatchView {
  const int* offsets;  // [seqs + 1]
  const int* kv_len;   // [seqs]
  const int* tables;   // [seqs][table_width], table_stride apart
  long long table_stride;
  int table_width;
  int seqs;
  int rows;
};

struct PoolView {
  uint8_t* data;
  uint8_t* scales;  // NULL: unit scale
  long long blocks;
  int heads, head_dim, block_size, bf16;
};

// The sequence whose rows hold `row`, or -1: the last one that starts at or
// before it, when it also ends after it.
__device__ __forceinline__ int sequence_of(const BatchView& b, int row) {
  int lo = 0, n = b.seqs;  // the answer, if any, is in [lo, lo + n)
  while (n > 1) {
    const int h = n >> 1;
    if (b.offsets[lo + h] <= row) {
      lo += h;
      n -= h;
    } else {
      n = h;
    }
  }
  return b.offsets[lo] <= row && row < b.offsets[lo + 1] ? lo : -1;
}

struct CacheRowsParams {
  PoolView pool;
  BatchView batch;
  const void* k;  // append: source rows; read: destination rows
  const void* v;
  long long k_head, k_row, v_head, v_row;
  int tokens_per_warp;     // up to 32
  unsigned inv_per_token;  // ceil(2^32 / (2 heads)): exact quotients of a warp's row numbers
  int* err;
};

// Where a packed row's token lies: its pool block (-1: no sequence's row, -2: a
// table entry that cannot be followed, -3: a position below 0) and the row in it.
__device__ __forceinline__ int2 pool_row(const PoolView& pool, const BatchView& b, int row) {
  const int s = sequence_of(b, row);
  if (s < 0) return {-1, 0};
  const int pos = b.kv_len[s] - b.offsets[s + 1] + row;
  if (pos < 0) return {-3, 0};
  const int lb = pos / pool.block_size;
  if (lb >= b.table_width) return {-2, 0};
  const int blk = b.tables[s * b.table_stride + lb];
  if (blk < 0 || blk >= pool.blocks) return {-2, 0};
  return {blk, pos - lb * pool.block_size};
}

// Both kernels: a warp takes tokens_per_warp consecutive packed rows; lane i
// follows row i's offsets, length and table entry (the chains of dependent
// loads run side by side), then the warp walks its (token, K/V, head) rows, 16
// elements a lane: 32-byte bf16 and 16-byte code accesses.  Bound by HBM; the
// loads of kRowsInFlight rows a lane are in flight together.
constexpr int kRowsInFlight = 4;

// Row r of a warp's n (token, K/V, head) rows.
struct CacheRow {
  int tok, which;   // token of the warp, is_v * heads + head
  int blk;          // as pool_row's, or -1 past the warp's rows
  long long prow;   // row of the pool, valid when blk >= 0
};

__device__ __forceinline__ CacheRow cache_row(const CacheRowsParams& p, int r, int n, int2 mine) {
  CacheRow c;
  const int per_token = 2 * p.pool.heads;
  c.tok = r < n ? static_cast<int>(__umulhi(static_cast<unsigned>(r), p.inv_per_token)) : 0;
  c.which = r - c.tok * per_token;
  c.blk = __shfl_sync(0xffffffffu, mine.x, c.tok);
  const int slot = __shfl_sync(0xffffffffu, mine.y, c.tok);
  if (r >= n) c.blk = -1;
  c.prow = (static_cast<long long>(c.blk) * per_token + c.which) * p.pool.block_size + slot;
  return c;
}

// Element offset of a packed row's head.
__device__ __forceinline__ const __nv_bfloat16* packed_row(const CacheRowsParams& p, long long row, int which) {
  const bool is_v = which >= p.pool.heads;
  return static_cast<const __nv_bfloat16*>(is_v ? p.v : p.k) +
         (is_v ? which - p.pool.heads : which) * (is_v ? p.v_head : p.k_head) + row * (is_v ? p.v_row : p.k_row);
}

template <int D>
__global__ void __launch_bounds__(256) cache_append_kernel(const CacheRowsParams p) {
  constexpr int kLanes = D / 16;      // lanes of a row: 8 or 16
  constexpr int kSide = 32 / kLanes;  // rows side by side
  const int lane = threadIdx.x & 31;
  const int l = lane % kLanes, side = lane / kLanes;
  const int tpw = p.tokens_per_warp;
  const PoolView& pool = p.pool;
  for (long long t0 = (blockIdx.x * 8LL + (threadIdx.x >> 5)) * tpw; t0 < p.batch.rows; t0 += gridDim.x * 8LL * tpw) {
    const int tokens = static_cast<int>(min(static_cast<long long>(tpw), p.batch.rows - t0));
    int2 mine = {-1, 0};
    if (lane < tokens) {
      mine = pool_row(pool, p.batch, static_cast<int>(t0) + lane);
      if (mine.x < -1) atomicCAS(p.err, 0, mine.x == -2 ? kErrBlockTable : kErrSequence);
    }
    const int n = tokens * 2 * pool.heads;
    for (int r0 = 0; r0 < n; r0 += kSide * kRowsInFlight) {
      uint4 x[kRowsInFlight][2];
      CacheRow c[kRowsInFlight];
#pragma unroll
      for (int u = 0; u < kRowsInFlight; ++u) {
        c[u] = cache_row(p, r0 + u * kSide + side, n, mine);
        x[u][0] = x[u][1] = make_uint4(0u, 0u, 0u, 0u);
        if (c[u].blk >= 0) {
          const uint4* src = reinterpret_cast<const uint4*>(packed_row(p, t0 + c[u].tok, c[u].which) + 16 * l);
          x[u][0] = src[0];
          x[u][1] = src[1];
        }
      }
#pragma unroll
      for (int u = 0; u < kRowsInFlight; ++u) {
        const bool live = c[u].blk >= 0;
        if (pool.bf16) {
          uint4* dst = reinterpret_cast<uint4*>(pool.data + (c[u].prow * D + 16 * l) * 2);
          if (live) dst[0] = x[u][0], dst[1] = x[u][1];
          continue;
        }
        float f[16];
        Vec8<__nv_bfloat16>{x[u][0]}.get(f);
        Vec8<__nv_bfloat16>{x[u][1]}.get(f + 8);
        if (pool.scales) {
          // Largest finite magnitude, as bits (they order like the values).
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t a = __float_as_uint(f[i]) & 0x7FFFFFFFu;
            if (a < 0x7F800000u) m = max(m, a);
          }
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          // 448 = 1.75 * 2^8: the least e with amax <= 448 * 2^e comes from
          // the exponent and whether the fraction is above 0.75.
          int e = static_cast<int>(m >> 23) - 127 - 8 + ((m & 0x7FFFFFu) > 0x600000u ? 1 : 0);
          e = m == 0 ? 0 : min(max(e, -100), 120);
          const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] *= inv;
          if (live && l == 0) pool.scales[c[u].prow] = static_cast<uint8_t>(e + 127);
        }
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = e4m3x2_from_floats(f[4 * i], f[4 * i + 1]) |
                 (static_cast<uint32_t>(e4m3x2_from_floats(f[4 * i + 2], f[4 * i + 3])) << 16);
        if (live) *reinterpret_cast<uint4*>(pool.data + c[u].prow * D + 16 * l) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheRowsParams p) {
  constexpr int kLanes = D / 16;
  constexpr int kSide = 32 / kLanes;
  const int lane = threadIdx.x & 31;
  const int l = lane % kLanes, side = lane / kLanes;
  const int tpw = p.tokens_per_warp;
  const PoolView& pool = p.pool;
  for (long long t0 = (blockIdx.x * 8LL + (threadIdx.x >> 5)) * tpw; t0 < p.batch.rows; t0 += gridDim.x * 8LL * tpw) {
    const int tokens = static_cast<int>(min(static_cast<long long>(tpw), p.batch.rows - t0));
    int2 mine = {-1, 0};
    if (lane < tokens) {
      mine = pool_row(pool, p.batch, static_cast<int>(t0) + lane);
      if (mine.x < -1) atomicCAS(p.err, 0, mine.x == -2 ? kErrBlockTable : kErrSequence);
    }
    const int n = tokens * 2 * pool.heads;
    for (int r0 = 0; r0 < n; r0 += kSide * kRowsInFlight) {
      uint4 x[kRowsInFlight][2];
      uint32_t sc[kRowsInFlight];
      CacheRow c[kRowsInFlight];
#pragma unroll
      for (int u = 0; u < kRowsInFlight; ++u) {
        c[u] = cache_row(p, r0 + u * kSide + side, n, mine);
        x[u][0] = x[u][1] = make_uint4(0u, 0u, 0u, 0u);
        sc[u] = 127;
        if (c[u].blk >= 0) {
          if (pool.bf16) {
            const uint4* src = reinterpret_cast<const uint4*>(pool.data + (c[u].prow * D + 16 * l) * 2);
            x[u][0] = src[0];
            x[u][1] = src[1];
          } else {
            x[u][0] = *reinterpret_cast<const uint4*>(pool.data + c[u].prow * D + 16 * l);
            if (pool.scales) sc[u] = pool.scales[c[u].prow];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kRowsInFlight; ++u) {
        if (c[u].blk != -2 && c[u].blk < 0) continue;  // -2: the token cannot be found, zeros
        uint4 o[2] = {x[u][0], x[u][1]};
        if (!pool.bf16) {
          uint4 h[2];
          e4m3x16_to_f16(x[u][0], h[0], h[1]);
          const float s = __uint_as_float(sc[u] << 23);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t hw[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hw[j]));
              w[j] = pack_bf16x2(f.x * s, f.y * s);  // four significant bits: exact
            }
            o[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        uint4* dst = reinterpret_cast<uint4*>(const_cast<__nv_bfloat16*>(packed_row(p, t0 + c[u].tok, c[u].which)) + 16 * l);
        dst[0] = o[0];
        dst[1] = o[1];
      }
    }
  }
}

}  // namespace pcp
