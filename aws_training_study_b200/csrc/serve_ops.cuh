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

// ------------------------------------------------------ pairs of fp32 values --
// Two fp32 values in a 64-bit register: sm_100 multiplies and adds both in one
// instruction, each rounded as the scalar form would.
typedef unsigned long long f32x2;

__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(f32x2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

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

template <typename T>
__device__ __forceinline__ void get_pairs(const Vec8<T>& v, f32x2* f) {
  float x[8];
  v.get(x);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = pair(x[2 * i], x[2 * i + 1]);
}

template <typename T>
__device__ __forceinline__ void store_pairs(void* p, const f32x2* f) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(f[i], x[2 * i], x[2 * i + 1]);
  Vec8<T>::store(p, x);
}

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
  const void* positions;
  int positions_64;
  const unsigned long long* turns;  // turns per position of each pair, as a 64-bit fraction
  float magnitude;
  float eps;
};

// sin and cos of 2 pi t / 2^64.  The nearest quarter turn comes off in integers
// (exactly), which leaves |x| <= pi / 4, where the Taylor series to x^9 and x^10
// are within 2e-9 of sine and cosine: below half a step of fp32, so that what
// is lost is x's rounding (pi / 4 * 2^-24) and the sums'.
__device__ __forceinline__ void sincos_turns(unsigned long long t, float& sn, float& cs) {
  const unsigned long long near = t + (1ull << 61);
  const unsigned quarter = static_cast<unsigned>(near >> 62);
  const int rest = static_cast<int>((t - (static_cast<unsigned long long>(quarter) << 62)) >> 32);
  const float x = static_cast<float>(rest) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float z = x * x;
  float s = fmaf(z, 2.7557319224e-6f, -1.9841269841e-4f);  // 1/9!, -1/7!
  s = fmaf(z, s, 8.3333333333e-3f);                        // 1/5!
  s = fmaf(z, s, -1.6666666667e-1f);                       // -1/3!
  s = fmaf(z * x, s, x);
  float c = fmaf(z, -2.7557319224e-7f, 2.4801587302e-5f);  // -1/10!, 1/8!
  c = fmaf(z, c, -1.3888888889e-3f);                       // -1/6!
  c = fmaf(z, c, 4.1666666667e-2f);                        // 1/4!
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.f);
  const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
  sn = quarter & 2 ? -a : a;
  cs = (quarter + 1) & 2 ? -b : b;
}

// A warp takes one row (token) and some of its heads, 16 elements of a head a
// lane: the mean of squares is one shuffle reduction, and a rotated pair's two
// halves sit in one lane -- half layout: eight elements at 8 l and the eight at
// 8 l + rotary_dim / 2; interleaved: sixteen in a row -- so nothing else moves
// between lanes.  cos and sin are made once per row and lane, from the position
// times the pair's turns in 64-bit integers (whole turns overflow away, so
// there is no table to read and no error that grows with the position), and
// used for every head of the warp.  HBM's share is one read and one write of
// each element; instructions are near it (the first version issued 322 a pass
// of 1 KB and reached half of HBM's rate), hence two values an instruction and
// pointers that step.  The next kUnroll passes' loads are in flight over the work
// on kUnroll.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(256, 2) qk_norm_rope_kernel(const NormRopeParams p) {
  constexpr int kUnroll = sizeof(T) == 4 ? 1 : 2;
  const int lane = threadIdx.x & 31;
  const int parts = (p.passes + p.per_warp - 1) / p.per_warp;
  const long long items = static_cast<long long>(p.rows) * parts;
  const int l = lane & (p.lanes - 1);
  const int sub = lane / p.lanes;       // which of the pass's heads
  const int per_pass = 32 / p.lanes;
  const bool live_lane = 16 * l < p.head_dim;
  const int half = p.rotary_dim / 2;
  // First elements of this lane's two runs of eight, and whether they turn.
  const bool turned = 16 * l < p.rotary_dim;
  int e0 = 16 * l, e1 = 16 * l + 8;
  if (turned && !kInterleaved) e0 = 8 * l, e1 = 8 * l + half;
  const float inv_d = 1.f / static_cast<float>(p.head_dim);

  for (long long item = blockIdx.x * 8LL + (threadIdx.x >> 5); item < items; item += gridDim.x * 8LL) {
    const int row = static_cast<int>(item / parts);
    const int p0 = static_cast<int>(item - static_cast<long long>(row) * parts) * p.per_warp;
    const int p1 = min(p0 + p.per_warp, p.passes);
    // The rotation as factors of pairs of values: half layout, (cos, cos') and
    // (sin, sin') of two neighbouring pairs; interleaved, (cos, cos) and
    // (-sin, sin) of one.
    constexpr int kPairs = kInterleaved ? 8 : 4;
    f32x2 co[kPairs], si[kPairs];
    bool have_angles = false;
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {  // q's passes, then k's
      const HeadRows& h = part ? p.k : p.q;
      const int base = part ? p.passes_q : 0;
      int a = max(p0, base) - base;
      const int b = (part ? p1 : min(p1, p.passes_q)) - base;
      if (a >= b) continue;
      const int heads = h.heads;
      const long long in_step = per_pass * h.in_head, out_step = per_pass * h.out_head;
      const T* in = static_cast<const T*>(h.in) + row * h.in_row + (a * per_pass + sub) * h.in_head;
      T* out = static_cast<T*>(h.out) + row * h.out_row + (a * per_pass + sub) * h.out_head;
      const bool norm = h.weight != nullptr;
      f32x2 w[8];
      if (norm && live_lane) {
        Vec8<T> x, y;
        x.load(static_cast<const T*>(h.weight) + e0);
        y.load(static_cast<const T*>(h.weight) + e1);
        get_pairs(x, w);
        get_pairs(y, w + 4);
      }
      Vec8<T> n0[kUnroll], n1[kUnroll];  // the next passes' loads, in flight over this one's work
      auto load = [&](int at, const T* from) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (live_lane && at + u < b && (at + u) * per_pass + sub < heads) {
            n0[u].load(from + u * in_step + e0);
            n1[u].load(from + u * in_step + e1);
          }
      };
      load(a, in);
#pragma unroll 1
      for (; a < b; a += kUnroll) {
        Vec8<T> x0[kUnroll], x1[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) x0[u] = n0[u], x1[u] = n1[u];
        in += kUnroll * in_step;
        load(a + kUnroll, in);
        if (!have_angles && p.rotary_dim) {  // behind the first loads
          have_angles = true;
          if (turned) {
            const long long pos = p.positions_64 ? static_cast<const long long*>(p.positions)[row]
                                                 : static_cast<const int*>(p.positions)[row];
            float c[8], s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              sincos_turns(static_cast<unsigned long long>(pos) * p.turns[8 * l + i], s[i], c[i]);
              s[i] *= p.magnitude;
              c[i] *= p.magnitude;
            }
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
              co[i] = kInterleaved ? pair(c[i], c[i]) : pair(c[(2 * i) & 7], c[(2 * i + 1) & 7]);
              si[i] = kInterleaved ? pair(-s[i], s[i]) : pair(s[(2 * i) & 7], s[(2 * i + 1) & 7]);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (a + u >= b) break;  // the same for the whole warp
          const bool live = live_lane && (a + u) * per_pass + sub < heads;
          f32x2 f[8];
          if (live) {
            get_pairs(x0[u], f);
            get_pairs(x1[u], f + 4);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = 0;
          }
          if (norm) {
            f32x2 sq = mul2(f[0], f[0]), sr = mul2(f[1], f[1]);
#pragma unroll
            for (int i = 2; i < 8; i += 2) {
              sq = fma2(f[i], f[i], sq);
              sr = fma2(f[i + 1], f[i + 1], sr);
            }
            float s0, s1, s2, s3;
            split(sq, s0, s1);
            split(sr, s2, s3);
            float ss = (s0 + s1) + (s2 + s3);
            for (int o = p.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = rsqrtf(fmaf(ss, inv_d, p.eps));
            const f32x2 rr = pair(r, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = mul2(mul2(f[i], rr), w[i]);
          }
          if (turned) {
            if (kInterleaved) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float x, y;
                split(f[i], x, y);
                f[i] = fma2(f[i], co[i], mul2(pair(y, x), si[i]));
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const f32x2 x = f[i], y = f[4 + i];
                f[4 + i] = fma2(y, co[i & (kPairs - 1)], mul2(x, si[i & (kPairs - 1)]));
                const f32x2 ys = mul2(y, si[i & (kPairs - 1)]);
                f[i] = fma2(x, co[i & (kPairs - 1)], ys ^ 0x8000000080000000ull);
              }
            }
          }
          if (live) {
            store_pairs<T>(out + u * out_step + e0, f);
            store_pairs<T>(out + u * out_step + e1, f + 4);
          }
        }
        out += kUnroll * out_step;
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

// 16 codes times a power of two as bf16: four significant bits, so exact.
__device__ __forceinline__ void e4m3x16_to_bf16(const uint4& codes, float s, uint4* out) {
  uint4 h[2];
  e4m3x16_to_f16(codes, h[0], h[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t hw[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hw[j]));
      w[j] = pack_bf16x2(f.x * s, f.y * s);
    }
    out[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
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
        if (!pool.bf16) e4m3x16_to_bf16(x[u][0], __uint_as_float(min(sc[u], 254u) << 23), o);
        uint4* dst = reinterpret_cast<uint4*>(const_cast<__nv_bfloat16*>(packed_row(p, t0 + c[u].tok, c[u].which)) + 16 * l);
        dst[0] = o[0];
        dst[1] = o[1];
      }
    }
  }
}

}  // namespace pcp
