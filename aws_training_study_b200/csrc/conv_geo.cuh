// The converter warps' mapping from raw e4m3 items to the 128B-swizzled f16
// operand layout, shared by attn_kv.cuh and chunk_tiles.cuh.
#pragma once

#include <cstdint>

namespace pcp {

// Where converter thread ct moves its chunks of one item.  A K half is 64
// raw rows of D bytes, a V half 128 raw rows of D/2 bytes: 4 x `boxes`
// 16-byte chunks per row, stored as `boxes` 128B-swizzled f16 boxes of 64
// columns.  The 16 quarter-warps (8 threads: one 128-bit shared-memory
// wavefront) take tasks (row pair, box): rows 2p and 2p+1 get four
// consecutive chunks each, of boxes b and b ^ 1, so the raw loads (16-byte
// bank group = row * cpr + chunk, mod 8) and the swizzled stores (group =
// (2 * (chunk % 4) [+1]) ^ (row & 7)) both hit 8 distinct groups.  Task
// m of a thread is 32 / boxes rows below its task 0 (same chunk, same
// row & 7), so a thread's m-th chunk is 2048 m raw bytes and
// 4096 / boxes * m operand bytes past its first.
struct ConvGeo {
  uint32_t raw;   // raw byte offset of chunk 0
  uint32_t lo;    // operand byte offsets of its two f16 halves
  uint32_t hi;
  int row;        // row (key) of chunk 0
};

__device__ __forceinline__ ConvGeo conv_geo(int ct, int boxes, uint32_t box_bytes) {
  const int j = ct & 7, q = ct >> 3;
  const int row = 2 * (q / boxes) + (j >> 2);
  const int cbox = boxes > 1 ? ((q % boxes) ^ (j >> 2)) : 0;
  const int c16 = 4 * cbox + (j & 3);
  const int ch = (j & 3) * 2;
  const uint32_t rowp = cbox * box_bytes + row * 128;
  return {static_cast<uint32_t>((row * 4 * boxes + c16) * 16), rowp + ((ch ^ (row & 7)) << 4),
          rowp + (((ch + 1) ^ (row & 7)) << 4), row};
}

}  // namespace pcp
