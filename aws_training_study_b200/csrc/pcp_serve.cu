// Host side of the C ABI declared in include/pcp_serve.h: argument checks and
// launches of the serving operators.
#include "pcp_serve.h"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <mutex>

#include "chunk_plan.cuh"
#include "chunk_rows.cuh"
#include "chunk_tiles.cuh"
#include "host_util.h"
#include "serve_ops.cuh"

namespace {

using pcp::fail;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int elt_bytes(int32_t dtype) { return dtype == PCP_F32 ? 4 : 2; }

// A packed tensor whose rows a kernel reads or writes 16 bytes at a time.
int check_heads(const pcp_heads_t* h, int32_t heads, int32_t rows, int elt, const char* name) {
  if (!h) return fail(PCP_ERR_INVALID_ARGUMENT, "%s is NULL", name);
  if (h->heads != heads) return fail(PCP_ERR_INVALID_ARGUMENT, "%s has %d heads, expected %d", name, h->heads, heads);
  if (rows == 0 || heads == 0) return PCP_OK;
  if (!h->data) return fail(PCP_ERR_INVALID_ARGUMENT, "%s has a NULL buffer", name);
  if (reinterpret_cast<uintptr_t>(h->data) % 16 || h->head_stride * elt % 16 || h->row_stride * elt % 16)
    return fail(PCP_ERR_INVALID_ARGUMENT, "%s: every row must be 16-byte aligned (strides %lld, %lld elements)", name,
                static_cast<long long>(h->head_stride), static_cast<long long>(h->row_stride));
  return PCP_OK;
}

int check_pool(const pcp_pool_t* p) {
  if (!p) return fail(PCP_ERR_INVALID_ARGUMENT, "pool is NULL");
  if (p->head_dim != 128 && p->head_dim != 256)
    return fail(PCP_ERR_UNSUPPORTED, "head_dim %d unsupported by the paged cache (128 or 256)", p->head_dim);
  if (p->num_kv_heads <= 0 || p->num_kv_heads > 1024)
    return fail(PCP_ERR_UNSUPPORTED, "num_kv_heads %d must be positive and at most 1024", p->num_kv_heads);
  if (p->block_size <= 0 || p->block_size % 16)
    return fail(PCP_ERR_UNSUPPORTED, "block_size %d must be a multiple of 16", p->block_size);
  if (p->kv_dtype != PCP_KV_E4M3 && p->kv_dtype != PCP_KV_BF16)
    return fail(PCP_ERR_INVALID_ARGUMENT, "kv_dtype %d unknown", p->kv_dtype);
  if (p->scales && p->kv_dtype != PCP_KV_E4M3) return fail(PCP_ERR_INVALID_ARGUMENT, "scales need an e4m3 cache");
  if (p->blocks <= 0 || p->blocks > INT_MAX) return fail(PCP_ERR_INVALID_ARGUMENT, "pool of %lld blocks",
                                                         static_cast<long long>(p->blocks));
  if (!p->data || reinterpret_cast<uintptr_t>(p->data) % 16 || reinterpret_cast<uintptr_t>(p->scales) % 16)
    return fail(PCP_ERR_INVALID_ARGUMENT, "the pool and its scales must be 16-byte aligned device memory");
  return PCP_OK;
}

int check_batch(const pcp_batch_t* b) {
  if (!b) return fail(PCP_ERR_INVALID_ARGUMENT, "batch is NULL");
  if (b->num_seqs < 0 || b->rows < 0 || b->table_width < 0)
    return fail(PCP_ERR_INVALID_ARGUMENT, "negative number of sequences, rows or table entries");
  if (b->num_seqs > 0 && (!b->offsets || !b->kv_len || (b->table_width > 0 && !b->block_tables)))
    return fail(PCP_ERR_INVALID_ARGUMENT, "offsets, kv_len or block_tables is NULL");
  if (b->table_stride < 0) return fail(PCP_ERR_INVALID_ARGUMENT, "table_stride must not be negative");
  return PCP_OK;
}

pcp::BatchView batch_view(const pcp_batch_t& b) {
  return {b.offsets, b.kv_len, b.block_tables, b.table_stride, b.table_width, b.num_seqs, b.rows};
}

pcp::PoolView pool_view(const pcp_pool_t& p) {
  return {static_cast<uint8_t*>(p.data), p.scales, p.blocks, p.num_kv_heads, p.head_dim, p.block_size,
          p.kv_dtype == PCP_KV_BF16};
}

int cache_rows(const pcp_pool_t* pool, const pcp_batch_t* batch, const pcp_heads_t* k, const pcp_heads_t* v,
               int32_t* device_status, void* stream, bool append) {
  PCP_TRY(check_pool(pool));
  PCP_TRY(check_batch(batch));
  PCP_TRY(check_heads(k, pool->num_kv_heads, batch->rows, 2, "k"));
  PCP_TRY(check_heads(v, pool->num_kv_heads, batch->rows, 2, "v"));
  if (!device_status) return fail(PCP_ERR_INVALID_ARGUMENT, "device_status is NULL");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (batch->num_seqs == 0 || batch->rows == 0) return PCP_OK;
  pcp::CacheRowsParams p{};
  p.pool = pool_view(*pool);
  p.batch = batch_view(*batch);
  p.k = k->data;
  p.v = v->data;
  p.k_head = k->head_stride;
  p.k_row = k->row_stride;
  p.v_head = v->head_stride;
  p.v_row = v->row_stride;
  p.err = device_status;
  // Tokens a warp: as many as leave 16 warps an SM, so that few tokens spread
  // over the GPU and many share the search for their sequence.
  int tpw = 32;
  while (tpw > 1 && ceil_div(batch->rows, tpw) < 148 * 16) tpw /= 2;
  p.tokens_per_warp = tpw;
  const uint64_t per_token = 2 * static_cast<uint64_t>(pool->num_kv_heads);
  p.inv_per_token = static_cast<unsigned>(((uint64_t(1) << 32) + per_token - 1) / per_token);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(ceil_div(batch->rows, tpw), 8), 148 * 8));
  if (append) {
    if (pool->head_dim == 256) pcp::cache_append_kernel<256><<<grid, 256, 0, st>>>(p);
    else pcp::cache_append_kernel<128><<<grid, 256, 0, st>>>(p);
  } else {
    if (pool->head_dim == 256) pcp::cache_read_kernel<256><<<grid, 256, 0, st>>>(p);
    else pcp::cache_read_kernel<128><<<grid, 256, 0, st>>>(p);
  }
  CUDA_TRY(cudaGetLastError());
  return PCP_OK;
}

// ------------------------------------------------------- chunk attention --
// Grids: one CTA, or half a CTA pair, per SM.  No CTA waits for another, so
// fewer SMs only queue them.
constexpr int kCtas = 148;
constexpr int kPairs = kCtas / 2;

size_t align_up(size_t a) { return (a + 255) / 256 * 256; }

struct ChunkLayout {
  size_t small_rec, tile_rec, small_o, small_lse, tile_o, tile_lse, copy, bytes;
  bool expand;  // tile units read a bf16 copy of their e4m3 pages
};

// An e4m3 cache is expanded for the tile units from kExpandRows rows a KV head
// on (4 tiles), while the copy of all sequences' tables stays within kExpandBytes.
// In place / expanded, us, of a cache with scales: heads of 256 over 32768 tokens, 512
// rows 92 / 81, 1024 122 / 99, 2048 188 / 135, 8192 588 / 360; over 131072, 512 226 /
// 236, 1024 345 / 298, 2048 662 / 481, 8192 2230 / 1365; heads of 128 over 32768, 512
// 271 / 150, 1024 388 / 194, 4096 1342 / 528.  At unit scale (no scales to apply in
// place): heads of 256 over 32768, 512 74 / 81, 1024 91 / 97, 2048 128 / 131, 8192 362
// / 360; over 131072, 512 167 / 222, 1024 223 / 300, 2048 422 / 497, 8192 1521 / 1485;
// heads of 128 over 32768, 512 132 / 147, 1024 186 / 191, 4096 588 / 517: there the
// copy pays from some 8192 rows (heads of 256) or 4096 (128) only, and costs up to a
// third between.
constexpr int64_t kExpandRows = 1024;
constexpr int64_t kExpandBytes = int64_t(1) << 30;

bool has_tiles(int32_t max_chunk, int32_t group) { return static_cast<int64_t>(max_chunk) * group > pcp::kSmallRows; }

// Rows of a sequence in the copy: what its table holds, in whole key tiles.
int copy_rows(int32_t block_size, int32_t table_width) {
  return static_cast<int>(ceil_div(static_cast<int64_t>(block_size) * table_width, 128) * 128);
}

ChunkLayout chunk_layout(const pcp_pool_t& pool, int32_t group, int32_t seqs, int32_t table_width, int32_t max_chunk) {
  ChunkLayout w{};
  const int32_t head_dim = pool.head_dim;
  const bool tiles = has_tiles(max_chunk, group);
  size_t at = 0;
  auto put = [&](size_t bytes) {
    const size_t here = at;
    at = align_up(at + bytes);
    return here;
  };
  w.small_rec = put(kCtas * sizeof(pcp::ChunkRecord));
  w.tile_rec = put(tiles ? 2 * kPairs * sizeof(pcp::ChunkRecord) : 0);
  w.small_o = put(size_t(2) * kCtas * pcp::kSmallRows * head_dim * 4);
  w.small_lse = put(size_t(2) * kCtas * pcp::kSmallRows * 4);
  w.tile_o = put(tiles ? size_t(2) * kPairs * pcp::kUnitRows * head_dim * 4 : 0);
  w.tile_lse = put(tiles ? size_t(2) * kPairs * pcp::kUnitRows * 4 : 0);
  const int64_t row = int64_t(2) * pool.num_kv_heads * head_dim * 2 * seqs;  // of every sequence
  w.expand = tiles && pool.kv_dtype == PCP_KV_E4M3 && static_cast<int64_t>(max_chunk) * group >= kExpandRows &&
             table_width > 0 && row > 0 &&
             static_cast<int64_t>(table_width) * pool.block_size <= kExpandBytes / row - 128;
  w.copy = put(w.expand ? static_cast<size_t>(row * copy_rows(pool.block_size, table_width)) : 0);
  w.bytes = at;
  return w;
}

int check_chunk(const pcp_pool_t* pool, int32_t q_heads, int32_t seqs, int32_t rows, int32_t max_chunk) {
  PCP_TRY(check_pool(pool));
  if (q_heads <= 0 || q_heads % pool->num_kv_heads)
    return fail(PCP_ERR_INVALID_ARGUMENT, "%d query heads must be a positive multiple of %d KV heads", q_heads,
                pool->num_kv_heads);
  if (seqs < 0 || rows < 0 || max_chunk <= 0)
    return fail(PCP_ERR_INVALID_ARGUMENT, "negative number of sequences or rows, or max_chunk not positive");
  const int64_t group = q_heads / pool->num_kv_heads;
  if (static_cast<int64_t>(rows) * group > INT_MAX - pcp::kUnitRows)
    return fail(PCP_ERR_UNSUPPORTED, "%d rows of %lld query heads a KV head are too many", rows,
                static_cast<long long>(group));
  return PCP_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

int encode(CUtensorMap* tm, CUtensorMapDataType type, int rank, void* base, const cuuint64_t* dims,
           const cuuint64_t* strides, const cuuint32_t* box, bool swizzle) {
  auto fn = encode_fn();
  if (!fn) return fail(PCP_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the CUDA driver");
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(tm, type, rank, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(PCP_ERR_CUDA, "cuTensorMapEncodeTiled (cache pool) failed (%d)", static_cast<int>(r));
  return PCP_OK;
}

// e4m3 cache blocks [blocks][2][Hkv][bs][D] as a 5-D tensor {D, bs, Hkv, K/V,
// blocks}; boxes of box_x bytes x box_rows rows of one head of K or V of one
// block, not swizzled.
int make_pool_map(CUtensorMap* tm, const pcp_pool_t& p, uint32_t box_x, uint32_t box_rows) {
  const uint64_t D = p.head_dim, bs = p.block_size, H = p.num_kv_heads;
  const cuuint64_t dims[5] = {D, bs, H, 2, static_cast<cuuint64_t>(p.blocks)};
  const cuuint64_t strides[4] = {D, bs * D, H * bs * D, 2 * H * bs * D};
  const cuuint32_t box[5] = {box_x, box_rows, 1, 1, 1};
  return encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, p.data, dims, strides, box, false);
}

// Cache blocks as {128 bytes, bs, 128-byte columns, Hkv, 2 * blocks}: a box is
// box_cols columns of box_rows rows of one head, of K or V or (box_kv 2) both,
// each column in the 128-byte swizzle.
int make_rows_map(CUtensorMap* tm, const pcp_pool_t& p, uint32_t box_rows, uint32_t box_cols, uint32_t box_kv) {
  const bool bf16 = p.kv_dtype == PCP_KV_BF16;
  const uint64_t bs = p.block_size, H = p.num_kv_heads, elt = bf16 ? 2 : 1, row = p.head_dim * elt;
  const uint32_t cols = static_cast<uint32_t>(row / 128);
  const cuuint64_t dims[5] = {128 / elt, bs, cols, H, 2 * static_cast<cuuint64_t>(p.blocks)};
  const cuuint64_t strides[4] = {row, 128, bs * row, H * bs * row};
  const cuuint32_t box[5] = {static_cast<cuuint32_t>(128 / elt), box_rows, box_cols, 1, box_kv};
  return encode(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, p.data, dims, strides,
                box, true);
}

// Q as {64 elements, query heads of a KV head, rows, 64-element columns, KV
// heads}: a box is the 128 rows (row * group + head) of a CTA, two columns, each
// in the 128-byte swizzle.
int make_q_map(CUtensorMap* tm, const pcp::ChunkParams& p, int D) {
  const uint64_t G = p.group, head = static_cast<uint64_t>(p.q_head) * 2, row = static_cast<uint64_t>(p.q_row) * 2;
  // (The stride of an axis of one is 0 here; any multiple of 16 does.)
  const cuuint64_t dims[5] = {64, G, static_cast<cuuint64_t>(p.batch.rows), static_cast<cuuint64_t>(D / 64),
                              static_cast<cuuint64_t>(p.pool.heads)};
  const cuuint64_t strides[4] = {std::max<uint64_t>(head, 16), std::max<uint64_t>(row, 16), 128,
                                 std::max<uint64_t>(G * head, 16)};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(128 / G), 2, 1};
  return encode(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<__nv_bfloat16*>(p.q), dims, strides, box, true);
}

// Scale bytes [blocks][2][Hkv][bs] as {bs, Hkv, 2 * blocks}: boxes of box_rows
// of K and of V of one head.
int make_scale_map(CUtensorMap* tm, const pcp_pool_t& p, uint32_t box_rows) {
  const uint64_t bs = p.block_size, H = p.num_kv_heads;
  const cuuint64_t dims[3] = {bs, H, 2 * static_cast<cuuint64_t>(p.blocks)};
  const cuuint64_t strides[2] = {bs, H * bs};
  const cuuint32_t box[3] = {box_rows, 1, 2};
  return encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p.scales, dims, strides, box, false);
}

// A kernel's dynamic shared memory is allowed once per device.
// Its compiled register count is checked there too where the kernel's register
// split (setmaxnreg) assumes one: with another the split would wait forever.
template <auto kKernel>
int allow_smem(int bytes, int regs = 0) {
  static std::mutex mutex;
  static bool done[64] = {};
  int device = 0;
  CUDA_TRY(cudaGetDevice(&device));
  std::lock_guard<std::mutex> lock(mutex);
  if (device < 64 && done[device]) return PCP_OK;
  if (regs) {
    cudaFuncAttributes a{};
    CUDA_TRY(cudaFuncGetAttributes(&a, kKernel));
    if (a.numRegs != regs) return fail(PCP_ERR_UNSUPPORTED, "kernel compiled to %d registers, %d assumed", a.numRegs, regs);
  }
  CUDA_TRY(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (device < 64) done[device] = true;
  return PCP_OK;
}

// A kernel whose blocks may be placed while the one before it ends; it waits for
// that one itself where it needs its results, and at the latest at its own end, so
// that whoever waits for it has waited for both.
template <typename... Args>
int launch_behind(void (*kernel)(Args...), unsigned grid, unsigned threads, size_t smem, cudaStream_t st,
                  const Args&... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = st;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  CUDA_TRY(cudaLaunchKernelEx(&config, kernel, args...));
  return PCP_OK;
}

template <int D, int kCache>
int launch_rows(const pcp_pool_t& pool, const pcp::ChunkParams& p, cudaStream_t st) {
  constexpr bool kFp8 = kCache != pcp::kCacheBf16;
  using L = pcp::RowsSmem<D, kFp8>;
  // Rows of a copy: as many as a page's length and a stage share.
  int shift = 4;
  while ((2 << shift) <= L::kStageKeys && pool.block_size % (2 << shift) == 0) ++shift;
  CUtensorMap tm, ts{};
  PCP_TRY(make_rows_map(&tm, pool, 1 << shift, L::kBoxes, 2));
  if (kCache == pcp::kCacheScaled) PCP_TRY(make_scale_map(&ts, pool, 1 << shift));
  PCP_TRY((allow_smem<pcp::chunk_rows_kernel<D, kCache>>(L::kBytes, kFp8 ? pcp::kRowsLaunchRegs : 0)));
  pcp::chunk_rows_kernel<D, kCache><<<kCtas, L::kThreads, L::kBytes, st>>>(tm, ts, shift, p);
  CUDA_TRY(cudaGetLastError());
  return PCP_OK;
}

template <int D, int kCache>
int launch_tiles(const pcp_pool_t& pool, const pcp::ChunkParams& p, cudaStream_t st) {
  using L = pcp::TilesSmem<D, kCache>;
  // Copies of as many rows as a page's length and a tile (K: half a tile) share.
  pcp::TileBoxes box{0, 64, 128, 0};
  while (pool.block_size % box.k_rows) box.k_rows /= 2;
  while (pool.block_size % box.v_rows) box.v_rows /= 2;
  box.all_cols = !L::kFp8 && box.k_rows == 64;
  CUtensorMap tq{}, tk, tv;
  // (Heads or rows that are all the same one, stride 0, have no such map.)
  box.q_copy = !L::kFp8 && 128 % p.group == 0 && (p.q_head > 0 || p.group * p.pool.heads == 1) &&
               (p.q_row > 0 || p.batch.rows == 1);
  if (box.q_copy) PCP_TRY(make_q_map(&tq, p, D));
  if (L::kFp8) {
    PCP_TRY(make_pool_map(&tk, pool, D, box.k_rows));
    PCP_TRY(make_pool_map(&tv, pool, D / 2, box.v_rows));
  } else {
    PCP_TRY(make_rows_map(&tk, pool, box.k_rows, box.all_cols ? D / 64 : 1, 1));
    PCP_TRY(make_rows_map(&tv, pool, box.v_rows, box.all_cols ? D / 128 : 1, 1));
  }
  PCP_TRY((allow_smem<pcp::chunk_tiles_kernel<D, kCache>>(L::kBytes, pcp::kTilesLaunchRegs)));
  return launch_behind(pcp::chunk_tiles_kernel<D, kCache>, 2 * kPairs, pcp::kTilesThreads, L::kBytes, st, tq, tk, tv,
                       box, p);
}

// Tile units over the bf16 copy of their pages.
template <int D>
int launch_expanded(const pcp_pool_t& pool, const pcp::ChunkParams& p, void* copy, cudaStream_t st) {
  const int rows = copy_rows(pool.block_size, p.batch.table_width);
  const int item_rows = pool.block_size % 64 ? 16 : 64;
  const pcp::ExpandParams e{p, static_cast<__nv_bfloat16*>(copy), rows, item_rows};
  const int64_t items = static_cast<int64_t>(p.batch.seqs) * p.batch.table_width * 2 * pool.num_kv_heads *
                        (pool.block_size / item_rows);
  PCP_TRY(launch_behind(pcp::chunk_expand_kernel<D>, static_cast<unsigned>(std::min<int64_t>(items, 8 * kCtas)), 256, 0,
                        st, e));
  // The copy as a cache of one page a sequence.
  pcp_pool_t dense = pool;
  dense.data = copy;
  dense.scales = nullptr;
  dense.blocks = p.batch.seqs;
  dense.block_size = rows;
  dense.kv_dtype = PCP_KV_BF16;
  pcp::ChunkParams d = p;
  d.pool = pool_view(dense);
  if (pool.scales) {
    d.scale_log2 = std::ldexp(p.scale_log2, pcp::kCopyShift);
    d.v_factor = std::ldexp(1.f, pcp::kCopyShift);
  }
  d.batch.tables = nullptr;
  d.batch.table_width = 1;
  return launch_tiles<D, pcp::kCacheBf16>(dense, d, st);
}

template <int D>
int launch_chunk(const pcp_pool_t& pool, const pcp::ChunkParams& p, void* copy, cudaStream_t st) {
  const bool bf16 = pool.kv_dtype == PCP_KV_BF16;
  if (bf16) PCP_TRY((launch_rows<D, pcp::kCacheBf16>(pool, p, st)));
  else if (pool.scales) PCP_TRY((launch_rows<D, pcp::kCacheScaled>(pool, p, st)));
  else PCP_TRY((launch_rows<D, pcp::kCacheE4m3>(pool, p, st)));
  if (p.tile_pairs) {
    if (copy) PCP_TRY(launch_expanded<D>(pool, p, copy, st));
    else if (bf16) PCP_TRY((launch_tiles<D, pcp::kCacheBf16>(pool, p, st)));
    else if (pool.scales) PCP_TRY((launch_tiles<D, pcp::kCacheScaled>(pool, p, st)));
    else PCP_TRY((launch_tiles<D, pcp::kCacheE4m3>(pool, p, st)));
  }
  return launch_behind(pcp::chunk_combine_kernel<D>, p.small_ctas * p.small_y + p.tile_pairs * (p.tile_y + 1), 256, 0, st, p);
}

}  // namespace

extern "C" {

int pcp_qk_norm_rope(int32_t dtype, int32_t rows, int32_t head_dim, int32_t rotary_dim, int32_t layout,
                     const pcp_heads_t* q, const pcp_heads_t* k, const pcp_heads_t* q_out, const pcp_heads_t* k_out,
                     const void* positions, int32_t positions_64, const uint64_t* turns, float magnitude,
                     const void* q_weight, const void* k_weight, float eps, void* stream) {
  if (dtype != PCP_F32 && dtype != PCP_F16 && dtype != PCP_BF16)
    return fail(PCP_ERR_INVALID_ARGUMENT, "dtype %d unknown", dtype);
  if (rows < 0) return fail(PCP_ERR_INVALID_ARGUMENT, "negative number of rows");
  if (head_dim <= 0 || head_dim % 16 || head_dim > 512)
    return fail(PCP_ERR_UNSUPPORTED, "head_dim %d must be a multiple of 16 up to 512", head_dim);
  if (rotary_dim < 0 || rotary_dim % 16 || rotary_dim > head_dim)
    return fail(PCP_ERR_UNSUPPORTED, "rotary_dim %d must be a multiple of 16 up to head_dim %d", rotary_dim, head_dim);
  if (layout != PCP_ROTARY_HALF && layout != PCP_ROTARY_INTERLEAVED)
    return fail(PCP_ERR_INVALID_ARGUMENT, "rotary layout %d unknown", layout);
  if (!q || !k || q->heads < 0 || k->heads < 0) return fail(PCP_ERR_INVALID_ARGUMENT, "q or k missing");
  const int elt = elt_bytes(dtype);
  PCP_TRY(check_heads(q, q->heads, rows, elt, "q"));
  PCP_TRY(check_heads(k, k->heads, rows, elt, "k"));
  PCP_TRY(check_heads(q_out, q->heads, rows, elt, "q_out"));
  PCP_TRY(check_heads(k_out, k->heads, rows, elt, "k_out"));
  if (rows == 0 || q->heads + k->heads == 0) return PCP_OK;
  if (rotary_dim > 0 && (!positions || !turns)) return fail(PCP_ERR_INVALID_ARGUMENT, "positions or turns is NULL");
  if (reinterpret_cast<uintptr_t>(q_weight) % 16 || reinterpret_cast<uintptr_t>(k_weight) % 16)
    return fail(PCP_ERR_INVALID_ARGUMENT, "weights must be 16-byte aligned");
  pcp::NormRopeParams p{};
  p.q = {q->data, q_out->data, q->head_stride, q->row_stride, q_out->head_stride, q_out->row_stride, q->heads, q_weight};
  p.k = {k->data, k_out->data, k->head_stride, k->row_stride, k_out->head_stride, k_out->row_stride, k->heads, k_weight};
  p.rows = rows;
  p.head_dim = head_dim;
  p.rotary_dim = rotary_dim;
  p.lanes = 1;
  while (p.lanes * 16 < head_dim) p.lanes *= 2;
  const int per_pass = 32 / p.lanes;
  p.passes_q = static_cast<int>(ceil_div(q->heads, per_pass));
  p.passes = p.passes_q + static_cast<int>(ceil_div(k->heads, per_pass));
  // Passes a warp: the split of a row that takes the fewest rounds of the 16
  // warps an SM holds, where a warp's start (its angles, its first loads) costs
  // about four passes.
  int64_t best = INT64_MAX;
  for (int parts = 1; parts <= p.passes; ++parts) {
    const int per = static_cast<int>(ceil_div(p.passes, parts));
    const int64_t cost = ceil_div(rows * ceil_div(p.passes, per), 148 * 16) * (per + 4);
    if (cost < best) best = cost, p.per_warp = per;
  }
  p.positions = positions;
  p.positions_64 = positions_64;
  p.turns = reinterpret_cast<const unsigned long long*>(turns);
  p.magnitude = magnitude;
  p.eps = eps;
  const int64_t warps = rows * ceil_div(p.passes, p.per_warp);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(warps, 8), 148 * 16));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(p); };
  const bool inter = layout == PCP_ROTARY_INTERLEAVED;
  if (dtype == PCP_F32) launch(inter ? pcp::qk_norm_rope_kernel<float, true> : pcp::qk_norm_rope_kernel<float, false>);
  else if (dtype == PCP_F16) launch(inter ? pcp::qk_norm_rope_kernel<__half, true> : pcp::qk_norm_rope_kernel<__half, false>);
  else launch(inter ? pcp::qk_norm_rope_kernel<__nv_bfloat16, true> : pcp::qk_norm_rope_kernel<__nv_bfloat16, false>);
  CUDA_TRY(cudaGetLastError());
  return PCP_OK;
}

int pcp_cache_append(const pcp_pool_t* pool, const pcp_batch_t* batch, const pcp_heads_t* k, const pcp_heads_t* v,
                     int32_t* device_status, void* stream) {
  return cache_rows(pool, batch, k, v, device_status, stream, true);
}

int pcp_cache_read(const pcp_pool_t* pool, const pcp_batch_t* batch, const pcp_heads_t* k_out,
                   const pcp_heads_t* v_out, int32_t* device_status, void* stream) {
  return cache_rows(pool, batch, k_out, v_out, device_status, stream, false);
}

int pcp_chunk_attention_workspace_size(const pcp_pool_t* pool, int32_t num_q_heads, int32_t num_seqs, int32_t rows,
                                       int32_t table_width, int32_t max_chunk, size_t* bytes) {
  PCP_TRY(check_chunk(pool, num_q_heads, num_seqs, rows, max_chunk));
  if (!bytes) return fail(PCP_ERR_INVALID_ARGUMENT, "bytes is NULL");
  *bytes = chunk_layout(*pool, num_q_heads / pool->num_kv_heads, num_seqs, std::max(table_width, 0), max_chunk).bytes;
  return PCP_OK;
}

int pcp_chunk_attention(const pcp_pool_t* pool, const pcp_batch_t* batch, const pcp_heads_t* q, const pcp_heads_t* out,
                        int32_t max_chunk, float softmax_scale, void* workspace, size_t workspace_bytes,
                        int32_t* device_status, void* stream) {
  PCP_TRY(check_batch(batch));
  if (!q) return fail(PCP_ERR_INVALID_ARGUMENT, "q is NULL");
  PCP_TRY(check_chunk(pool, q->heads, batch->num_seqs, batch->rows, max_chunk));
  PCP_TRY(check_heads(q, q->heads, batch->rows, 2, "q"));
  PCP_TRY(check_heads(out, q->heads, batch->rows, 2, "out"));
  if (!device_status) return fail(PCP_ERR_INVALID_ARGUMENT, "device_status is NULL");
  if (!(softmax_scale > 0) || std::isinf(softmax_scale))
    return fail(PCP_ERR_INVALID_ARGUMENT, "softmax_scale %g must be positive and finite", softmax_scale);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (batch->num_seqs == 0 || batch->rows == 0) return PCP_OK;
  const int32_t group = q->heads / pool->num_kv_heads;
  const ChunkLayout w = chunk_layout(*pool, group, batch->num_seqs, batch->table_width, max_chunk);
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < w.bytes)
    return fail(PCP_ERR_INVALID_ARGUMENT, "workspace of %zu bytes, aligned to 256, is needed (got %zu)", w.bytes,
                workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  pcp::ChunkParams p{};
  p.batch = batch_view(*batch);
  p.pool = pool_view(*pool);
  p.work.small_rec = reinterpret_cast<pcp::ChunkRecord*>(ws + w.small_rec);
  p.work.tile_rec = reinterpret_cast<pcp::ChunkRecord*>(ws + w.tile_rec);
  p.work.small_o = reinterpret_cast<float*>(ws + w.small_o);
  p.work.small_lse = reinterpret_cast<float*>(ws + w.small_lse);
  p.work.tile_o = reinterpret_cast<float*>(ws + w.tile_o);
  p.work.tile_lse = reinterpret_cast<float*>(ws + w.tile_lse);
  p.q = static_cast<const __nv_bfloat16*>(q->data);
  p.out = static_cast<__nv_bfloat16*>(out->data);
  p.q_head = q->head_stride;
  p.q_row = q->row_stride;
  p.out_head = out->head_stride;
  p.out_row = out->row_stride;
  p.group = group;
  p.capacity = static_cast<int64_t>(batch->table_width) * pool->block_size;
  p.max_chunk = max_chunk;
  p.scale_log2 = static_cast<float>(static_cast<double>(softmax_scale) * 1.4426950408889634);
  p.v_factor = 1.f;
  p.small_ctas = kCtas;
  p.tile_pairs = has_tiles(max_chunk, group) ? kPairs : 0;
  // Rows of the longest small and tile unit, over the rows a block merges.
  const int64_t longest = std::min<int64_t>(max_chunk, batch->rows) * group;
  p.small_y = static_cast<int>(ceil_div(std::min<int64_t>(longest, pcp::kSmallRows), 8 / pcp::kCombineSmallW));
  p.tile_y = static_cast<int>(ceil_div(std::min<int64_t>(longest, pcp::kUnitRows), 8 / pcp::kCombineTileW));
  p.status = device_status;
  // (A scale that the copy's power of two would take out of fp32: in place.)
  const bool fits = !pool->scales || !std::isinf(std::ldexp(p.scale_log2, pcp::kCopyShift));
  void* copy = w.expand && fits ? ws + w.copy : nullptr;
  return pool->head_dim == 256 ? launch_chunk<256>(*pool, p, copy, st) : launch_chunk<128>(*pool, p, copy, st);
}

int pcp_chunk_cut_parts(const int32_t* states, const int32_t* failed, int32_t ranges, int32_t range, int32_t* parts) {
  if (!states || !failed || !parts || ranges <= 0 || range < 0 || range >= ranges)
    return fail(PCP_ERR_INVALID_ARGUMENT, "bad arguments");
  *parts = pcp::cut_parts(range, ranges, failed[range] != 0, [&](int b, uint32_t& stop, uint32_t& end) {
    stop = end = 0;
    for (int i = 0; i < 32; ++i) {
      const int state = b + i < ranges && !failed[b + i] ? states[b + i] : 0;
      stop |= static_cast<uint32_t>(state != 1) << i;
      end |= static_cast<uint32_t>(state == 2) << i;
    }
  });
  return PCP_OK;
}

}  // extern "C"
