// Host side of the C ABI declared in include/pcp_serve.h: argument checks and
// launches of the serving operators.
#include "pcp_serve.h"

#include <algorithm>
#include <climits>

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
  if (p->num_kv_heads <= 0) return fail(PCP_ERR_INVALID_ARGUMENT, "num_kv_heads must be positive");
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
  CUDA_TRY(cudaMemsetAsync(device_status, 0, sizeof(int32_t), st));
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
  // Passes a warp: all of a row's when that leaves 32 warps an SM (its angles
  // are then made once), fewer while the GPU has idle warps.
  p.per_warp = p.passes;
  while (p.per_warp > 1 && rows * ceil_div(p.passes, p.per_warp) < 148 * 32) p.per_warp = (p.per_warp + 1) / 2;
  p.interleaved = layout == PCP_ROTARY_INTERLEAVED;
  p.positions = positions;
  p.positions_64 = positions_64;
  p.turns = reinterpret_cast<const unsigned long long*>(turns);
  p.magnitude = magnitude;
  p.eps = eps;
  const int64_t warps = rows * ceil_div(p.passes, p.per_warp);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(warps, 8), 148 * 16));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PCP_F32) pcp::qk_norm_rope_kernel<float><<<grid, 256, 0, st>>>(p);
  else if (dtype == PCP_F16) pcp::qk_norm_rope_kernel<__half><<<grid, 256, 0, st>>>(p);
  else pcp::qk_norm_rope_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
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

}  // extern "C"
