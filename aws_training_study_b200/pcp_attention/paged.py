"""Paged KV cache on the device: the producer that writes new tokens into a
rank's block pool, and the history attention that reads a pool through block
tables.

The reference builds each rank's cache on the host: ``shard_history``
(``pcp_attention/layout.py:54-98``) stripes a global K/V over the ranks and
reshapes each shard to ``[blocks, Hkv, bs, D]``; ``pack_local_kv``
(``pcp_attention/kernel.py:17-29``) packs a block's K then V into the ring
payload; FP8 comes from ``tensor.to(torch.float8_e4m3fn)`` (``run_poc.py:81-134``).
Here the same cache is produced by a CUDA kernel, token by token, into a pool
of physical blocks addressed through a block table (logical local block b of
this rank -> pool block ``block_table[b]``), so a serving loop can append the
tokens of each prefill without host copies and without contiguous shards.

Pool layout: ``[pool_blocks, 2 * Hkv * bs * D]`` in the cache dtype (e4m3fn or
bf16) -- the packed payload format, one block per row.

A batch of whole sequences on one GPU (``cache_append``, ``cache_read``,
``chunk_attention``) shares one convention: rows ``offsets[b] .. offsets[b + 1]`` of a packed
``[heads, rows, D]`` tensor are sequence b's tokens of the call, and they are
the last of the ``kv_len[b]`` tokens it then has; position p lives in row
``p % block_size`` of pool block ``block_tables[b, p // block_size]``.  An e4m3
pool may carry ``scales`` (``make_scales``): a power of two for each token, head
and K or V, so that rows of any size keep e4m3's relative precision and what is
read back is exact in bf16.  Such a pool is for these three calls alone: a pool does
not know its scales, and the other entries here, which stripe one sequence over ranks,
read its codes at unit scale.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _capi
from .config import PCPAttentionConfig
from .cuda_backend import _cuda_stream_ptr, _kv_code, make_dims, payload_elements
from .rotary import _allocate, _capturing, _check_apart, _check_rows, _check_writable, _heads, _launch


def make_pool(config: PCPAttentionConfig, pool_blocks: int, kv_dtype: torch.dtype = torch.float8_e4m3fn,
              device: int | torch.device | str = "cuda") -> torch.Tensor:
    """A zeroed block pool ``[pool_blocks, payload]``."""
    if pool_blocks <= 0:
        raise ValueError("pool_blocks must be positive")
    return torch.zeros((pool_blocks, payload_elements(config)), dtype=kv_dtype, device=device)


def make_scales(config: PCPAttentionConfig, pool_blocks: int,
                device: int | torch.device | str = "cuda") -> torch.Tensor:
    """Scale bytes of an e4m3 pool, ``[pool_blocks, 2 * Hkv * bs]`` uint8: a
    byte b, 27 to 247, stands for ``2 ** (b - 127)``; all at unit scale."""
    if pool_blocks <= 0:
        raise ValueError("pool_blocks must be positive")
    shape = (pool_blocks, 2 * config.num_kv_heads * config.block_size)
    return torch.full(shape, 127, dtype=torch.uint8, device=device)


def local_blocks_needed(config: PCPAttentionConfig, rank: int, total_len: int) -> int:
    """Logical blocks rank ``rank`` needs to hold its share of positions
    ``[0, total_len)``."""
    return -(-config_source_len(config, rank, total_len) // config.block_size)


def config_source_len(config: PCPAttentionConfig, rank: int, total_len: int) -> int:
    """Positions of ``[0, total_len)`` that rank ``rank`` owns (stripe layout,
    ``layout.py:10-31``)."""
    stride = config.pcp_size * config.interleave_size
    return (total_len // stride) * config.interleave_size + min(
        max(total_len % stride - rank * config.interleave_size, 0), config.interleave_size
    )


def _check_pool(config: PCPAttentionConfig, pool: torch.Tensor, kv_dtype: torch.dtype) -> None:
    if pool.dim() != 2 or pool.shape[1] != payload_elements(config) or pool.dtype != kv_dtype:
        raise ValueError(f"pool must be [blocks, {payload_elements(config)}] {kv_dtype}, got "
                         f"{tuple(pool.shape)} {pool.dtype}")
    if not (pool.is_cuda and pool.is_contiguous()):
        raise ValueError("pool must be a contiguous CUDA tensor")


def _check_table(table: torch.Tensor, device: torch.device) -> None:
    if table.dtype != torch.int32 or not table.is_contiguous() or table.device != device:
        raise ValueError(f"block table must be a contiguous int32 tensor on {device}")


def cache_write(config: PCPAttentionConfig, rank: int, first_position: int, k_src: torch.Tensor,
                v_src: torch.Tensor, block_table: torch.Tensor, pool: torch.Tensor,
                status: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Write the tokens of ``k_src``/``v_src`` (``[Hkv, T, D]`` bf16, sequence
    order, token t at absolute position ``first_position + t``) that rank
    ``rank`` owns into its pool, quantised to the pool's dtype.  Returns the
    device int32 status word (0, or 109 when a table entry lies outside the
    pool; that token is skipped).  Asynchronous on ``stream``."""
    kv_dtype = pool.dtype
    dims = make_dims(config, kv_dtype)
    _check_pool(config, pool, kv_dtype)
    _check_table(block_table, pool.device)
    shape = (config.num_kv_heads, k_src.shape[1] if k_src.dim() == 3 else -1, config.head_dim)
    for name, t in (("k_src", k_src), ("v_src", v_src)):
        if t.dim() != 3 or tuple(t.shape) != shape or t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be [Hkv, T, D] bf16 {shape}, got {tuple(t.shape)} {t.dtype}")
        if not t.is_contiguous() or t.device != pool.device:
            raise ValueError(f"{name} must be contiguous on {pool.device}")
    if status is None:
        status = torch.empty(1, dtype=torch.int32, device=pool.device)
    with torch.cuda.device(pool.device):
        _capi.check(
            _capi.lib().pcp_cache_write(
                ctypes.byref(dims), config.interleave_size, rank, int(first_position), int(k_src.shape[1]),
                ctypes.c_void_p(k_src.data_ptr()), ctypes.c_void_p(v_src.data_ptr()),
                ctypes.c_void_p(block_table.data_ptr()), int(block_table.numel()), ctypes.c_void_p(pool.data_ptr()),
                int(pool.shape[0]), ctypes.c_void_p(status.data_ptr()), _cuda_stream_ptr(stream)
            )
        )
    return status


def history_attention_paged_single(q: torch.Tensor, pool: torch.Tensor, block_tables: torch.Tensor, valid_len,
                                   config: PCPAttentionConfig, out: torch.Tensor | None = None,
                                   stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """``history_attention_single`` over paged shards: source s's logical
    blocks are pool blocks ``block_tables[s]`` (``[sources, max_local_blocks]``
    int32 on the device)."""
    kv_dtype = pool.dtype
    dims = make_dims(config, kv_dtype)
    _check_pool(config, pool, kv_dtype)
    vals = [int(v) for v in valid_len]
    nsrc = len(vals)
    _check_table(block_tables, pool.device)
    if tuple(block_tables.shape) != (nsrc, config.max_local_blocks):
        raise ValueError(f"block_tables must be [{nsrc}, {config.max_local_blocks}]")
    if q.dtype != torch.bfloat16 or tuple(q.shape) != (config.num_q_heads, config.local_q_len, config.head_dim):
        raise ValueError("bad Q")
    if not (q.is_cuda and q.is_contiguous()):
        raise ValueError("q must be a contiguous CUDA tensor")
    lib = _capi.lib()
    nbytes = ctypes.c_size_t()
    _capi.check(lib.pcp_history_attention_workspace_size(ctypes.byref(dims), sum(vals), ctypes.byref(nbytes)))
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=q.device)
    if out is None:
        out = torch.empty_like(q)
    with torch.cuda.device(q.device):
        _capi.check(
            lib.pcp_history_attention_paged(
                ctypes.byref(dims), ctypes.c_void_p(q.data_ptr()), ctypes.c_void_p(pool.data_ptr()),
                int(pool.shape[0]), ctypes.c_void_p(block_tables.data_ptr()), nsrc, _capi.int32_array(vals),
                ctypes.c_void_p(out.data_ptr()), ctypes.c_void_p(ws.data_ptr()), nbytes.value,
                _cuda_stream_ptr(stream)
            )
        )
        _capi.check(lib.pcp_history_attention_status(ctypes.c_void_p(ws.data_ptr()), _cuda_stream_ptr(stream)))
    return out


def _pool_struct(config: PCPAttentionConfig, pool: torch.Tensor, scales: torch.Tensor | None) -> _capi.PcpPool:
    heads, block, dim, dtype = config.num_kv_heads, config.block_size, config.head_dim, pool.dtype
    if config.pcp_size != 1:
        raise ValueError(f"a batch holds whole sequences: pcp_size must be 1, got {config.pcp_size}")
    if block % 16:
        raise ValueError(f"block_size must be a multiple of 16, got {block}")
    code = _kv_code(dtype)
    _check_pool(config, pool, dtype)
    blocks = pool.shape[0]
    if scales is None:
        return _capi.PcpPool(pool.data_ptr(), 0, blocks, heads, dim, block, code)
    data = scales.data_ptr()
    if code != _capi.PCP_KV_E4M3:
        raise ValueError("scales need an e4m3 pool")
    if scales.shape != (blocks, 2 * heads * block) or scales.dtype != torch.uint8 or scales.device != pool.device or \
            data % 16 or not scales.is_contiguous():
        raise ValueError(f"scales must be a contiguous, 16-byte aligned uint8 {(blocks, 2 * heads * block)} tensor on "
                         f"{pool.device}")
    return _capi.PcpPool(pool.data_ptr(), data, blocks, heads, dim, block, code)


def _batch_struct(offsets: torch.Tensor, kv_len: torch.Tensor, block_tables: torch.Tensor, rows: int,
                  device: torch.device) -> _capi.PcpBatch:
    int32, shape = torch.int32, block_tables.shape
    if offsets.dtype != int32 or kv_len.dtype != int32 or block_tables.dtype != int32 or offsets.dim() != 1 or \
            kv_len.dim() != 1 or len(shape) != 2 or offsets.device != device or kv_len.device != device or \
            block_tables.device != device or not offsets.is_contiguous() or not kv_len.is_contiguous() or \
            (block_tables.stride(1) != 1 and block_tables.numel()):
        given = ", ".join(f"{name} {tuple(t.shape)} {t.dtype} on {t.device}" for name, t in
                          (("offsets", offsets), ("kv_len", kv_len), ("block_tables", block_tables)))
        raise ValueError("offsets, kv_len and block_tables must be int32 tensors of 1, 1 and 2 dimensions with "
                         f"contiguous rows on {device}, got {given}")
    seqs, (tables, width) = kv_len.shape[0], shape
    if offsets.shape[0] != seqs + 1 or tables != seqs:
        raise ValueError(f"{seqs} sequences need {seqs + 1} offsets and {seqs} block tables, got {offsets.shape[0]} "
                         f"and {tables}")
    return _capi.PcpBatch(offsets.data_ptr(), kv_len.data_ptr(), block_tables.data_ptr(),
                          block_tables.stride(0) if seqs > 1 else 0, width, seqs, rows, 0)


class _Status:
    """The device status word of a call: the caller's (the call stays
    asynchronous, and a word that is not 0 is kept), or an own one that is read
    after the call, which then raises what the kernels reported."""

    def __init__(self, status: torch.Tensor | None, device: torch.device, stream: torch.cuda.Stream | None):
        self.own = status is None
        if self.own:
            if _capturing(stream):
                raise ValueError("a captured call needs a status tensor: its result cannot be read while recording")
            with torch.cuda.stream(stream):
                status = torch.zeros(1, dtype=torch.int32, device=device)
        elif status.dtype != torch.int32 or status.numel() != 1 or status.device != device:
            raise ValueError(f"status must be an int32 tensor of one element on {device}")
        self.word, self.ptr = status, status.data_ptr()

    def finish(self, stream: torch.cuda.Stream | None) -> None:
        if self.own:
            _launch(self.word.device, stream, _capi.lib().pcp_history_attention_status, self.ptr)


def cache_append(config: PCPAttentionConfig, k_src: torch.Tensor, v_src: torch.Tensor, offsets: torch.Tensor,
                 kv_len: torch.Tensor, block_tables: torch.Tensor, pool: torch.Tensor,
                 scales: torch.Tensor | None = None, status: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None) -> None:
    """Write the new tokens of a batch of sequences (``k_src``/``v_src``
    ``[Hkv, rows, D]`` bf16, heads and rows at any 16-byte aligned stride) into
    their pages: ``offsets`` int32 ``[B + 1]``, ``kv_len`` int32 ``[B]`` (the
    tokens of each sequence once these are in), ``block_tables`` int32
    ``[B, width]``.  A bf16 pool takes copies, an e4m3 pool codes at unit scale
    or, with ``scales``, codes and a scale byte for each token and head.  Rows
    of no sequence are ignored.  With ``status`` (device int32, one element)
    the call is asynchronous and stores 109 (a page outside the pool or the
    table; its tokens are skipped) or 112 (a position below 0) there unless an
    earlier call's code still stands (the caller clears it); without, it waits
    and raises."""
    ps = _pool_struct(config, pool, scales)
    rows = k_src.shape[1] if k_src.dim() == 3 else -1
    device, shape = pool.device, (config.num_kv_heads, rows, config.head_dim)
    hk = _check_rows("k_src", k_src, shape, torch.bfloat16, device)
    hv = _check_rows("v_src", v_src, shape, torch.bfloat16, device)
    batch = _batch_struct(offsets, kv_len, block_tables, rows, device)
    st = _Status(status, device, stream)
    _launch(device, stream, _capi.lib().pcp_cache_append, ps, batch, hk, hv, st.ptr)
    st.finish(stream)


def cache_read(config: PCPAttentionConfig, offsets: torch.Tensor, kv_len: torch.Tensor, block_tables: torch.Tensor,
               pool: torch.Tensor, rows: int | None = None, scales: torch.Tensor | None = None,
               k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None,
               status: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Read tokens of a batch of sequences back from their pages as bf16: the
    last ``offsets[b + 1] - offsets[b]`` tokens of each sequence's ``kv_len[b]``
    land in rows ``offsets[b] ..`` of ``k_out``/``v_out`` ``[Hkv, rows, D]``
    (allocated for ``rows`` when not given; rows of no sequence are left as
    they were).  Every value is exact: codes times a power of two.  ``status``
    as in ``cache_append``; a page that cannot be followed reads as zeros."""
    ps = _pool_struct(config, pool, scales)
    if rows is None:
        if k_out is None:
            raise ValueError("cache_read needs rows, or k_out and v_out")
        rows = k_out.shape[1] if k_out.dim() == 3 else -1
    device, shape = pool.device, (config.num_kv_heads, int(rows), config.head_dim)
    outs, structs = [], []
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is None:
            t = torch.empty(shape, dtype=torch.bfloat16, device=device) if stream is None else \
                _allocate(stream, torch.empty, shape, dtype=torch.bfloat16, device=device)
            structs.append(_heads(t))
        else:
            structs.append(_check_rows(name, t, shape, torch.bfloat16, device))
            _check_writable(name, t)
        outs.append(t)
    _check_apart("k_out", outs[0], "v_out", outs[1])
    batch = _batch_struct(offsets, kv_len, block_tables, int(rows), device)
    st = _Status(status, device, stream)
    _launch(device, stream, _capi.lib().pcp_cache_read, ps, batch, *structs, st.ptr)
    st.finish(stream)
    return outs[0], outs[1]


def chunk_attention(q: torch.Tensor, pool: torch.Tensor, block_tables: torch.Tensor, offsets: torch.Tensor,
                    kv_len: torch.Tensor, config: PCPAttentionConfig, scales: torch.Tensor | None = None,
                    max_chunk: int | None = None, out: torch.Tensor | None = None, softmax_scale: float | None = None,
                    status: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Causal attention of a batch of sequences' new tokens over their paged
    caches, which hold those tokens too (``cache_append`` first): the query at
    position p sees positions 0 .. p of its sequence.  ``q`` ``[Hq, rows, D]``
    bf16 (heads and rows at any 16-byte aligned stride; so may ``out``, and be ``q`` itself);
    single tokens, chunks and whole prompts may be mixed.  ``max_chunk`` (default
    ``rows``) bounds the rows of every sequence; 1 for a decode step saves the
    launches that longer chunks would need.  ``softmax_scale`` defaults to
    ``config.softmax_scale``.  Weights are rounded to bf16 over a bf16 pool, and over an
    e4m3 one where ``max_chunk`` times the query heads of a KV head reaches 1024 (it is read
    through a bf16 copy then, while all tables' tokens need no more than 1 GiB of it), else to
    f16.  The call's workspace, that copy included, is allocated for it.  Rows that see nothing are zeros; rows of no
    sequence are left as they were.  ``status`` as in ``cache_append`` (112 also
    for a sequence of more than ``max_chunk`` rows, which is not written)."""
    ps = _pool_struct(config, pool, scales)
    rows = q.shape[1] if q.dim() == 3 else -1
    shape = (config.num_q_heads, rows, config.head_dim)
    device = pool.device
    hq = _check_rows("q", q, shape, torch.bfloat16, device)
    if out is None:
        out = torch.empty_like(q) if stream is None else _allocate(stream, torch.empty_like, q)
        ho = _heads(out)
    else:
        ho = _check_rows("out", out, shape, torch.bfloat16, device)
        _check_writable("out", out)
    batch = _batch_struct(offsets, kv_len, block_tables, rows, device)
    max_chunk = max(1, rows) if max_chunk is None else int(max_chunk)
    if max_chunk <= 0:
        raise ValueError(f"max_chunk must be positive, got {max_chunk}")
    scale = config.softmax_scale if softmax_scale is None else float(softmax_scale)
    lib = _capi.lib()
    nbytes = ctypes.c_size_t()
    _capi.check(lib.pcp_chunk_attention_workspace_size(ps, config.num_q_heads, batch.num_seqs, rows,
                                                       batch.table_width, max_chunk, ctypes.byref(nbytes)))
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device) if stream is None else \
        _allocate(stream, torch.empty, nbytes.value, dtype=torch.uint8, device=device)
    st = _Status(status, device, stream)
    _launch(device, stream, lib.pcp_chunk_attention, ps, batch, hq, ho, max_chunk, scale,
            ws.data_ptr(), nbytes.value, st.ptr)
    st.finish(stream)
    return out
