"""Host side of the serving operators (no GPU needed): frequencies of the
rotation, and the C ABI's refusals, which come before any device work."""

from __future__ import annotations

import contextlib
import ctypes
import math

import pytest
import torch

from aws_training_study_b200 import _capi
from aws_training_study_b200.pcp_attention import PCPAttentionConfig
from aws_training_study_b200.pcp_attention import paged, rotary
from aws_training_study_b200.pcp_attention.rotary import Rotary, qk_norm_rope, rotary_frequencies


def test_frequencies():
    plain, magnitude = rotary_frequencies(64, 10000.0)
    assert magnitude == 1.0 and plain == [10000.0 ** (-i / 32) for i in range(32)]
    assert rotary_frequencies(64, 10000.0, "linear", factor=4.0)[0] == [f / 4.0 for f in plain]
    bands, _ = rotary_frequencies(64, 10000.0, "bands", factor=8.0, original_len=8192, low=1.0, high=4.0)
    for f, b in zip(plain, bands):
        turns = 8192 * f / (2 * math.pi)
        assert b == f if turns >= 4 else b == pytest.approx(f / 8) if turns <= 1 else f / 8 < b < f
    ramp, magnitude = rotary_frequencies(64, 10000.0, "ramp", factor=16.0, original_len=4096)
    assert magnitude == pytest.approx(0.1 * math.log(16.0) + 1)
    assert ramp[0] == plain[0] and ramp[-1] == pytest.approx(plain[-1] / 16)
    assert all(f / 16 * (1 - 1e-12) <= r <= f for f, r in zip(plain, ramp))


def test_turns_are_the_frequencies():
    r = Rotary(128, 128, base=1e6)
    for t, f in zip(r._turns_host.tolist(), r.frequencies):
        assert (t % 2 ** 64) / 2.0 ** 64 == pytest.approx(f / (2 * math.pi), rel=1e-15, abs=2.0 ** -64)


@pytest.mark.parametrize("args", [
    dict(head_dim=100), dict(head_dim=528), dict(head_dim=128, rotary_dim=24), dict(head_dim=128, rotary_dim=144),
    dict(head_dim=128, layout="other"), dict(head_dim=128, base=1.0), dict(head_dim=128, scaling="other", factor=2.0),
    dict(head_dim=128, scaling="linear", factor=0.0), dict(head_dim=128, scaling="ramp", factor=2.0),
    dict(head_dim=128, scaling="bands", factor=2.0, original_len=8192, low=4.0, high=4.0)])
def test_rotary_refusals(args):
    with pytest.raises(ValueError):
        Rotary(**args)


def _heads(data=16, head=128, row=128, heads=2):
    return _capi.PcpHeads(data, head, row, heads, 0)


def test_qk_norm_rope_refusals():
    lib = _capi.lib()

    def call(dtype=2, rows=4, D=128, r=64, layout=0, q=None, k=None, q_out=None, k_out=None, positions=16, turns=16,
             wq=0):
        q, k = q or _heads(), k or _heads(heads=0, data=0)
        return lib.pcp_qk_norm_rope(dtype, rows, D, r, layout, q, k, q_out or q, k_out or k, positions, 1, turns, 1.0,
                                    wq, 0, 1e-6, None)

    for args in (dict(dtype=3), dict(rows=-1), dict(D=120), dict(D=528), dict(r=8), dict(r=144), dict(layout=2),
                 dict(q=_heads(data=8)), dict(q=_heads(row=100)), dict(q=_heads(head=4)), dict(q=_heads(data=0)),
                 dict(q_out=_heads(heads=3)), dict(positions=0), dict(turns=0), dict(wq=8)):
        assert call(**args) in (1, 2), args
        assert lib.pcp_last_error()
    assert call(rows=0) == 0
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(torch.zeros(1, 1, 128), None, torch.zeros(1, dtype=torch.int64), Rotary(128))


def test_an_output_in_place_may_not_overlap_itself(monkeypatch):
    """Broadcast heads or rows are inputs like any other, but not outputs: the
    kernel would norm and rotate the same memory several times."""
    launched = []
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(rotary, "_launch", lambda *args: launched.append(args))
    plain, positions, turn = torch.zeros(4, 5, 128), torch.zeros(5, dtype=torch.int64), Rotary(128)
    wide = [torch.zeros(1, 5, 128).expand(4, 5, 128), torch.zeros(4, 1, 128).expand(4, 5, 128),
            torch.zeros(4 * 5 * 128).as_strided((4, 5, 128), (64, 512, 1))]
    for x in wide:
        with pytest.raises(ValueError, match="q_out overlaps"):
            qk_norm_rope(x, None, positions, turn, q_out=x)
        with pytest.raises(ValueError, match="k_out overlaps"):
            qk_norm_rope(plain, x, positions, turn, k_out=x)
    assert not launched
    for x in [plain, *wide]:
        out, _ = qk_norm_rope(x, None, positions, turn)
        assert out.shape == x.shape and launched.pop()
    assert qk_norm_rope(plain, plain.clone(), positions, turn, q_out=plain)[0] is plain and launched


def test_two_outputs_may_not_be_the_same_memory(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    launched = []
    for module in (rotary, paged):
        monkeypatch.setattr(module, "_launch", lambda *args: launched.append(args))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    x, y, positions, turn = torch.zeros(2, 5, 128), torch.zeros(2, 5, 128), torch.zeros(5, dtype=torch.int64), Rotary(128)
    for args in (dict(q_out=x, k_out=x), dict(q_out=y), dict(k_out=x), dict(q_out=torch.zeros(4, 5, 128)[2:], k_out=x)):
        with pytest.raises(ValueError, match="the same memory"):
            qk_norm_rope(x, y, positions, turn, **args)
    qk_norm_rope(x, y, positions, turn, q_out=x, k_out=y)
    cfg = PCPAttentionConfig(1, 64, 1024, 1024, 64, 16, 4, 2, 128)
    pool, ints = torch.zeros(2, 2 * 2 * 64 * 128, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    both = torch.zeros(2, 5, 2, 128, dtype=torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32)
    read = lambda k, v: paged.cache_read(cfg, ints, ints[:1], ints[None], pool, k_out=k, v_out=v, status=status)
    with pytest.raises(ValueError, match="the same memory"):
        read(both[:, :, 0], both[:, :, 0])
    assert len(launched) == 1 and read(both[:, :, 0], both[:, :, 1]) and len(launched) == 2


def test_a_capture_of_the_given_stream_is_seen(monkeypatch):
    """What a call cannot do while its stream is captured is refused, whether
    that stream is the current one or the one it was given."""
    current = [None]

    @contextlib.contextmanager
    def stream(s):
        before, current[0] = current[0], s
        yield
        current[0] = before

    capturing = {None: False, "idle": False, "captured": True}
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[current[0]])
    cpu, table = torch.device("cpu"), Rotary(128)
    with pytest.raises(ValueError, match="captured"):
        paged._Status(None, cpu, "captured")
    with pytest.raises(RuntimeError, match="before the capture"):
        table.turns(cpu, "captured")
    paged._Status(torch.zeros(1, dtype=torch.int32), cpu, "captured")
    assert paged._Status(None, cpu, "idle").own and paged._Status(None, cpu, None).own
    with stream("captured"):
        for given in (None, "idle"):
            with pytest.raises(ValueError, match="captured"):
                paged._Status(None, cpu, given)
            with pytest.raises(RuntimeError, match="before the capture"):
                table.turns(cpu, given)
    assert table.turns(cpu, "idle") is table.turns(cpu, "captured")


@pytest.mark.parametrize("entry", ["pcp_cache_append", "pcp_cache_read"])
def test_cache_refusals(entry):
    lib = _capi.lib()

    def call(pool=None, batch=None, k=None, v=None, status=16):
        pool = {"data": 16, "scales": 16, "blocks": 4, "num_kv_heads": 2, "head_dim": 128, "block_size": 64,
                "kv_dtype": 0, **(pool or {})}
        batch = {"offsets": 16, "kv_len": 16, "block_tables": 16, "table_stride": 4, "table_width": 4, "num_seqs": 1,
                 "rows": 4, **(batch or {})}
        return getattr(lib, entry)(ctypes.byref(_capi.PcpPool(**pool)), ctypes.byref(_capi.PcpBatch(**batch)),
                                   k or _heads(), v or _heads(), status, None)

    for args in (dict(pool={"head_dim": 64}), dict(pool={"block_size": 24}), dict(pool={"kv_dtype": 2}),
                 dict(pool={"kv_dtype": 1}), dict(pool={"blocks": 0}), dict(pool={"data": 8}),
                 dict(pool={"scales": 8}), dict(pool={"num_kv_heads": 0}), dict(batch={"rows": -1}),
                 dict(batch={"num_seqs": -1}), dict(batch={"offsets": 0}), dict(batch={"table_stride": -1}),
                 dict(k=_heads(heads=1)), dict(v=_heads(row=4)), dict(k=_heads(data=0)), dict(status=0)):
        assert call(**args) in (1, 2), args
        assert lib.pcp_last_error()


def test_batches_hold_whole_sequences():
    cfg = PCPAttentionConfig(2, 64, 1024, 1024, 64, 16, 4, 2, 128)
    pool = torch.zeros(2, 2 * 2 * 64 * 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="pcp_size"):
        paged._pool_struct(cfg, pool, None)


def test_chunk_attention_refusals():
    lib = _capi.lib()

    def call(pool=None, batch=None, q=None, out=None, max_chunk=4, scale=0.1, ws=256, nbytes=1 << 40, status=16):
        pool = {"data": 16, "scales": 16, "blocks": 4, "num_kv_heads": 2, "head_dim": 128, "block_size": 64,
                "kv_dtype": 0, **(pool or {})}
        batch = {"offsets": 16, "kv_len": 16, "block_tables": 16, "table_stride": 4, "table_width": 4, "num_seqs": 1,
                 "rows": 4, **(batch or {})}
        return lib.pcp_chunk_attention(ctypes.byref(_capi.PcpPool(**pool)), ctypes.byref(_capi.PcpBatch(**batch)),
                                       q or _heads(heads=4), out or _heads(heads=4), max_chunk, scale, ws, nbytes,
                                       status, None)

    nan, inf = float("nan"), float("inf")
    for args in (dict(pool={"head_dim": 64}), dict(pool={"block_size": 24}), dict(pool={"kv_dtype": 2}),
                 dict(pool={"kv_dtype": 1}), dict(pool={"data": 0}), dict(pool={"scales": 8}),
                 dict(pool={"num_kv_heads": 3}), dict(batch={"rows": -1}), dict(batch={"num_seqs": -1}),
                 dict(batch={"kv_len": 0}), dict(batch={"block_tables": 0}), dict(q=_heads(heads=3)),
                 dict(q=_heads(heads=4, row=4)), dict(q=_heads(heads=4, data=8)), dict(out=_heads(heads=4, data=0)),
                 dict(out=_heads(heads=2)), dict(max_chunk=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=nan),
                 dict(scale=inf), dict(ws=0), dict(ws=128), dict(nbytes=1000), dict(status=0)):
        assert call(**args) in (1, 2), args
        assert lib.pcp_last_error()
    assert call(batch={"rows": 0}) == 0 and call(batch={"num_seqs": 0}) == 0  # nothing to do


def test_chunk_attention_workspace():
    """Small while every chunk is small; a bf16 copy of the cache from 1024 rows a KV head on, up to 1 GiB of it."""
    lib = _capi.lib()

    def need(q_heads=8, seqs=2, rows=4096, width=16, max_chunk=1, **pool):
        pool = _capi.PcpPool(**{"data": 16, "scales": 16, "blocks": 4, "num_kv_heads": 2, "head_dim": 128,
                                "block_size": 64, "kv_dtype": 0, **pool})
        nbytes = ctypes.c_size_t()
        rc = lib.pcp_chunk_attention_workspace_size(ctypes.byref(pool), q_heads, seqs, rows, width, max_chunk,
                                                    ctypes.byref(nbytes))
        return nbytes.value if rc == 0 else -rc

    copy = 2 * 2 * 128 * 2 * 2 * 1024  # K and V of 2 heads, bf16, 2 sequences of 16 pages of 64
    assert need() == need(max_chunk=8) < need(max_chunk=9) == need(max_chunk=255) == need(max_chunk=256) - copy
    assert need(max_chunk=256, kv_dtype=1, scales=0) == need(max_chunk=255)
    assert need(max_chunk=256, width=1 << 20) == need(max_chunk=255) == need(max_chunk=256, width=0)
    assert need(q_heads=3) == need(max_chunk=0) == need(rows=-1) == -1
    assert need(rows=2 ** 30, q_heads=64) in (-1, -2)


@pytest.mark.parametrize("P", [1, 4])
def test_prefill_positions(P):
    """The current tokens' global positions of every rank, from the first on, each once."""
    from aws_training_study_b200.pcp_attention.cuda_backend import HistoryAttention

    got = []
    for rank in range(P):
        attn = HistoryAttention.__new__(HistoryAttention)
        attn.config, attn.rank, attn.device = PCPAttentionConfig(P, 512, 1024, 1024, 64, 32, 4, 2, 128), rank, torch.device("cpu")
        attn._striped, attn._handle = None, None
        first = attn._positions(1000)
        assert first.dtype == torch.int64 and first[0] == 1000 + 32 * rank
        assert torch.equal(attn._positions(0), first - 1000)
        got.append(first)
    assert torch.equal(torch.cat(got).sort().values, torch.arange(1000, 1512))
