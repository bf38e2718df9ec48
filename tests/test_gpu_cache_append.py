"""Scaled paged cache (needs a B200): codes, scale bytes and read-back against
the definition in 64 bits, bit for bit -- products by powers of two and the
rounding to e4m3 leave nothing to tolerate."""

from __future__ import annotations

import pytest
import torch

from aws_training_study_b200._capi import PcpError
from aws_training_study_b200.pcp_attention import PCPAttentionConfig
from aws_training_study_b200.pcp_attention.paged import cache_append, cache_read, cache_write, make_pool, make_scales

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _config(heads=2, D=128, bs=64, blocks=16):
    return PCPAttentionConfig(1, 16, blocks * bs, blocks * bs, bs, 16, heads, heads, D)


def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantised(x):
    """(values, scale bytes) of bf16 rows, in 64 bits, on the CPU."""
    y = x.cpu().double()
    size = torch.where(y.isfinite(), y.abs(), 0.0).amax(-1)
    m, e = torch.frexp(size)
    e = torch.where(m > 0.875, e - 8, e - 9)  # 448 = 0.875 * 2^9
    e = torch.where(size == 0, torch.zeros_like(e), e.clamp(-100, 120))
    z = y / _two_to(e)[..., None]
    _, p = torch.frexp(z.abs())
    step = _two_to(((p - 1).clamp(min=-6) - 3))
    z = torch.where(z.isfinite(), torch.round(z / step) * step, torch.nan)
    return z * _two_to(e)[..., None], (e + 127).to(torch.uint8)


def _batch(new, kv, bs, blocks, seed=0, spare=3):
    """Offsets, lengths and shuffled tables of sequences with `new` tokens each of `kv`."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(blocks, generator=g).to(torch.int32)
    width = max(1, max(-(-t // bs) for t in kv))
    tables, used = torch.full((len(kv), width + spare), -7, dtype=torch.int32), 0
    for b, t in enumerate(kv):
        n = -(-t // bs)
        tables[b, :n] = order[used:used + n]
        used += n
    offsets = torch.tensor([0] + list(new)).cumsum(0).to(torch.int32)
    return offsets.to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV), tables.to(DEV)


def _rows_of(pool, scales, cfg, table, pos):
    """(codes or values, scale bytes) [2, Hkv, D] of one position, straight from the pool."""
    page, slot = int(table[pos // cfg.block_size]), pos % cfg.block_size
    shape = (-1, 2, cfg.num_kv_heads, cfg.block_size)
    row = pool.view(torch.uint8).view(*shape, cfg.head_dim * pool.element_size())[page, :, :, slot]
    return row.view(pool.dtype), None if scales is None else scales.view(shape)[page, :, :, slot]


@pytest.mark.parametrize("D,heads,bs", [(128, 2, 64), (256, 1, 16), (256, 3, 48), (128, 8, 512)])
@pytest.mark.parametrize("new,kv", [([1], [1]), ([3, 0, 5, 1], [200, 40, 5, 77]), ([130] * 2, [131, 500])])
def test_append_and_read_back_scaled(new, kv, D, heads, bs):
    cfg = _config(heads, D, bs)
    blocks = sum(-(-t // bs) for t in kv) + 2
    offsets, kv_len, tables = _batch(new, kv, bs, blocks)
    g = torch.Generator().manual_seed(D + bs)
    rows = sum(new) + 2  # two rows of no sequence behind the last
    size = torch.exp2(torch.randint(-30, 30, (heads, rows, 1), generator=g).float())
    k = (torch.randn(heads, rows, D, generator=g) * size).to(torch.bfloat16)
    v = (torch.randn(heads, rows, D, generator=g) / size).to(torch.bfloat16)
    k[:, 0] = 0.0
    pool, scales = make_pool(cfg, blocks, device=DEV), make_scales(cfg, blocks, DEV)
    cache_append(cfg, k.to(DEV), v.to(DEV), offsets, kv_len, tables, pool, scales=scales)
    touched = torch.zeros_like(scales.view(-1, 2, heads, bs))
    kq, ke = _quantised(k)
    vq, ve = _quantised(v)
    for b in range(len(new)):
        for i in range(new[b]):
            r, pos = int(offsets[b]) + i, kv[b] - new[b] + i
            codes, e = _rows_of(pool, scales, cfg, tables[b].cpu(), pos)
            value = codes.float().cpu().double() * _two_to(e.cpu().long() - 127)[..., None]
            assert torch.equal(e.cpu(), torch.stack((ke[:, r], ve[:, r])))
            assert torch.equal(value, torch.stack((kq[:, r], vq[:, r])))
            touched[int(tables[b, pos // bs]), :, :, pos % bs] = 1
    # everything else is as it was
    untouched = pool.view(torch.uint8).view(-1, 2, heads, bs, D)[touched == 0]
    assert int(untouched.count_nonzero()) == 0 and (scales.view(-1, 2, heads, bs)[touched == 0] == 127).all()
    out = [torch.full((heads, rows, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    cache_read(cfg, offsets, kv_len, tables, pool, scales=scales, k_out=out[0], v_out=out[1])
    n = sum(new)
    assert torch.equal(out[0][:, :n].cpu().double(), kq[:, :n]) and torch.equal(out[1][:, :n].cpu().double(), vq[:, :n])
    assert (out[0][:, n:] == 7).all() and (out[1][:, n:] == 7).all()


@pytest.mark.parametrize("kv_dtype", [torch.float8_e4m3fn, torch.bfloat16], ids=["e4m3", "bf16"])
def test_pages_and_rows_far_into_memory(kv_dtype):
    """Pages beyond 2^32 bytes (and elements) of the pool, heads 2^31 elements
    apart: what goes in comes back out, and the pages are a small pool's."""
    cfg = _config(2, 256, 512)
    offsets, kv_len, tables = _batch([70, 1], [1000, 300], 512, 5)
    extra = (1 << 32) // (2 * 2 * 512 * 256) + 1
    small = make_pool(cfg, 5, kv_dtype, DEV)
    pool = torch.empty(5 + extra, small.shape[1], dtype=kv_dtype, device=DEV)
    pool.view(torch.uint8)[extra:] = 0
    e4m3 = kv_dtype == torch.float8_e4m3fn
    small_scales, scales = (make_scales(cfg, n, DEV) if e4m3 else None for n in (5, 5 + extra))
    gap = 1 << 31
    far = torch.empty(2 * gap, dtype=torch.bfloat16, device=DEV)
    k, v, k_out, v_out = (far.as_strided((2, 71, 256), (gap, 256, 1), n * gap // 4) for n in range(4))
    g = torch.Generator(device=DEV).manual_seed(6)
    for x in (k, v):
        x.copy_(torch.randn(2, 71, 256, generator=g, device=DEV))
    cache_append(cfg, k.contiguous(), v.contiguous(), offsets, kv_len, tables, small, scales=small_scales)
    cache_append(cfg, k, v, offsets, kv_len, tables + extra, pool, scales=scales)
    assert torch.equal(pool[extra:].view(torch.uint8), small.view(torch.uint8))
    assert not e4m3 or torch.equal(scales[extra:], small_scales)
    want = cache_read(cfg, offsets, kv_len, tables, small, rows=71, scales=small_scales)
    cache_read(cfg, offsets, kv_len, tables + extra, pool, scales=scales, k_out=k_out, v_out=v_out)
    assert torch.equal(k_out, want[0]) and torch.equal(v_out, want[1])


def test_every_bf16_pattern():
    """All 65536 patterns against one large element: every rounding, ties
    included; infinities and NaN become NaN and spare their row."""
    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = bits.reshape(512, 128).clone()
    cfg = _config(1, 128, 512, 1)
    offsets, kv_len, tables = _batch([512], [512], 512, 1)
    pool, scales = make_pool(cfg, 1, device=DEV), make_scales(cfg, 1, DEV)
    k = x[None].to(DEV)
    cache_append(cfg, k, k, offsets, kv_len, tables, pool, scales=scales)
    got, _ = cache_read(cfg, offsets, kv_len, tables, pool, 512, scales=scales)
    want, e = _quantised(x)
    assert torch.equal(scales.view(2, 512)[0].cpu(), e)
    # The eight largest patterns of each sign, from 248 * 2^120 on, are nearest to 256 * 2^120 = 2^128, and that
    # is above the largest bf16 value, (2 - 2^-7) * 2^127: it reads as infinity.  All else is exact.
    beyond = want.abs() == 2.0 ** 128
    assert int(beyond.sum()) == 16 and (x.double().abs()[beyond] >= 248 * 2.0 ** 120).all()
    want = torch.where(beyond, want * torch.inf, want)
    assert torch.equal(got[0].cpu().double().nan_to_num(1e300, 1e301, -1e301), want.nan_to_num(1e300, 1e301, -1e301))
    assert torch.equal(got[0].isnan().cpu(), ~x.isfinite())


@pytest.mark.parametrize("kv_dtype", [torch.float8_e4m3fn, torch.bfloat16], ids=["e4m3", "bf16"])
def test_unscaled_append_equals_cache_write(kv_dtype):
    cfg = _config(2, 256, 64)
    table = torch.tensor([[3, 0, 2, 5]], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(2, 200, 256, device=DEV).mul(200).to(torch.bfloat16) for _ in range(2))
    a, b = make_pool(cfg, 6, kv_dtype, DEV), make_pool(cfg, 6, kv_dtype, DEV)
    assert int(cache_write(cfg, 0, 0, k, v, table[0].contiguous(), a).item()) == 0
    offsets = torch.tensor([0, 200], dtype=torch.int32, device=DEV)
    kv_len = torch.tensor([200], dtype=torch.int32, device=DEV)
    cache_append(cfg, k, v, offsets, kv_len, table, b)
    assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    kr, vr = cache_read(cfg, offsets, kv_len, table, b, 200)
    want = (x.to(kv_dtype).to(torch.bfloat16) for x in (k, v))
    for got, w in zip((kr, vr), want):
        assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got.nan_to_num(), w.nan_to_num())


def test_strided_rows_and_side_stream():
    """Projections [rows, heads, D] passed transposed; read back into such a
    tensor; the newest tokens only, of an offset view of the tables."""
    cfg = _config(2, 128, 16)
    new, kv = [40, 9], [100, 30]
    offsets, kv_len, tables = _batch(new, kv, 16, 12)
    qkv = torch.randn(49, 8, 128, device=DEV).to(torch.bfloat16)
    k, v = qkv[:, 4:6].transpose(0, 1), qkv[:, 6:8].transpose(0, 1)
    pools = [make_pool(cfg, 12, device=DEV) for _ in range(2)]
    scales = [make_scales(cfg, 12, DEV) for _ in range(2)]
    cache_append(cfg, k.contiguous(), v.contiguous(), offsets, kv_len, tables.contiguous(), pools[0], scales=scales[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    wide = torch.cat((torch.zeros_like(tables), tables), 1)[:, tables.shape[1]:]
    cache_append(cfg, k, v, offsets, kv_len, wide, pools[1], scales=scales[1], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(pools[0].view(torch.uint8), pools[1].view(torch.uint8)) and torch.equal(*scales)
    last = torch.tensor([0, 5, 6], dtype=torch.int32, device=DEV)
    out = torch.zeros(6, 4, 128, dtype=torch.bfloat16, device=DEV)
    cache_read(cfg, last, kv_len, tables, pools[0], scales=scales[0], k_out=out[:, :2].transpose(0, 1),
               v_out=out[:, 2:].transpose(0, 1))
    want, _ = _quantised(torch.cat((k[:, 35:40], k[:, 48:49]), 1))
    assert torch.equal(out[:, :2].transpose(0, 1).cpu().double(), want)


def test_pages_that_cannot_be_followed():
    """An entry outside the pool, a position past the table, more new tokens
    than the sequence has: reported, the rest written, nothing else touched."""
    cfg = _config(1, 128, 16)
    pool, scales = make_pool(cfg, 2, device=DEV), make_scales(cfg, 2, DEV)
    k = torch.ones(1, 20, 128, device=DEV, dtype=torch.bfloat16)
    one = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for table, length, code in ((one(1, 2)[None], 20, 109), (one(1)[None], 20, 109), (one(1, 0)[None], 15, 112)):
        status = one(0)
        pool.view(torch.uint8).zero_()
        cache_append(cfg, k, k, one(0, 20), one(length), table, pool, scales=scales, status=status)
        assert int(status) == code
        with pytest.raises(PcpError, match=f"code {code}"):
            cache_append(cfg, k, k, one(0, 20), one(length), table, pool, scales=scales)
        written = pool.float().view(2, 2, 16, 128)[..., 0] != 0
        assert int(written[1].sum()) == 2 * min(16, length) and int(written[0].sum()) == 0
        out = [torch.full((1, 20, 128), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        cache_read(cfg, one(0, 20), one(length), table, pool, scales=scales, k_out=out[0], v_out=out[1], status=status)
        assert int(status) == code
        if code == 109:
            assert (out[0][:, :16] == 1).all() and (out[0][:, 16:] == 0).all()
        else:
            assert (out[0][:, :5] == 7).all() and (out[0][:, 5:] == 1).all()


def test_empty_batches():
    cfg = _config()
    pool, scales = make_pool(cfg, 2, device=DEV), make_scales(cfg, 2, DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    k = torch.ones(2, 3, 128, device=DEV, dtype=torch.bfloat16)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache_append(cfg, k, k, zero, none, torch.zeros(0, 4, dtype=torch.int32, device=DEV), pool, scales=scales)
    cache_append(cfg, k[:, :0], k[:, :0], torch.zeros(2, dtype=torch.int32, device=DEV), zero,
                 torch.zeros(1, 4, dtype=torch.int32, device=DEV), pool, scales=scales)
    assert int(pool.view(torch.uint8).count_nonzero()) == 0


def test_captured_and_replayed():
    """Lengths and tables change between replays; a status tensor is needed."""
    cfg = _config(1, 128, 16, 4)
    pool, scales = make_pool(cfg, 4, device=DEV), make_scales(cfg, 4, DEV)
    k = torch.full((1, 2, 128), 3.0, device=DEV, dtype=torch.bfloat16)
    offsets, kv_len, tables = _batch([1, 1], [16, 16], 16, 4)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache_append(cfg, k, k, offsets, kv_len, tables, pool, scales=scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache_append(cfg, k, k, offsets, kv_len, tables, pool, scales=scales, status=status)
        out, _ = cache_read(cfg, offsets, kv_len, tables, pool, 2, scales=scales, status=status)
    for length, value in ((1, 5.0), (9, -0.625)):
        kv_len.fill_(length)
        k.fill_(value)
        graph.replay()
        assert (out == value).all() and int(status) == 0
        for b in range(2):
            assert (pool.view(4, 2, 16, 128)[int(tables[b, 0]), :, length - 1].float() != 0).all()


def test_refusals():
    cfg = _config()
    pool, scales = make_pool(cfg, 2, device=DEV), make_scales(cfg, 2, DEV)
    k = torch.zeros(2, 3, 128, device=DEV, dtype=torch.bfloat16)
    offsets, kv_len, tables = _batch([3], [3], 64, 2)
    good = dict(k=k, v=k, offsets=offsets, kv_len=kv_len, tables=tables, pool=pool, scales=scales)
    for bad in (dict(k=k.float()), dict(v=k[:, :2]), dict(k=k[:1]), dict(offsets=offsets.long()), dict(offsets=offsets[:1]),
                dict(tables=tables.cpu()), dict(tables=tables[0]), dict(pool=pool[:, :128]), dict(scales=scales[:1]),
                dict(scales=scales.int()), dict(pool=pool.to(torch.bfloat16)),
                dict(status=torch.zeros(2, dtype=torch.int32, device=DEV))):
        a = {**good, **bad}
        with pytest.raises(ValueError):
            cache_append(cfg, a["k"], a["v"], a["offsets"], a["kv_len"], a["tables"], a["pool"], scales=a["scales"],
                         status=a.get("status"))
    with pytest.raises(ValueError):
        cache_read(cfg, offsets, kv_len, tables, pool, scales=scales)
    with pytest.raises(ValueError, match="overlaps"):
        cache_read(cfg, offsets, kv_len, tables, pool, scales=scales, k_out=k[:1].expand(2, 3, 128), v_out=k)
