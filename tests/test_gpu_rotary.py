"""Norm and rotation of query and key heads (needs a B200) against the formula
in 64 bits.

Tolerance: half a step of the output type, plus what fp32 arithmetic may lose
of the terms a pair is summed from, 2e-6 * magnitude * (|a| + |b|): the angle
is rounded once (pi / 4 * 2^-24), sine and cosine, the magnitude, two
products and a sum are each within about 2^-24, and the norm's sum of squares
over at most 16 serial and 5 shuffled terms, its square root and two products
within 1e-6."""

from __future__ import annotations

import math

import pytest
import torch

from aws_training_study_b200.pcp_attention import PCPAttentionConfig
from aws_training_study_b200.pcp_attention.rotary import Rotary, qk_norm_rope, rotary_frequencies

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _formula(x, positions, rotary, weight, eps):
    """(value, sum of the magnitudes it is made of) in 64 bits."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    r = rotary.rotary_dim
    size = y.abs()
    out = y.clone()
    if r:
        pair = torch.arange(r // 2, device=x.device)
        one, two = (pair, pair + r // 2) if rotary.layout == "half" else (2 * pair, 2 * pair + 1)
        t = positions.double()[:, None] * torch.tensor(rotary.frequencies, dtype=torch.float64, device=x.device)
        c, s = t.cos() * rotary.magnitude, t.sin() * rotary.magnitude
        a, b = y[..., one], y[..., two]
        out[..., one], out[..., two] = a * c - b * s, b * c + a * s
        size[..., one] = size[..., two] = (a.abs() + b.abs()) * rotary.magnitude
    return out, size


def _check(got, x, positions, rotary, weight, eps=1e-6):
    want, size = _formula(x, positions, rotary, weight, eps)
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() + 2e-6 * size
    if x.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of its subnormals
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("head_dim,rotary_dim", [(256, 64), (128, 128), (96, 48), (64, 0), (512, 512), (16, 16)])
@pytest.mark.parametrize("rows,heads", [(1, (32, 2)), (7, (5, 3)), (301, (8, 1))])
def test_against_the_formula(rows, heads, head_dim, rotary_dim, layout, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows + head_dim)
    rotary = Rotary(head_dim, rotary_dim, base=500000.0, layout=layout)
    q = (torch.randn(heads[0], rows, head_dim, generator=g, device=DEV) * 3).to(dtype)
    k = (torch.randn(heads[1], rows, head_dim, generator=g, device=DEV) * 0.01).to(dtype)
    wq = (1 + 0.3 * torch.randn(head_dim, generator=g, device=DEV)).to(dtype)
    wk = (1 + 0.3 * torch.randn(head_dim, generator=g, device=DEV)).to(dtype)
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, device=DEV)
    for weights in ((wq, wk), (None, None), (wq, None)):
        a, b = qk_norm_rope(q, k, pos, rotary, q_weight=weights[0], k_weight=weights[1])
        _check(a, q, pos, rotary, weights[0])
        _check(b, k, pos, rotary, weights[1])


@pytest.mark.parametrize("scaling,args", [
    ("linear", {"factor": 4.0}), ("bands", {"factor": 8.0, "original_len": 8192}),
    ("ramp", {"factor": 16.0, "original_len": 4096})])
def test_scaled_frequencies_and_far_positions(scaling, args):
    """Positions up to 2^31 - 1 and below zero: the angle is exact at any."""
    g = torch.Generator(device=DEV).manual_seed(3)
    rotary = Rotary(128, base=10000.0, scaling=scaling, **args)
    pos = torch.tensor([0, 1, -1, 8191, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -(1 << 31)], device=DEV)
    q = torch.randn(4, pos.numel(), 128, generator=g, device=DEV)
    for p in (pos, pos.to(torch.int32)):
        out, none = qk_norm_rope(q, None, p, rotary)
        assert none is None
        # at 2^31 the 64-bit product of the formula itself is off by 2^31 * 2^-53 of a radian: within the bound
        _check(out, q, p, rotary, None)


def test_strides_in_place_and_streams():
    """Projections of [rows, (q, k, v) heads, D] seen as [heads, rows, D]; in
    place; on a side stream; rows left alone between them."""
    g = torch.Generator(device=DEV).manual_seed(4)
    rows, hq, hk, D = 37, 6, 2, 128
    qkv = torch.randn(rows, hq + 2 * hk, D, generator=g, device=DEV).to(torch.bfloat16)
    before = qkv.clone()
    rotary = Rotary(D, 32, layout="interleaved")
    pos = torch.arange(100, 100 + rows, device=DEV, dtype=torch.int32)
    q, k = qkv[:, :hq].transpose(0, 1), qkv[:, hq:hq + hk].transpose(0, 1)
    want_q, want_k = qk_norm_rope(q.contiguous(), k.contiguous(), pos, rotary)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a, b = qk_norm_rope(q, k, pos, rotary, q_out=q, k_out=k, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert a is q and torch.equal(q, want_q) and torch.equal(k, want_k)
    assert torch.equal(qkv[:, hq + hk:], before[:, hq + hk:])
    # a broadcast input (one head seen by several) is read, and its gap rows are not touched
    one = before[:, :1].transpose(0, 1).expand(4, rows, D)
    out, _ = qk_norm_rope(one, None, pos, rotary)
    assert all(torch.equal(out[i], out[0]) for i in range(4))


def test_heads_far_apart_in_memory():
    gap = 1 << 31
    far = torch.empty(3 * gap, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    q = far.as_strided((2, 9, 128), (gap, 128, 1)).copy_(torch.randn(2, 9, 128, generator=g, device="cuda"))
    out = far.as_strided((2, 9, 128), (gap, 128, 1), gap // 2)
    positions = torch.arange(9, device="cuda") + (1 << 40)
    want, _ = qk_norm_rope(q.contiguous(), None, positions, Rotary(128))
    qk_norm_rope(q, None, positions, Rotary(128), q_out=out)
    assert torch.equal(out, want)


def test_captured_and_replayed():
    rotary = Rotary(256, 64)
    q = torch.randn(32, 5, 256, device=DEV).to(torch.bfloat16)
    k = torch.randn(2, 5, 256, device=DEV).to(torch.bfloat16)
    w = torch.ones(256, device=DEV, dtype=torch.bfloat16)
    pos = torch.arange(5, device=DEV)
    rotary.turns(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = qk_norm_rope(q, k, pos, rotary, q_weight=w, k_weight=w)
    for shift in (0, 90000):
        pos.copy_(torch.arange(5, device=DEV) + shift)
        graph.replay()
        _check(a, q, pos, rotary, w)
        _check(b, k, pos, rotary, w)


def test_non_finite_rows_stay_alone():
    rotary = Rotary(128)
    q = torch.randn(2, 6, 128, device=DEV)
    clean = q.clone()
    q[0, 2, 5], q[1, 4, 100] = float("nan"), float("inf")
    w = torch.ones(128, device=DEV)
    pos = torch.arange(6, device=DEV)
    got, want = qk_norm_rope(q, None, pos, rotary, q_weight=w)[0], qk_norm_rope(clean, None, pos, rotary, q_weight=w)[0]
    assert torch.isnan(got[0, 2]).all() and torch.isnan(got[1, 4]).any()
    got[0, 2], got[1, 4] = want[0, 2], want[1, 4]
    assert torch.equal(got, want)


def test_refusals():
    rotary = Rotary(128, 64)
    pos = torch.arange(4, device=DEV)
    q = torch.zeros(2, 4, 128, device=DEV, dtype=torch.bfloat16)
    for bad in (dict(q=q.cpu()), dict(q=q.double()), dict(q=q[..., :64]), dict(pos=pos[:3]), dict(pos=pos.float()),
                dict(q=torch.zeros(2, 4, 132, device=DEV, dtype=torch.bfloat16)[..., :128]),
                dict(q=torch.zeros(2 * 4 * 128 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(2, 4, 128)),
                dict(q_weight=torch.zeros(128, device=DEV)), dict(k_weight=torch.zeros(128, device=DEV, dtype=q.dtype)),
                dict(q_out=torch.zeros(1, 4, 128, device=DEV, dtype=q.dtype).expand(2, 4, 128))):
        args = {"q": q, "k": None, "pos": pos, **bad}
        with pytest.raises(ValueError):
            qk_norm_rope(args.pop("q"), args.pop("k"), args.pop("pos"), rotary, **args)
    empty = qk_norm_rope(q[:, :0], q[:1, :0], pos[:0], rotary)
    assert empty[0].shape == (2, 0, 128) and empty[1].shape == (1, 0, 128)


def test_prefill_prepares_its_queries_and_keys():
    """HistoryAttention.prefill with a rotation: the same as preparing q and k
    first, at the positions behind the history or where told; on a side stream."""
    from aws_training_study_b200.pcp_attention.cuda_backend import HistoryAttention

    from parity import make_case, make_current, packed_shards

    cfg = PCPAttentionConfig(1, 1024, 4096, 4096, 512, 64, 16, 2, 128)
    _, _, _, q_shards, k_shards, v_shards = make_case(cfg, seed=31)
    _, _, kc_shards, vc_shards = make_current(cfg, seed=31)
    q, kv = q_shards[0].cuda(), packed_shards(cfg, k_shards, v_shards)[0].cuda()
    k, v = kc_shards[0].cuda(), vc_shards[0].cuda()
    g = torch.Generator(device="cuda").manual_seed(3)
    wq, wk = (torch.rand(128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    rotary = Rotary(128, 64)
    attn = HistoryAttention(cfg, rank=0, device=0)
    keep = q.clone(), k.clone()
    for first, args in ((4096, {}), (7, {"first_position": 7}), (3000, {"valid_len": [3000]})):
        pos = torch.arange(first, first + 1024, device="cuda")
        qn, kn = qk_norm_rope(q, k, pos, rotary, wq, wk, 1e-5)
        want = attn.prefill(qn, kv, kn, v, valid_len=args.get("valid_len"))
        assert torch.equal(attn.prefill(q, kv, k, v, rotary=rotary, q_weight=wq, k_weight=wk, eps=1e-5, **args), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = attn.prefill(q, kv, k, v, rotary=rotary, q_weight=wq, k_weight=wk, eps=1e-5, valid_len=[3000], stream=side)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(q, keep[0]) and torch.equal(k, keep[1])
    with pytest.raises(ValueError, match="rotary"):
        attn.prefill(q, kv, k, v, q_weight=wq)
    with pytest.raises(ValueError, match="heads of 256"):
        attn.prefill(q, kv, k, v, rotary=Rotary(256))
    attn.status()
    attn.close()
