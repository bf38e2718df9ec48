"""Attention of new tokens over a paged cache (needs a B200) against the
definition in 64 bits.

Tolerance, per element, with A = sum_j w_j |v_j| (w: the softmax's weights):
  * the output's rounding, half a step: 2^-8 |o|;
  * the weights' rounding before the second product: 2^-8 A in bf16 (bf16
    caches, and chunks of more than 32 rows a KV head in calls whose max_chunk
    reaches 1024 rows, which read a bf16 copy of an e4m3 cache), 2^-11 A in f16
    (other e4m3 caches), and below f16's normal range half its least step, 2^-25,
    of weights whose largest is 1 or more: n 2^-25 max|v|;
  * the scores: fp32 sums over D / 16 tensor-core steps, each within 2^-22 of
    the terms' magnitudes, and ex2 within 2^-22: (D / 16 * 2^-22 * max_j scale *
    sum_d |q_d k_jd| + 2^-20) * 2 A."""

from __future__ import annotations

import math

import pytest
import torch

from aws_training_study_b200._capi import PcpError
from aws_training_study_b200.pcp_attention import PCPAttentionConfig
from aws_training_study_b200.pcp_attention.paged import cache_append, chunk_attention, make_pool, make_scales
from aws_training_study_b200.pcp_attention.rotary import Rotary, qk_norm_rope

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
CACHES = ["bf16", "e4m3", "scaled"]


class Case:
    """A batch over shuffled pages: everything not of a sequence is NaN (codes
    0x7F, scale bytes 255), so a read past a length shows."""

    def __init__(self, new, kv, heads, D, bs, cache, seed=0, padding=0, size=1.0):
        self.new, self.kv, self.cache = new, kv, cache
        self.cfg = PCPAttentionConfig(1, 16, 1 << 20, 1 << 20, bs, 16, heads[0], heads[1], D)
        g = torch.Generator(device=DEV).manual_seed(seed)
        blocks = sum(-(-t // bs) for t in kv) + 2
        order = torch.randperm(blocks, generator=g, device=DEV)[: blocks - 2].to(torch.int32)
        width = max(1, max((-(-t // bs) for t in kv), default=1))
        self.tables = torch.zeros(len(kv), width, dtype=torch.int32, device=DEV)
        used = 0
        for b, t in enumerate(kv):
            n = -(-t // bs)
            self.tables[b, :n] = order[used:used + n]
            used += n
        self.offsets = torch.tensor([0] + list(new), device=DEV).cumsum(0).to(torch.int32)
        self.kv_len = torch.tensor(kv, dtype=torch.int32, device=DEV)
        e4m3 = cache != "bf16"
        self.pool = make_pool(self.cfg, blocks, torch.float8_e4m3fn if e4m3 else torch.bfloat16, DEV)
        (self.pool.view(torch.uint8) if e4m3 else self.pool).fill_(0x7F if e4m3 else torch.nan)
        self.scales = make_scales(self.cfg, blocks, DEV).fill_(255) if cache == "scaled" else None
        self.k, self.v = [], []
        shape = (-1, 2, heads[1], bs)
        for b, t in enumerate(kv):
            x = torch.randn(2, heads[1], t, D, generator=g, device=DEV) * size
            page = self.tables[b, torch.arange(t, device=DEV) // bs].long()
            slot = torch.arange(t, device=DEV) % bs
            if e4m3:
                e = torch.zeros(2, heads[1], t, 1, device=DEV, dtype=torch.int32)
                if cache == "scaled":
                    e = torch.randint(-9, 3, e.shape, generator=g, device=DEV, dtype=torch.int32)
                    self.scales.view(shape)[page, :, :, slot] = (e + 127).to(torch.uint8)[..., 0].permute(2, 0, 1)
                codes = x.clamp(-448, 448).to(torch.float8_e4m3fn)
                x = codes.double() * ((e.long() + 1023) << 52).view(torch.float64)
                self.pool.view(torch.uint8).view(*shape, D)[page, :, :, slot] = \
                    codes.view(torch.uint8).permute(2, 0, 1, 3)
            else:
                x = x.to(torch.bfloat16)
                self.pool.view(*shape, D)[page, :, :, slot] = x.permute(2, 0, 1, 3)
                x = x.double()
            self.k.append(x[0])
            self.v.append(x[1])
        rows = sum(new) + padding
        self.q = torch.randn(rows, heads[0], D, generator=g, device=DEV).to(torch.bfloat16).transpose(0, 1)

    def run(self, **args):
        a = dict(q=self.q, pool=self.pool, block_tables=self.tables, offsets=self.offsets, kv_len=self.kv_len,
                 config=self.cfg, scales=self.scales, max_chunk=max(self.new))
        a.update(args)
        return chunk_attention(**a)

    def expected(self, b, scale=None):
        """(o, bound) [Hq, new, D] of sequence b, in 64 bits."""
        cfg, n, t = self.cfg, self.new[b], self.kv[b]
        scale = cfg.softmax_scale if scale is None else scale
        first = int(self.offsets[b])
        q = self.q[:, first:first + n].double()
        group = cfg.num_q_heads // cfg.num_kv_heads
        o, bound = torch.zeros_like(q), torch.zeros_like(q)
        pos = torch.arange(t - n, t, device=DEV)
        hidden = torch.arange(t, device=DEV) > pos[:, None]
        for h in range(cfg.num_q_heads):
            k, v = self.k[b][h // group], self.v[b][h // group]
            if t == 0:
                continue
            s = (q[h] @ k.T * scale).masked_fill(hidden, -math.inf)
            top = s.amax(-1, keepdim=True)
            w = torch.where(hidden, 0.0, torch.exp(s - torch.where(top == -math.inf, 0.0, top)))
            total = w.sum(-1, keepdim=True)
            w = torch.where(total > 0, w / total, 0.0)
            o[h] = w @ v
            a = w @ v.abs()
            terms = (q[h].abs() @ k.abs().T * scale).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
            expanded = max(self.new) * group >= 1024 and n * group > 32
            weights = 2.0 ** -8 if self.cache == "bf16" or expanded else 2.0 ** -11
            bound[h] = 2.0 ** -8 * o[h].abs() + weights * a + 2 * a * (cfg.head_dim / 16 * 2.0 ** -22 * terms + 2.0 ** -20)
            if self.cache != "bf16":
                bound[h] += t * 2.0 ** -25 * v.abs().amax()
        return o, bound

    def check(self, out, **args):
        for b in range(len(self.new)):
            if self.new[b] == 0:
                continue
            first = int(self.offsets[b])
            got = out[:, first:first + self.new[b]].double()
            want, bound = self.expected(b, **args)
            bad = ~((got - want).abs() <= bound)
            assert not bad.any(), (f"sequence {b}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst "
                                   f"{float(((got - want).abs() / bound.clamp(min=1e-30)).nan_to_num(torch.inf).max()):.3g} of it")


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,D,bs", [((32, 2), 256, 512), ((8, 8), 128, 16), ((20, 4), 128, 48), ((7, 1), 256, 64)])
@pytest.mark.parametrize("new,kv", [
    ([1], [1]), ([1], [127]), ([1, 1, 1], [128, 129, 2000]), ([1] * 6, [3, 700, 16, 17, 4096, 1]),
])
def test_single_tokens(new, kv, heads, D, bs, cache):
    case = Case(new, kv, heads, D, bs, cache, seed=sum(kv))
    case.check(case.run())


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,D,bs", [((32, 2), 256, 64), ((8, 2), 128, 48)])
def test_drafts_of_a_few_tokens(heads, D, bs, cache):
    """17 to 32 rows a KV head, and fewer, in one batch; the last queries see
    keys that the first do not."""
    most = 32 // (heads[0] // heads[1])
    new = [most, 1, most - 1, (most + 1) // 2, most]
    case = Case(new, [most, 900, 130, 64 + most, 2500], heads, D, bs, cache, seed=5)
    case.check(case.run())


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,D,bs", [((32, 2), 256, 512), ((8, 8), 128, 16), ((20, 4), 128, 48), ((33, 1), 256, 64)])
@pytest.mark.parametrize("new,kv", [([33], [33]), ([300], [300]), ([40, 257, 64], [1000, 257, 3001]), ([129], [130])])
def test_chunks(new, kv, heads, D, bs, cache):
    case = Case(new, kv, heads, D, bs, cache, seed=sum(kv))
    case.check(case.run())


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("D,heads", [(256, (16, 2)), (128, (32, 8))])
def test_mixed_batch_with_empty_sequences_and_padding(D, heads, cache):
    """Decodes, chunks, a whole prompt, sequences without new tokens or without
    any, and rows behind the last sequence that stay as they were."""
    new = [1, 0, 350, 1, 0, 77, 1, 1, 3]
    kv = [900, 40, 350, 1, 0, 1500, 2222, 64, 3]
    case = Case(new, kv, heads, D, 64, cache, seed=8, padding=9)
    out = torch.full_like(case.q, 7.0)
    got = case.run(out=out)
    assert got is out and (out[:, sum(new):] == 7).all()
    case.check(out)


@pytest.mark.parametrize("cache", CACHES)
def test_large_scores_and_growing_maxima(cache):
    """Keys that grow along the sequence move the running maximum again and
    again; softmax weights close to one-hot."""
    case = Case([1, 200], [3000, 1800], (16, 2), 256, 128, cache, seed=9, size=4.0)
    case.check(case.run())
    case.check(case.run(softmax_scale=0.5), scale=0.5)


def test_exponents_of_any_size():
    """Scaled rows from 2^-60 to 2^30 times unit size, in K and in V: weights
    stay finite and exact in their proportions."""
    case = Case([1, 60], [700, 500], (16, 2), 128, 64, "scaled", seed=10)
    shape = (-1, 2, 2, 64)
    for b in range(2):
        t = case.kv[b]
        page = case.tables[b, torch.arange(t, device=DEV) // 64].long()
        slot = torch.arange(t, device=DEV) % 64
        old = case.scales.view(shape)[page, :, :, slot].long()  # [t, 2, Hkv]
        e = torch.randint(-30, -6, (t, 2, 2), device=DEV, generator=torch.Generator(device=DEV).manual_seed(b))
        e[:, 1] += torch.where(torch.arange(t, device=DEV) % 3 == 0, 36, -30)[:, None]
        case.scales.view(shape)[page, :, :, slot] = (e + 127).to(torch.uint8)
        change = ((e + 127 - old + 1023) << 52).view(torch.float64)
        case.k[b] = case.k[b] * change[:, 0].T[..., None]
        case.v[b] = case.v[b] * change[:, 1].T[..., None]
    case.check(case.run())


@pytest.mark.parametrize("cache", ["e4m3", "scaled"])
@pytest.mark.parametrize("power", [100, -100])
def test_queries_of_any_size(cache, power):
    """Queries far outside f16's range, with a scale that brings the scores back."""
    case = Case([1, 70], [300, 200], (8, 2), 128, 64, cache, seed=11)
    want = case.run()
    case.q = (case.q.float() * 2.0 ** power).to(torch.bfloat16)
    assert torch.equal(case.run(softmax_scale=case.cfg.softmax_scale * 2.0 ** -power), want)


def test_rows_that_see_nothing():
    """More new tokens than the sequence has: the rows below position 0 are
    zeros, the others attend as ever."""
    for new, kv in (([40], [7]), ([3], [1]), ([100], [0]), ([1], [0])):
        case = Case(new, kv, (16, 2), 128, 16, "scaled", seed=12)
        out = case.run(out=torch.full_like(case.q, 7.0))
        empty = new[0] - kv[0]
        assert (out[:, :empty] == 0).all()
        if kv[0]:
            tail = Case(kv, kv, (16, 2), 128, 16, "scaled", seed=12)
            tail.q = case.q[:, empty:]
            assert torch.equal(tail.run(max_chunk=new[0])[:, :].isfinite(), torch.ones_like(tail.q, dtype=torch.bool))
            tail.check(out[:, empty:])


@pytest.mark.parametrize("cache", CACHES)
def test_long_chunks_that_mostly_see_nothing(cache):
    case = Case([600, 300], [100, 0], (16, 2), 128, 16, cache, seed=21)
    out = case.run(out=torch.full_like(case.q, 7.0))
    assert (out[:, :500] == 0).all() and (out[:, 600:] == 0).all()
    want, bound = case.expected(0)
    assert ((out[:, 500:600].double() - want[:, 500:]).abs() <= bound[:, 500:]).all()


@pytest.mark.parametrize("heads,dim,bs", [((16, 2), 256, 64), ((8, 1), 128, 48)])
def test_chunks_among_many_decodes_with_wide_tables(heads, dim, bs):
    """70 sequences, two of them with chunks, tables far wider than the
    sequences are long, whose unused entries lead outside the pool."""
    new = [1] * 70
    kv = [10 + 37 * b % 900 for b in range(70)]
    new[33], new[69] = 140, 133
    kv[33], kv[69] = 500, 133
    case = Case(new, kv, heads, dim, bs, "scaled", seed=22)
    wide = torch.full((70, case.tables.shape[1] + 60), -1, dtype=torch.int32, device=DEV)
    for b, t in enumerate(kv):
        wide[b, :-(-t // bs)] = case.tables[b, :-(-t // bs)]
    case.check(case.run(block_tables=wide))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new", [1, 50])
def test_a_nan_key_spoils_only_rows_that_see_it(new, cache):
    case = Case([new, new], [400, 300], (16, 2), 128, 64, cache, seed=13)
    clean = case.run()
    page = case.pool.view(torch.uint8).view(-1, 2, 2, 64, 128 * case.pool.element_size())
    page[int(case.tables[1, 1]), 0, 1, 10] = 0xFF  # position 74 of sequence 1, K of head 1: NaN in both types
    got = case.run()
    group = 8
    assert got[group:, new:].isnan().all()
    got[group:, new:] = clean[group:, new:]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new,kv,heads,dim", [(2, 40, (8, 2), 128), (9, 9, (2, 2), 256), (32, 100, (2, 2), 128), (3, 300, (16, 2), 256),
                                              (40, 200, (16, 2), 128), (70, 70, (8, 8), 256), (300, 300, (4, 4), 128),
                                              (300, 1000, (16, 2), 256), (300, 1000, (32, 4), 128)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(new, kv, heads, dim, cache):
    """V of one new token has one (bf16: infinite) element that is not finite; V of another is NaN altogether."""
    case = Case([new, 1], [kv, 50], heads, dim, 64, cache, seed=18)
    clean = case.run()
    group = heads[0] // heads[1]
    one, all_ = kv - new + new // 2, kv - 1  # positions
    page = case.pool.view(torch.uint8).view(-1, 2, heads[1], 64, dim * case.pool.element_size())
    at = page[int(case.tables[0, one // 64]), 1, 0, one % 64]
    if cache == "bf16":
        at.view(torch.bfloat16)[37] = -torch.inf
    else:
        at[37] = 0x7F
    page[int(case.tables[0, all_ // 64]), 1, 1 % heads[1], all_ % 64] = 0xFF
    got = case.run()
    spoilt = torch.zeros_like(got, dtype=torch.bool)
    spoilt[:group, new // 2:new, 37] = True
    spoilt[(1 % heads[1]) * group:(1 % heads[1] + 1) * group, new - 1] = True
    assert torch.equal(~got.isfinite(), spoilt)
    assert torch.equal(got[~spoilt], clean[~spoilt])


@pytest.mark.parametrize("new,heads,dim", [(2, (8, 2), 128), (40, (16, 2), 256), (600, (16, 4), 128)])
def test_a_byte_that_is_no_scale_reaches_only_rows_that_see_it(new, heads, dim):
    case = Case([new], [700], heads, dim, 64, "scaled", seed=20)
    clean = case.run()
    case.scales.view(torch.uint8).view(-1, 2, heads[1], 64)[int(case.tables[0, 699 // 64]), :, :, 699 % 64] = 255
    assert torch.equal(case.run()[:, :new - 1], clean[:, :new - 1])


@pytest.mark.parametrize("new,heads,dim", [(2, (8, 2), 128), (7, (8, 2), 256), (40, (16, 2), 256), (60, (16, 4), 128)])
def test_a_large_value_that_a_row_does_not_see_costs_it_nothing(new, heads, dim):
    """The last token's V is 2^100 times the others': the rows before it keep their accuracy."""
    case = Case([new], [200], heads, dim, 64, "scaled", seed=19)
    clean = case.run()
    sc = case.scales.view(torch.uint8).view(-1, 2, heads[1], 64)
    sc[int(case.tables[0, 199 // 64]), 1, :, 199 % 64] += 100
    got = case.run()
    assert torch.equal(got[:, :new - 1], clean[:, :new - 1])
    assert (got[:, new - 1].float().abs().amax(-1) > 2.0 ** 60).all()


def test_strides_streams_and_views():
    """Contiguous [heads, rows, D], [rows, heads, D] seen transposed, a view of
    wider rows; on a side stream; tables as a view of wider ones."""
    case = Case([1, 90, 4], [500, 300, 44], (8, 2), 128, 64, "scaled", seed=14)
    want = case.run()
    side = torch.cuda.Stream()
    wide = torch.zeros(8, 95, 160, dtype=torch.bfloat16, device=DEV)
    wide[:, :, 32:] = case.q
    out = torch.zeros(95, 10, 128, dtype=torch.bfloat16, device=DEV)[:, 2:].transpose(0, 1)
    tables = torch.cat((torch.zeros_like(case.tables), case.tables), 1)[:, case.tables.shape[1]:]
    side.wait_stream(torch.cuda.current_stream())
    got = case.run(q=wide[:, :, 32:], out=out, block_tables=tables, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert torch.equal(case.run(q=case.q.contiguous()), want)


def test_memory_of_a_call_on_a_side_stream_is_that_streams(monkeypatch):
    """What a call allocates may not be memory that work still to run on the
    current stream uses (a freed block goes back to its own stream alone)."""
    from aws_training_study_b200.pcp_attention import paged

    seen = []
    launch = paged._launch
    monkeypatch.setattr(paged, "_launch", lambda *args: (seen.append(args), launch(*args)))
    case = Case([1, 50], [300, 200], (8, 2), 128, 64, "scaled", seed=25)
    side, status = torch.cuda.Stream(), torch.zeros(1, dtype=torch.int32, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    want = case.run(status=status).clone()
    busy = [case.run(status=status).data_ptr(), seen[-1][-3]]  # output and workspace, both free again
    out = case.run(status=status, stream=side)
    assert out.data_ptr() not in busy and seen[-1][-3] not in busy
    side.synchronize()
    assert torch.equal(out, want)
    args = (case.cfg, case.offsets, case.kv_len, case.tables, case.pool, 51, case.scales)
    busy = [t.data_ptr() for t in paged.cache_read(*args, status=status)]
    got = paged.cache_read(*args, status=status, stream=side)
    assert not {t.data_ptr() for t in got} & set(busy)
    busy = qk_norm_rope(case.q, None, torch.arange(51, device=DEV), Rotary(128))[0].data_ptr()
    side.wait_stream(torch.cuda.current_stream())
    assert qk_norm_rope(case.q, None, torch.arange(51, device=DEV), Rotary(128), stream=side)[0].data_ptr() != busy
    side.synchronize()


def test_output_over_the_queries():
    for new, kv, cache in (([1, 3, 0, 90], [700, 40, 5, 91], "scaled"), ([400, 1], [1000, 30], "bf16")):
        case = Case(new, kv, (16, 2), 128, 64, cache, seed=23)
        want = case.run()
        q = case.q.clone()
        assert case.run(q=q, out=q) is q
        assert torch.equal(q, want)


@pytest.mark.parametrize("cache", ["bf16", "scaled"])
@pytest.mark.parametrize("new,kv", [([1, 2], [900, 1500]), ([100, 1], [1500, 900])])
def test_pages_and_rows_far_into_memory(new, kv, cache):
    """Pages beyond 2^32 bytes (and elements) of the pool, heads of q and out
    2^31 elements apart: the same as a small pool, bit for bit."""
    case = Case(new, kv, (2, 2), 256, 512, cache, seed=24)
    want = case.run()
    small, scales = case.pool, case.scales
    extra = (1 << 32) // (2 * 2 * 512 * 256) + 1
    case.pool = torch.empty(small.shape[0] + extra, small.shape[1], dtype=small.dtype, device=DEV)
    case.pool.view(torch.uint8)[extra:] = small.view(torch.uint8)
    if scales is not None:
        case.scales = torch.cat((torch.full((extra, scales.shape[1]), 255, dtype=torch.uint8, device=DEV), scales))
    rows, gap = case.q.shape[1], 1 << 31
    far = torch.empty(2 * gap + gap // 2, dtype=torch.bfloat16, device=DEV)
    out = far.as_strided((2, rows, 256), (gap, 256, 1), gap // 2)
    case.q = far.as_strided((2, rows, 256), (gap, 256, 1)).copy_(case.q)
    assert torch.equal(case.run(block_tables=case.tables + extra, out=out), want)


def test_two_captured_graphs_and_new_lengths():
    """Graphs with workspaces of their own, replayed at once on two streams,
    with lengths, tables and queries that changed since the capture."""
    cases = [Case([1, 1], [600, 300], (32, 2), 256, 64, "scaled", seed=15), Case([80], [700], (32, 2), 256, 64, "scaled", seed=16)]
    graphs, outs, states = [], [], []
    for case in cases:
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        case.run(status=status)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(case.run(status=status))
        graphs.append(graph)
        states.append(status)
    cases[0].kv_len.copy_(torch.tensor([37, 299], dtype=torch.int32))
    cases[0].kv = [37, 299]
    cases[0].k, cases[0].v = ([x[b][:, :t] for b, t in enumerate(cases[0].kv)] for x in (cases[0].k, cases[0].v))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for case, out, status in zip(cases, outs, states):
        assert int(status) == 0
        case.check(out)


def test_repeatable():
    """The same call gives the same bits: no order of atomics enters."""
    case = Case([1] * 5 + [400], [5000, 100, 3, 2222, 800, 900], (32, 2), 256, 64, "scaled", seed=17)
    first = case.run()
    for _ in range(4):
        assert torch.equal(case.run(), first)


def test_reported_batches():
    """Bad pages, lengths past the table, chunks over the bound and broken
    offsets are reported, never followed; the next call is sound."""
    case = Case([1, 60], [300, 200], (16, 2), 128, 64, "scaled", seed=18)
    want = case.run()
    bad = case.tables.clone()
    bad[1, 2] = case.pool.shape[0]
    for args, code in ((dict(block_tables=bad), 109), (dict(kv_len=case.kv_len + 100000), 109),
                       (dict(max_chunk=59), 112), (dict(offsets=case.offsets.flip(0).contiguous()), 112),
                       (dict(offsets=case.offsets + 1), 112), (dict(kv_len=-case.kv_len), 112)):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        case.run(status=status, **args)
        assert int(status) == code
        with pytest.raises(PcpError, match=f"code {code}"):
            case.run(**args)
    out = case.run(max_chunk=59, out=torch.full_like(case.q, 7.0), status=torch.zeros(1, dtype=torch.int32, device=DEV))
    assert torch.equal(out[:, :1], want[:, :1]) and (out[:, 1:] == 7).all()
    assert torch.equal(case.run(), want)


def test_refusals():
    case = Case([1, 2], [30, 20], (16, 2), 128, 64, "scaled", seed=19)
    for bad in (dict(q=case.q.float()), dict(q=case.q[:8]), dict(q=case.q.cpu()), dict(out=case.q[:, :2]),
                dict(out=case.q[:1].expand(16, 3, 128)), dict(max_chunk=0), dict(offsets=case.offsets[:2]),
                dict(kv_len=case.kv_len.long()), dict(scales=case.scales[:1])):
        with pytest.raises(ValueError):
            case.run(**bad)
    with pytest.raises(PcpError, match="softmax_scale"):
        case.run(softmax_scale=-1.0)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    out = case.run(offsets=torch.zeros(1, dtype=torch.int32, device=DEV), kv_len=none, block_tables=case.tables[:0],
                   out=torch.full_like(case.q, 7.0))
    assert (out == 7).all()


@pytest.mark.parametrize("D,heads", [(256, (32, 2)), (128, (16, 4))])
def test_a_layer_step_by_step_equals_its_prompt_at_once(D, heads):
    """Norm and rotation, append and attention as a layer uses them: a prompt in
    one chunk, and the same tokens as a chunk, single tokens and a draft, give
    the same outputs up to rounding (twice the bound of one call)."""
    T, bs = 150, 16
    cfg = PCPAttentionConfig(1, 16, 4096, 4096, bs, 16, heads[0], heads[1], D)
    rotary = Rotary(D, D // 2, base=10000.0)
    g = torch.Generator(device=DEV).manual_seed(20)
    x = torch.randn(T, heads[0] + 2 * heads[1], D, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.ones(D, device=DEV, dtype=torch.bfloat16)
    blocks = -(-T // bs)
    table = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)[None]

    def serve(cuts):
        pool, scales = make_pool(cfg, blocks, device=DEV), make_scales(cfg, blocks, DEV)
        outs = []
        for a, b in zip(cuts[:-1], cuts[1:]):
            rows = x[a:b]
            q, k, v = rows.transpose(0, 1).split([heads[0], heads[1], heads[1]])
            q, k = qk_norm_rope(q, k, torch.arange(a, b, device=DEV), rotary, q_weight=w, k_weight=w)
            offsets = torch.tensor([0, b - a], dtype=torch.int32, device=DEV)
            kv_len = torch.tensor([b], dtype=torch.int32, device=DEV)
            cache_append(cfg, k, v, offsets, kv_len, table, pool, scales=scales)
            outs.append(chunk_attention(q, pool, table, offsets, kv_len, cfg, scales=scales))
        return torch.cat(outs, 1), pool, scales

    whole, pool, scales = serve([0, T])
    steps, pool2, scales2 = serve([0, 100, 101, 102, 104, T - 1, T])
    assert torch.equal(pool.view(torch.uint8), pool2.view(torch.uint8)) and torch.equal(scales, scales2)
    case = Case([T], [T], heads, D, bs, "scaled")
    case.q = qk_norm_rope(x.transpose(0, 1)[: heads[0]], None, torch.arange(T, device=DEV), rotary, q_weight=w)[0]
    page, slot = table[0, torch.arange(T, device=DEV) // bs].long(), torch.arange(T, device=DEV) % bs
    codes = pool.view(torch.uint8).view(-1, 2, heads[1], bs, D)[page, :, :, slot].view(torch.float8_e4m3fn).double()
    e = scales.view(-1, 2, heads[1], bs)[page, :, :, slot].long()
    values = codes * ((e - 127 + 1023) << 52).view(torch.float64)[..., None]
    case.k, case.v = [values[:, 0].transpose(0, 1)], [values[:, 1].transpose(0, 1)]
    case.check(whole)
    case.check(steps)
