"""Attention over a paged cache whose scales, scores and maxima go to their ends
(needs a B200), against the definition in 64 bits.

Tolerance, per element, with A = sum_j w_j |v_j| (w: the softmax's weights):
  * the output's rounding, half a step: 2^-8 |o|;
  * the weights' rounding before the second product: 2^-8 A in bf16 (bf16
    caches and bf16 copies of e4m3 ones), 2^-11 A in f16 (e4m3 caches read in
    place), where the scale is part of the weight: the largest w_j 2^e_j of a row
    is 1 or more in f16, and half of f16's least step, 2^-25, is what the others may
    lose: 2^-25 max_j (w_j 2^e_j) sum_j |code_j| over the keys that the row sees;
  * the ends of the number formats: half of bf16's least step, 2^-134, and one least
    step of fp32 for each product with 16 keys, 2^-149 (2^16 times that in a copy,
    which holds 2^-16 of the values): (1 + t / 8) 2^-134;
  * the scores: fp32 sums over D / 16 tensor-core steps, each within 2^-22 of
    the terms' magnitudes; the sum of score and exponent (below 2^9 here, so half
    a step is 2^-16) and the products with its factors; ex2 within 2^-22:
    (D / 16 * 2^-22 * max_j scale * sum_d |q_d k_jd| + 2^-15) * 2 A."""

from __future__ import annotations

import math

import pytest
import torch

from aws_training_study_b200.pcp_attention.paged import cache_append
from test_gpu_chunk_attention import CACHES, DEV, Case

pytestmark = pytest.mark.gpu

# Where a batch of `new` tokens over `kv` is computed, with eight query heads a KV head.
PATHS = [("rows", [1], [200]), ("rows", [4, 1], [700, 5000]), ("tiles", [60], [333]), ("tiles", [40, 5, 90], [900, 60, 91]),
         ("copy", [130], [200]), ("copy", [150, 1], [1100, 300])]


def two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


class Rows(Case):
    """A batch whose cached rows are set one by one; `wide` puts a table behind
    it that holds too many tokens for a copy."""

    def __init__(self, new, kv, D=128, cache="scaled", seed=0, heads=(16, 2), bs=64, wide=False):
        super().__init__(new, kv, heads, D, bs, cache, seed=seed)
        self.bs, self.wide = bs, wide
        if wide:
            tables = torch.full((len(kv), (1 << 30) // (4 * heads[1] * D * bs * len(kv)) + 1), -1, dtype=torch.int32,
                                device=DEV)
            tables[:, : self.tables.shape[1]] = self.tables
            self.tables = tables
        self.e = [torch.zeros(2, heads[1], t, dtype=torch.long, device=DEV) for t in kv]
        for b in range(len(kv)):
            self.put(b)

    def _at(self, b):
        pos = torch.arange(self.kv[b], device=DEV)
        return self.tables[b, pos // self.bs].long(), pos % self.bs

    def put(self, b, k=None, v=None, ke=None, ve=None):
        """Rows of sequence b as values over 2^e ([Hkv, t, D], [Hkv, t]); None: as they are."""
        cfg, (page, slot) = self.cfg, self._at(b)
        shape = (-1, 2, cfg.num_kv_heads, self.bs)
        rows = self.pool.view(*shape, cfg.head_dim)
        for which, (x, e) in enumerate(((k, ke), (v, ve))):
            if x is not None:
                rows.view(torch.uint8 if rows.element_size() == 1 else rows.dtype)[page, which, :, slot] = (
                    x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) if rows.element_size() == 1
                    else x.to(torch.bfloat16)).transpose(0, 1)
            if e is not None:
                self.scales.view(shape)[page, which, :, slot] = (e + 127).to(torch.uint8).T
        self.load(b)

    def load(self, b):
        """What the pages hold, in 64 bits."""
        cfg, (page, slot) = self.cfg, self._at(b)
        shape = (-1, 2, cfg.num_kv_heads, self.bs)
        codes = self.pool.view(*shape, cfg.head_dim)
        codes = codes.view(torch.uint8)[page, :, :, slot].view(codes.dtype) if codes.element_size() == 1 else \
            codes[page, :, :, slot]
        x = codes.double().permute(1, 2, 0, 3)
        if self.scales is not None:
            self.e[b] = self.scales.view(shape)[page, :, :, slot].long().permute(1, 2, 0) - 127
        x = x * two_to(self.e[b])[..., None]
        self.k[b], self.v[b] = x[0], x[1]

    def codes(self, b, which):
        return (self.k if which == 0 else self.v)[b] * two_to(-self.e[b][which])[..., None]

    def expected(self, b, scale=None):
        cfg, n, t = self.cfg, self.new[b], self.kv[b]
        scale = cfg.softmax_scale if scale is None else scale
        q = self.q[:, int(self.offsets[b]):int(self.offsets[b]) + n].double()
        group = cfg.num_q_heads // cfg.num_kv_heads
        o, bound = torch.zeros_like(q), torch.zeros_like(q)
        hidden = torch.arange(t, device=DEV) > torch.arange(t - n, t, device=DEV)[:, None]
        copied = self.cache != "bf16" and max(self.new) * group >= 1024 and n * group > 32 and not self.wide
        for h in range(cfg.num_q_heads):
            k, v = self.k[b][h // group], self.v[b][h // group]
            s = (q[h] @ k.T * scale).masked_fill(hidden, -math.inf)
            w = torch.softmax(s, -1)
            o[h] = w @ v
            a = w @ v.abs()
            terms = (q[h].abs() @ k.abs().T * scale).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
            weights = 2.0 ** -8 if self.cache == "bf16" or copied else 2.0 ** -11
            bound[h] = 2.0 ** -8 * o[h].abs() + weights * a + 2 * a * (cfg.head_dim / 16 * 2.0 ** -22 * terms + 2.0 ** -15)
            bound[h] += (1 + t / 8) * 2.0 ** -134
            if self.cache != "bf16" and not copied:
                e = self.e[b][1, h // group]
                top = (w * two_to(e)).amax(-1, keepdim=True)
                bound[h] += 2.0 ** -25 * top * ((~hidden).double() @ self.codes(b, 1)[h // group].abs())
        return o, bound


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("power", [12, 26, 40])
@pytest.mark.parametrize("path,new,kv", PATHS)
def test_a_large_value_of_no_weight_costs_nothing(path, new, kv, power, D):
    """Visible keys whose score is 60 log2 units below the others' and whose V is
    2^power times theirs: less than half a step of the output, and no more than
    that for the others' weights."""
    case = Rows(new, kv, D, seed=power)
    u = torch.where(torch.rand(D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) < 0.5, -1.0, 1.0)
    case.q = (case.q * 0.25 + u).to(torch.bfloat16)
    low = 60 * math.log(2) * math.sqrt(D) / D
    for b, t in enumerate(kv):
        at = torch.arange(min(5, t - new[b]), t - new[b] + 1, 97, device=DEV)
        k, e = case.codes(b, 0), case.e[b].clone()
        k -= (k @ u.double())[..., None] / D * u.double()  # nothing along u but in those keys
        e[0], e[1] = 0, torch.randint(-3, 1, e[1].shape, device=DEV)
        k[:, at] = -u.double() * low
        e[1][:, at] = power
        case.put(b, k=k, ke=e[0], ve=e[1])
    case.check(case.run())


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("exponents", [(120,), (-100,), (-100, 120), (-100, -60, 0, 60, 120)])
@pytest.mark.parametrize("path,new,kv", PATHS)
def test_exponents_that_an_append_may_write(path, new, kv, exponents, D):
    """V's scales at the ends of what is written (bytes 27 and 247), alone and
    mixed, under weights that fall off over many powers of two."""
    case = Rows(new, kv, D, seed=len(exponents))
    g = torch.Generator(device=DEV).manual_seed(2)
    for b in range(len(kv)):
        pick = torch.randint(len(exponents), case.e[b][1].shape, device=DEV, generator=g)
        case.put(b, ke=torch.full_like(case.e[b][0], 1), ve=torch.tensor(exponents, device=DEV)[pick])
    case.check(case.run())
    case.check(case.run(softmax_scale=0.5), scale=0.5)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("where", ["seen by all", "seen by some"])
@pytest.mark.parametrize("path,new,kv", PATHS)
def test_values_that_round_up_to_2_128(path, new, kv, where, D):
    """An appended element of 255 * 2^120 is stored as 256 * 2^120: finite in the
    cache, too large for bf16.  The rows that see it get its weight times 2^128."""
    case = Rows(new, kv, D, seed=4)
    b = 0
    pos = 7 if where == "seen by all" else kv[b] - new[b] + new[b] // 2
    v = torch.zeros(2, 1, D, dtype=torch.bfloat16, device=DEV)
    v[:, :, 37] = 255 * 2.0 ** 120
    k = torch.zeros_like(v)  # of score 0, as every key's is about
    offsets = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    cache_append(case.cfg, k, v, offsets, torch.tensor([pos + 1], dtype=torch.int32, device=DEV), case.tables[b:b + 1],
                 case.pool, scales=case.scales)
    case.load(b)
    assert float(case.v[b][0, pos, 37]) == 2.0 ** 128
    out = case.run()
    want, bound = case.expected(b)
    got = out[:, :new[b]].double()
    most = float(torch.finfo(torch.bfloat16).max)
    fits = want.abs() + bound < most  # (bf16 has nothing for the rest)
    assert int(fits.sum()) > 0.99 * fits.numel() and (got[fits].isfinite()).all()
    bad = fits & ~((got - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} beyond the bound"
    assert (got[:, :, 37].abs() > 2.0 ** 100).sum() == (want[:, :, 37].abs() > 2.0 ** 100).sum() > 0


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("power", [110, -100])
@pytest.mark.parametrize("path,new,kv", PATHS)
def test_keys_of_any_size(path, new, kv, power, D):
    """K far from unit size, with queries that bring the scores back."""
    case = Rows(new, kv, D, seed=3)
    for b in range(len(kv)):
        case.put(b, ke=case.e[b][0].clamp(-4, 1) + power)
    case.q = (case.q.float() * 2.0 ** -power).to(torch.bfloat16)
    case.check(case.run())


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,D", [((16, 2), 128), ((16, 2), 256), ((7, 7), 128)])
@pytest.mark.parametrize("new,kv,wide", [([1], [4000], False), ([2, 1], [1500, 9000], False), ([60], [1500], False),
                                         ([150, 33], [2100, 700], False), ([150, 33], [2100, 700], True)])
def test_maxima_that_grow_with_every_tile(new, kv, wide, heads, D, cache):
    """Scores that grow by 12 log2 units with every 128 keys for half of the
    queries, and stay for the others: O goes over to a new reference tile by tile."""
    case = Rows(new, kv, D, cache, seed=5, heads=heads, wide=wide)
    u = torch.where(torch.rand(D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) < 0.5, -1.0, 1.0)
    grows = torch.arange(case.q.shape[1], device=DEV)[None, :, None] + torch.arange(heads[0], device=DEV)[:, None, None]
    case.q = (case.q * 0.25 + u * (grows % 2)).to(torch.bfloat16)
    for b, t in enumerate(kv):
        x = torch.randn(heads[1], t, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(b)).double()
        x += (torch.arange(t, device=DEV) // 128)[:, None] * (12 * math.log(2) / math.sqrt(D)) * u.double()
        case.put(b, k=x, ke=torch.zeros_like(case.e[b][0]) if cache == "scaled" else None)
    case.check(case.run())


@pytest.mark.parametrize("cache", ["e4m3", "scaled"])
@pytest.mark.parametrize("heads,D", [((16, 2), 128), ((32, 2), 256), ((20, 4), 128)])
@pytest.mark.parametrize("new,kv", [([300], [1500]), ([130, 1, 400, 7], [130, 900, 3001, 64])])
def test_long_chunks_without_room_for_a_copy(new, kv, heads, D, cache):
    """Units of many tiles over an e4m3 cache read in place."""
    case = Rows(new, kv, D, cache, seed=6, heads=heads, wide=True)
    case.check(case.run())
