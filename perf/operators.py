"""The serving operators of one attention layer, as they are measured: their plain forms, the framework's
calls of the same operators, and the cases.

* ``qk_norm_rope`` -- RMS norm of every query and key head, and the position rotation, in one pass.
* ``cache`` -- new tokens' keys and values appended to a paged cache (e4m3 codes with a power-of-two scale for
  each token and head, or bf16), and tokens of the cache read back.
* ``chunk_attention`` -- causal attention of each sequence's new tokens over its paged cache.

Sequences share one convention: ``offsets[b] .. offsets[b + 1]`` are the rows of sequence b's tokens in a packed
``[heads, rows, head_dim]`` tensor, and they are the last tokens of its ``kv_len[b]`` tokens.
"""

import json
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
E4M3_MAX = 448.0


# ------------------------------------------------------------------ cases --
def listed():
    rope = {"op": "qk_norm_rope", "q_heads": 32, "kv_heads": 2, "head_dim": 256, "rotary_dim": 64, "layout": "half",
            "scaling": "none", "norm": True, "dtype": "bf16", "far": 131072}
    cache = {"op": "cache", "kv_heads": 2, "head_dim": 256, "block": 512, "dtype": "e4m3", "read": "new"}
    attn = {"op": "chunk_attention", "q_heads": 32, "kv_heads": 2, "head_dim": 256, "block": 512, "dtype": "e4m3",
            "scaled": True, "decodes": 0, "padding": 0}
    return [
        # One decode step of a batch of 16: latency.
        dict(rope, name="rope decode 16", tokens=16),
        # A prefill chunk of the full preset (4096 current tokens, 32 / 2 heads of 256, a quarter rotated).
        dict(rope, name="rope prefill 4096", tokens=4096),
        # Many heads of 128 rotated whole, interleaved pairs, positions far past the trained length.
        dict(rope, name="rope long 8191", tokens=8191, q_heads=64, kv_heads=8, head_dim=128, rotary_dim=128,
             layout="interleaved", scaling="ramp", far=500000),
        # One decode step of 32 sequences: a token each is appended and read back.
        dict(cache, name="cache decode 32", seqs=32, new=1, history=8192),
        # A prefill chunk appended (in 64-token pages) and read back, several sequences of odd lengths.
        dict(cache, name="cache prefill 5 x 1000", seqs=5, new=1000, history=4000, block=64, kv_heads=8, head_dim=128),
        # A long cache read back whole after a chunk was appended to it (30001 tokens, as the ragged workload).
        dict(cache, name="cache read 30001", seqs=1, new=513, history=29488, read="all"),
        # A single short sequence's decode step: latency.
        dict(attn, name="decode 1 x 500", seqs=1, chunk=1, history=500),
        # A batch of decode steps over long ragged caches: bandwidth.
        dict(attn, name="decode 16 x 32768", seqs=16, chunk=1, history=32768, decodes=16),
        # The same with bf16 caches, heads of 128 and four queries a KV head, small pages.
        dict(attn, name="decode 64 x 4096 bf16", seqs=64, chunk=1, history=4096, decodes=64, q_heads=32, kv_heads=8,
             head_dim=128, block=64, dtype="bf16", scaled=False),
        # One long prompt's next chunk over 131072 cached tokens.
        dict(attn, name="chunk 512 over 131072", seqs=1, chunk=512, history=131072),
        # A mixed step: most sequences decode, three bring a chunk of prompt; padding rows behind them.
        dict(attn, name="mixed 24 + 3", seqs=27, chunk=700, history=6000, decodes=24, padding=5),
        # Whole prompts of different lengths packed together, nothing cached before them.
        dict(attn, name="prompts 4 x 2048 bf16", seqs=4, chunk=2048, history=0, q_heads=64, kv_heads=8, head_dim=128,
             block=128, dtype="bf16", scaled=False),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "cache", "chunk_attention", "chunk_attention"])
    kv_heads, group = rng.choice([(1, 8), (2, 16), (2, 5), (4, 8), (8, 4), (8, 8), (8, 1), (3, 7)])
    head_dim = rng.choice([128, 256])
    if op == "qk_norm_rope":
        head_dim = rng.choice([64, 96, 128, 256])
        tokens = _spread(rng, 1, 8191)
        return {"op": op, "tokens": tokens, "q_heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim,
                "rotary_dim": rng.choice([16, head_dim // 2, head_dim]),
                "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "bands", "ramp"]), "norm": rng.random() < 0.7,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "far": _spread(rng, 4096, 1000000)}
    block = rng.choice([16, 48, 64, 128, 512])
    dtype = rng.choice(["e4m3", "e4m3", "bf16"])
    if op == "cache":
        seqs = _spread(rng, 1, 64)
        new = _spread(rng, 1, max(1, 8000 // seqs))
        return {"op": op, "seqs": seqs, "new": new, "history": _spread(rng, 1, max(2, 30000 // seqs)),
                "kv_heads": kv_heads, "head_dim": head_dim, "block": block, "dtype": dtype,
                "read": rng.choice(["new", "all"])}
    case = {"op": op, "q_heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim, "block": block,
            "dtype": dtype, "scaled": dtype == "e4m3" and rng.random() < 0.8, "padding": rng.choice([0, 0, 3, 17])}
    kind = rng.choice(["decode", "chunk", "mixed"])
    if kind == "decode":
        seqs = _spread(rng, 1, 64)
        # up to four tokens a sequence, as when drafted tokens are checked
        return dict(case, seqs=seqs, chunk=rng.choice([1, 1, 2, 3, 4]), decodes=rng.choice([0, seqs]),
                    history=_spread(rng, 1, max(2, 500000 // seqs // kv_heads)))
    if kind == "chunk":
        seqs = rng.choice([1, 1, 2, 3, 5])
        chunk = _spread(rng, 2, max(3, 4096 // seqs // kv_heads))
        return dict(case, seqs=seqs, chunk=chunk, decodes=0, history=_spread(rng, 1, max(2, 40000 // seqs)))
    seqs = _spread(rng, 3, 40)
    return dict(case, seqs=seqs, chunk=_spread(rng, 16, 600), decodes=seqs - rng.choice([1, 2, 3]),
                history=_spread(rng, 16, 8000))


def _lengths(case):
    """New tokens and cached tokens (the new ones included) of every sequence: the first one that brings a chunk has
    the case's largest sizes, the others are ragged, by the case alone."""
    rng = random.Random(json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True))
    largest = case["new"] if case["op"] == "cache" else case["chunk"]
    decodes = case.get("decodes", 0)
    new, kv = [], []
    for b in range(case["seqs"]):
        first = b == (decodes if decodes < case["seqs"] else 0)
        n = 1 if b < decodes else largest if first else rng.randint((largest + 1) // 2, largest)
        h = case["history"] if first else rng.randint(case["history"] // 4, case["history"])
        new.append(n)
        kv.append(n + h)
    return new, kv


def work(case):
    D = case["head_dim"]
    if case["op"] == "qk_norm_rope":
        heads = case["q_heads"] + case["kv_heads"]
        elt = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["tokens"] * (2 * heads * D * elt + 8),
                "flops": case["tokens"] * heads * ((4 * D if case["norm"] else 0) + 3 * case["rotary_dim"])}
    new, kv = _lengths(case)
    row = D + 1 if case["dtype"] == "e4m3" and case.get("scaled", True) else D if case["dtype"] == "e4m3" else 2 * D
    Hkv = case["kv_heads"]
    if case["op"] == "cache":
        read = sum(new if case["read"] == "new" else kv)
        return {"bytes": 2 * Hkv * (sum(new) * (2 * D + row) + read * (row + 2 * D)),
                "flops": 2 * Hkv * D * (2 * sum(new) + read)}
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, kv))
    return {"bytes": 2 * 2 * sum(new) * case["q_heads"] * D + 2 * Hkv * sum(kv) * row,
            "flops": 4 * case["q_heads"] * D * pairs}


# ----------------------------------------------------------------- inputs --
SCALING = {"linear": {"factor": 8.0}, "bands": {"factor": 8.0, "original_len": 8192, "low": 1.0, "high": 4.0},
           "ramp": {"factor": 16.0, "original_len": 32768, "low": 1.0, "high": 32.0}}
BASE = 1000000.0


def _inverse_frequencies(case):
    """The angle a position of every rotated pair, in 64 bits, and what scales the rotated pairs."""
    r = case["rotary_dim"]
    f = BASE ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    s = SCALING.get(case["scaling"])
    if s is None:
        return f, 1.0
    if case["scaling"] == "linear":
        return f / s["factor"], 1.0
    if case["scaling"] == "bands":  # by wavelengths in the trained length
        turns = s["original_len"] * f / (2 * math.pi)
        keep = ((turns - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        return f * (keep + (1 - keep) / s["factor"]), 1.0
    # by the pair's index, between those that make `high` and `low` turns in the trained length
    at = [r * math.log(s["original_len"] / (2 * math.pi * t)) / (2 * math.log(BASE)) for t in (s["high"], s["low"])]
    first, last = max(0, math.floor(at[0])), min(r - 1, math.ceil(at[1]))
    far = ((torch.arange(r // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0, 1)
    return f * (1 - far + far / s["factor"]), 0.1 * math.log(s["factor"]) + 1.0


def _config(case, blocks):
    from aws_training_study_b200.pcp_attention import PCPAttentionConfig

    longest = blocks * case["block"]
    return PCPAttentionConfig(1, 16, longest, longest, case["block"], 16, case.get("q_heads", case["kv_heads"]),
                              case["kv_heads"], case["head_dim"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    D = case["head_dim"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    s = {"case": case}
    if case["op"] == "qk_norm_rope":
        t = TYPES[case["dtype"]]
        T = case["tokens"]
        # as projections leave them: [tokens, heads, head_dim], seen as [heads, tokens, head_dim]
        s["q"] = normal(T, case["q_heads"], D, scale=2.0).to(t).transpose(0, 1)
        s["k"] = normal(T, case["kv_heads"], D, scale=2.0).to(t).transpose(0, 1)
        s["positions"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda")
        s["q_weight"] = (1 + normal(D, scale=0.2)).to(t) if case["norm"] else None
        s["k_weight"] = (1 + normal(D, scale=0.2)).to(t) if case["norm"] else None
        f, s["magnitude"] = _inverse_frequencies(case)
        s["frequencies"] = f.cuda()
        if own:
            from aws_training_study_b200.pcp_attention.rotary import Rotary

            s["rotary"] = Rotary(D, case["rotary_dim"], base=BASE, layout=case["layout"],
                                 scaling=None if case["scaling"] == "none" else case["scaling"],
                                 **SCALING.get(case["scaling"], {}))
        return s

    new, kv = _lengths(case)
    block, Hkv, e4m3 = case["block"], case["kv_heads"], case["dtype"] == "e4m3"
    rows = sum(new) + case.get("padding", 0)
    s["rows"], s["longest_new"], s["longest"] = rows, max(new), max(kv)

    def offsets(n):
        return torch.tensor([0] + n, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()

    s["offsets"], s["kv_len"] = offsets(new), torch.tensor(kv, dtype=torch.int32).cuda()
    width = max(-(-t // block) for t in kv)
    blocks = sum(-(-t // block) for t in kv)
    # pages in no order, the table's unused entries at page 0
    order = torch.randperm(blocks + 2, generator=g, device="cuda")[:blocks].to(torch.int32)
    used = torch.arange(width, device="cuda")[None, :] * block < s["kv_len"][:, None]
    s["tables"] = torch.zeros((len(kv), width), dtype=torch.int32, device="cuda")
    s["tables"][used] = order
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    shape = (blocks + 2, 2, Hkv, block)
    scaled = e4m3 and case.get("scaled", True)
    s["scales"] = None
    if case["op"] == "cache" and not e4m3 or case["op"] == "chunk_attention" and not e4m3:
        s["pool"] = normal(*shape, D, scale=0.5).to(torch.bfloat16).reshape(blocks + 2, -1)
    else:
        # codes over the range that scaled rows take; exponents that differ from token to token
        s["pool"] = normal(*shape, D, scale=100.0 if scaled else 0.5).clamp(-448, 448).to(torch.float8_e4m3fn)
        s["pool"] = s["pool"].reshape(blocks + 2, -1)
        if scaled:
            e = torch.randint(117, 121, shape, generator=g, device="cuda", dtype=torch.uint8)
            s["scales"] = e.reshape(blocks + 2, -1)
    if case["op"] == "cache":
        # heads of very different sizes, tokens too
        size = torch.exp2(torch.randint(-6, 4, (rows, Hkv, 1), generator=g, device="cuda").float())
        s["k"] = (normal(rows, Hkv, D) * size).to(torch.bfloat16).transpose(0, 1)
        s["v"] = (normal(rows, Hkv, D) * size).to(torch.bfloat16).transpose(0, 1)
        s["read"] = s["offsets"] if case["read"] == "new" else offsets(kv)
        s["tokens"] = sum(new if case["read"] == "new" else kv)
        s["longest_read"] = max(new if case["read"] == "new" else kv)
    else:
        s["q"] = normal(rows, case["q_heads"], D).to(torch.bfloat16).transpose(0, 1)
        s["out"] = torch.zeros((rows, case["q_heads"], D), dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    if own:
        s["config"] = _config(case, width)
    return s


# ------------------------------------------------------------ plain forms --
def _plain_norm_rope(s):
    case = s["case"]
    r = case["rotary_dim"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos = (angle.cos() * s["magnitude"]).float()
    sin = (angle.sin() * s["magnitude"]).float()

    def one(x, weight):
        y = x.float()
        if weight is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
        a, b = (y[..., : r // 2], y[..., r // 2 : r]) if case["layout"] == "half" else (y[..., 0:r:2], y[..., 1:r:2])
        c, d = a * cos - b * sin, b * cos + a * sin
        turned = torch.cat((c, d), -1) if case["layout"] == "half" else torch.stack((c, d), -1).flatten(-2)
        return torch.cat((turned, y[..., r:]), -1).to(x.dtype)

    return {"q": one(s["q"], s["q_weight"]), "k": one(s["k"], s["k_weight"])}


def _places(offsets, kv_len, rows):
    """Sequence and position of each packed row that belongs to a sequence (the last rows of its tokens)."""
    row = torch.arange(rows, device=offsets.device)
    seq = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp(max=offsets.numel() - 2)
    return seq, kv_len[seq] - offsets[seq + 1] + row


def _pages(s):
    case = s["case"]
    return s["pool"].view(-1, 2, case["kv_heads"], case["block"], case["head_dim"])


def _power(e):
    """2^e in 32 bits, exactly, for whole e of -126 to 127 (exp2 may be a rounding off, which would break ties)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _exponents(s):
    case = s["case"]
    return _power(s["scales"].view(-1, 2, case["kv_heads"], case["block"]).int() - 127)


def _plain_cache(s):
    case = s["case"]
    block, D = case["block"], case["head_dim"]
    pages = _pages(s)
    seq, pos = _places(s["offsets"], s["kv_len"], s["rows"])
    page, slot = s["tables"][seq, pos // block].long(), pos % block
    for which, x in enumerate((s["k"], s["v"])):
        x = x.transpose(0, 1)  # [rows, heads, head_dim]
        if s["scales"] is None:
            pages[page, which, :, slot] = x
            continue
        y = x.float()
        m, e = torch.frexp(y.abs().amax(-1))
        e = torch.where(m > 0.875, e - 8, e - 9)  # least e with amax <= 448 * 2^e
        e = torch.where(m == 0, torch.zeros_like(e), e.clamp(-100, 120))
        codes = (y * _power(-e)[..., None]).to(torch.float8_e4m3fn)
        pages.view(torch.uint8)[page, which, :, slot] = codes.view(torch.uint8)
        s["scales"].view(-1, 2, case["kv_heads"], block)[page, which, :, slot] = (e + 127).to(torch.uint8)
    seq, pos = _places(s["read"], s["kv_len"], s["tokens"])
    page, slot = s["tables"][seq, pos // block].long(), pos % block
    out = {}
    for which, name in enumerate("kv"):
        y = pages.view(torch.uint8)[page, which, :, slot].view(pages.dtype) if s["scales"] is not None else pages[page, which, :, slot]
        y = y.float()
        if s["scales"] is not None:
            y = y * _exponents(s)[page, which, :, slot][..., None]
        out[name] = y.to(torch.bfloat16).transpose(0, 1)
    return out


def _plain_attention(s):
    case = s["case"]
    Hq, Hkv, D, B = case["q_heads"], case["kv_heads"], case["head_dim"], s["kv_len"].numel()
    tables = s["tables"].long()

    def gathered(which):  # [B, Hkv, longest, D]
        if s["scales"] is not None:
            y = _pages(s).view(torch.uint8)[tables, which].view(torch.float8_e4m3fn).float()
            y = y * _exponents(s)[tables, which][..., None]
        elif case["dtype"] == "e4m3":
            y = _pages(s).view(torch.uint8)[tables, which].view(torch.float8_e4m3fn).float()
        else:
            y = _pages(s)[tables, which].float()
        return y.permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)[:, :, : s["longest"]]

    n = s["longest_new"]
    first, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    row = first[:, None] + torch.arange(n, device="cuda")  # [B, n], past the end for shorter chunks
    live = row < end[:, None]
    q = s["q"][:, row.clamp(max=s["rows"] - 1)].float()  # [Hq, B, n, D]
    q = q.reshape(Hkv, Hq // Hkv, B, n, D).permute(2, 0, 1, 3, 4).reshape(B, Hkv, -1, D)
    p = (q @ gathered(0).transpose(-1, -2)).mul_(1 / math.sqrt(D))  # [B, Hkv, group * n, longest]
    last = s["kv_len"].long()[:, None] - end[:, None] + row  # last visible position
    hidden = torch.arange(s["longest"], device="cuda") > last[..., None]
    p.view(B, Hkv, -1, n, s["longest"]).masked_fill_(hidden[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = (p @ gathered(1)).div_(p.sum(-1, keepdim=True))
    o = o.reshape(B, Hq, n, D).transpose(0, 1).to(torch.bfloat16)
    out = torch.zeros_like(s["q"])
    out[:, row[live]] = o[:, live]
    return {"out": out}


# -------------------------------------------------------------------- run --
def run(s):
    op = s["case"]["op"]
    if not own:
        return {"qk_norm_rope": _plain_norm_rope, "cache": _plain_cache, "chunk_attention": _plain_attention}[op](s)
    if op == "qk_norm_rope":
        from aws_training_study_b200.pcp_attention.rotary import qk_norm_rope

        q, k = qk_norm_rope(s["q"], s["k"], s["positions"], s["rotary"], q_weight=s["q_weight"],
                            k_weight=s["k_weight"], eps=EPS)
        return {"q": q, "k": k}
    from aws_training_study_b200.pcp_attention.paged import cache_append, cache_read, chunk_attention

    if op == "cache":
        cache_append(s["config"], s["k"], s["v"], s["offsets"], s["kv_len"], s["tables"], s["pool"],
                     scales=s["scales"], status=s["status"])
        k, v = cache_read(s["config"], s["read"], s["kv_len"], s["tables"], s["pool"], s["tokens"],
                          scales=s["scales"], status=s["status"])
        return {"k": k, "v": v}
    out = chunk_attention(s["q"], s["pool"], s["tables"], s["offsets"], s["kv_len"], s["config"], scales=s["scales"],
                          max_chunk=s["longest_new"], out=s["out"], status=s["status"])
    return {"out": out}


# ------------------------------------------------- definitions in 64 bits --
def _two_to(e):
    """2^e in 64 bits from its bits, for whole e: pow may be a rounding off."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(x):
    """Nearest e4m3 value of a 64-bit one, ties to even: steps of 2^-9, or an eighth of the power of two below."""
    power = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -40)))
    power = torch.where(_two_to(power) > x.abs(), power - 1, power)
    power = torch.where(_two_to(power + 1) <= x.abs(), power + 1, power)
    step = _two_to(power.clamp(min=-6) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    D = case["head_dim"]
    if case["op"] == "qk_norm_rope":
        r = case["rotary_dim"]
        pair = torch.arange(r // 2, device="cuda")
        f, magnitude = _inverse_frequencies(case)
        turn = torch.polar(torch.full((case["tokens"], r // 2), magnitude, dtype=torch.float64, device="cuda"),
                           torch.outer(s["positions"].double(), f.cuda()))
        one, two = (pair, pair + r // 2) if case["layout"] == "half" else (2 * pair, 2 * pair + 1)
        out = {}
        for name in "qk":
            y = s[name].double()
            w = s[name + "_weight"]
            if w is not None:
                y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / D + EPS) * w.double()
            z = torch.complex(y[..., one], y[..., two]) * turn
            y = y.clone()
            y[..., one], y[..., two] = z.real, z.imag
            out[name] = y
        return out

    new, kv = _lengths(case)
    block, Hkv = case["block"], case["kv_heads"]
    pages = s["pool"].view(-1, 2, Hkv, block, D)
    if case["op"] == "cache":
        starts = [sum(new[:b]) for b in range(len(new))]
        got = {"k": [], "v": []}
        for b in range(len(new)):
            page = s["tables"][b, : -(-kv[b] // block)].long()
            for which, name in enumerate("kv"):
                old = pages.view(torch.uint8)[page, which].view(pages.dtype) if s["scales"] is not None else pages[page, which]
                old = old.double()
                x = s[name][:, starts[b] : starts[b] + new[b]].double()
                if s["scales"] is not None:
                    old = old * _two_to(s["scales"].view(-1, 2, Hkv, block)[page, which].long() - 127)[..., None]
                    size = x.abs().amax(-1, keepdim=True)
                    e = torch.ceil(torch.log2((size / E4M3_MAX).clamp(min=2.0 ** -100)))
                    e = torch.where(size > E4M3_MAX * _two_to(e), e + 1, e)
                    e = torch.where(size <= E4M3_MAX * _two_to(e - 1), e - 1, e).clamp(-100, 120)
                    x = _round_e4m3(x / _two_to(e)) * _two_to(e)
                whole = torch.cat((old.transpose(0, 1).reshape(Hkv, -1, D)[:, : kv[b] - new[b]], x), 1)
                got[name].append(whole[:, kv[b] - new[b] :] if case["read"] == "new" else whole)
        return {name: torch.cat(x, 1) for name, x in got.items()}

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, start = case["q_heads"] // Hkv, 0
    for b in range(len(new)):
        page = s["tables"][b, : -(-kv[b] // block)].long()
        for h in range(Hkv):
            both = []
            for which in range(2):
                x = pages.view(torch.uint8)[page, which, h].view(pages.dtype) if case["dtype"] == "e4m3" else pages[page, which, h]
                x = x.double()
                if s["scales"] is not None:
                    x = x * _two_to(s["scales"].view(-1, 2, Hkv, block)[page, which, h].long() - 127)[..., None]
                both.append(x.reshape(-1, D)[: kv[b]])
            seen = torch.ones(new[b], kv[b], dtype=torch.bool, device="cuda").tril(kv[b] - new[b])
            for head in range(h * group, (h + 1) * group):
                score = s["q"][head, start : start + new[b]].double() @ both[0].T / math.sqrt(D)
                weight = torch.where(seen, torch.exp(score - score.masked_fill(~seen, -math.inf).amax(1, keepdim=True)), 0.0)
                out[head, start : start + new[b]] = (weight / weight.sum(1, keepdim=True)) @ both[1]
        start += new[b]
    return {"out": out}
