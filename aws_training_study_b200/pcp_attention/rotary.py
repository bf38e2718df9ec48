"""Norm and position rotation of query and key heads, in one pass.

The reference takes queries and keys that a layer has already prepared
(``run_poc.py:81-134`` draws them); a layer that serves them first norms every
head and rotates it by its token's position.  ``qk_norm_rope`` does both for q
and k in one kernel:

    y = x * rsqrt(mean(x^2) + eps) * weight                (with a weight)
    (a, b) -> magnitude * (a cos t - b sin t, b cos t + a sin t)
    t = position * frequency[i]      for pair i of the first rotary_dim elements

computed in fp32 and rounded once.  ``Rotary`` holds what the rotation needs.
The angle is made on the device from the position and the pair's turns per
position as a 64-bit fraction, so whole turns fall away exactly: there is no
cos/sin table, and positions of any size are as exact as small ones.
"""

from __future__ import annotations

import math

import torch

from .. import _capi

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # enum pcp_float_dtype
_LAYOUTS = {"half": 0, "interleaved": 1}                           # enum pcp_rotary_layout
SCALINGS = ("linear", "bands", "ramp")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_len: int | None = None, low: float = 1.0,
                       high: float | None = None) -> tuple[list[float], float]:
    """The angle per position of each of the ``rotary_dim / 2`` pairs, and the
    magnitude of the rotated pairs.

    ``base ** (-2 i / rotary_dim)`` for pair i, stretched for contexts
    ``factor`` times the trained ``original_len``:

    * ``None``: as it is.
    * ``"linear"``: every frequency divided by ``factor``.
    * ``"bands"``: by the turns a pair makes in ``original_len``: ``high``
      (default 4) or more keep their frequency, ``low`` or fewer are divided by
      ``factor``, those between are blended linearly in their turns.
    * ``"ramp"``: the same with the blend linear in the pair's index, between
      the pairs that make ``high`` (default 32) and ``low`` turns (rounded
      outwards), and the magnitude ``0.1 ln(factor) + 1``.
    """
    f = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling is None:
        return f, 1.0
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be None or one of {SCALINGS}, got {scaling!r}")
    if not factor > 0:
        raise ValueError(f"factor must be positive, got {factor}")
    if scaling == "linear":
        return [x / factor for x in f], 1.0
    if original_len is None or original_len <= 0:
        raise ValueError(f"scaling {scaling!r} needs the trained original_len")
    high = high if high is not None else (4.0 if scaling == "bands" else 32.0)
    if not 0 < low < high:
        raise ValueError(f"needs 0 < low < high, got {low}, {high}")
    if scaling == "bands":
        def keep(x: float) -> float:
            return min(max((original_len * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0)

        return [x * (keep(x) + (1 - keep(x)) / factor) for x in f], 1.0

    def pair_with(turns: float) -> float:
        return rotary_dim * math.log(original_len / (2 * math.pi * turns)) / (2 * math.log(base))

    first, last = max(0, math.floor(pair_with(high))), min(rotary_dim - 1, math.ceil(pair_with(low)))
    out = []
    for i, x in enumerate(f):
        far = min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0)
        out.append(x * (1 - far + far / factor))
    return out, 0.1 * math.log(factor) + 1.0


def _capturing(stream: torch.cuda.Stream | None) -> bool:
    """Whether the current stream is being captured, or the one a call was given."""
    if torch.cuda.is_current_stream_capturing():
        return True
    if stream is None:
        return False
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


class Rotary:
    """The rotation of the first ``rotary_dim`` (default all) elements of heads
    of ``head_dim``: ``layout`` ``"half"`` pairs i with i + rotary_dim / 2,
    ``"interleaved"`` 2 i with 2 i + 1; the frequencies are those of
    ``rotary_frequencies``.  ``rotary_dim`` 0 is a norm without rotation."""

    def __init__(self, head_dim: int, rotary_dim: int | None = None, base: float = 10000.0, layout: str = "half",
                 scaling: str | None = None, **scaling_args):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim <= 0 or head_dim % 16 or head_dim > 512:
            raise ValueError(f"head_dim must be a multiple of 16 up to 512, got {head_dim}")
        if rotary_dim < 0 or rotary_dim % 16 or rotary_dim > head_dim:
            raise ValueError(f"rotary_dim must be a multiple of 16 up to head_dim {head_dim}, got {rotary_dim}")
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}, got {layout!r}")
        if not base > 1:
            raise ValueError(f"base must be above 1, got {base}")
        self.head_dim, self.rotary_dim, self.layout = head_dim, rotary_dim, layout
        self.frequencies, self.magnitude = rotary_frequencies(rotary_dim, base, scaling, **scaling_args)
        # Turns per position as a fraction of 2^64, in the bits of an int64.
        turns = [round(f * (2.0 ** 64 / (2 * math.pi))) % 2 ** 64 for f in self.frequencies]
        self._turns_host = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64)
        self._turns: dict[torch.device, torch.Tensor] = {}

    def turns(self, device: torch.device, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """The pairs' turns on ``device`` (copied there once; before any graph
        capture that uses them, on the current stream or ``stream``)."""
        t = self._turns.get(device)
        if t is None:
            if _capturing(stream):
                raise RuntimeError("the rotation's table is not on this device yet: call once before the capture")
            t = self._turns[device] = self._turns_host.to(device)
        return t


def _heads(t: torch.Tensor | None) -> _capi.PcpHeads:
    if t is None:
        return _capi.PcpHeads(0, 0, 0, 0, 0)
    heads, rows, _ = t.shape
    head, row, _ = t.stride()
    # an axis of one has no step to check
    return _capi.PcpHeads(t.data_ptr(), head if heads > 1 else 0, row if rows > 1 else 0, heads, 0)


def _check_rows(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device) -> _capi.PcpHeads:
    """A packed tensor ``[heads, rows, head_dim]`` whose rows are contiguous
    and 16-byte aligned; the heads and rows may lie at any stride.  Returns it
    as the C ABI takes it."""
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"expected {name} {shape} {dtype}, got {tuple(t.shape)} {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    head, row, one = t.stride()
    heads, rows, _ = shape
    head, row = head if heads > 1 else 0, row if rows > 1 else 0  # an axis of one has no step to check
    data, unit = t.data_ptr(), 4 if dtype == torch.float32 else 8
    if heads and rows and (one != 1 or data % 16 or head % unit or row % unit):
        raise ValueError(f"{name} needs contiguous, 16-byte aligned rows, got strides {t.stride()}")
    return _capi.PcpHeads(data, head, row, heads, 0)


def _check_writable(name: str, t: torch.Tensor) -> None:
    """An output's rows may not lie on one another."""
    heads, rows, reach = t.shape
    head, row, _ = t.stride()
    for stride, n in ((head, heads), (row, rows)) if head < row else ((row, rows), (head, heads)):
        if n > 1:
            if stride < reach:
                raise ValueError(f"{name} overlaps itself: strides {t.stride()}")
            reach += stride * (n - 1)


def _check_apart(name: str, t: torch.Tensor | None, other: str, o: torch.Tensor | None) -> None:
    """An output may not be another tensor of the call over again."""
    if t is not None and o is not None and t.numel() and o.numel() and t.data_ptr() == o.data_ptr():
        raise ValueError(f"{name} and {other} are the same memory")


def _allocate(stream: torch.cuda.Stream, make, *args, **kwargs) -> torch.Tensor:
    """``make(...)`` with memory of ``stream``, for a call that was given one: a
    block that the current stream freed may still be in use by work it has yet to
    run."""
    with torch.cuda.stream(stream):
        return make(*args, **kwargs)


def _launch(device: torch.device, stream: torch.cuda.Stream | None, entry, *args) -> None:
    """``entry(*args, stream)`` on ``device`` and ``stream`` (default: the
    current one of the device); raises its error.  The device and stream are
    read without torch.cuda's wrappers, which cost a small call more host time
    than everything else in it."""
    index = device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return _launch(device, stream, entry, *args)
    _capi.check(entry(*args, stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(index)))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, rotary: Rotary,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Norms (with ``q_weight`` / ``k_weight``, ``[head_dim]``) and rotates the
    heads of ``q`` ``[Hq, rows, head_dim]`` and ``k`` ``[Hkv, rows, head_dim]``
    (or None) by ``positions`` ``[rows]`` (int32 or int64).  bf16, fp16 or
    fp32, weights of the same type; heads and rows at any 16-byte aligned
    stride, so ``[rows, heads, head_dim]`` projections are passed transposed.
    ``q_out``/``k_out`` may be ``q``/``k`` themselves (no row of which may then lie
    on another).  Returns both outputs
    (new ones have the inputs' layout)."""
    if not q.is_cuda or q.dim() != 3:
        raise ValueError("q must be a CUDA tensor [heads, rows, head_dim]")
    if q.dtype not in _DTYPES:
        raise ValueError(f"dtype {q.dtype} is not supported (bfloat16, float16 or float32)")
    rows, D, dev = q.shape[1], rotary.head_dim, q.device
    hq, hk = _check_rows("q", q, (q.shape[0], rows, D), q.dtype, dev), _heads(None)
    if k is not None:
        if k.dim() != 3:
            raise ValueError("k must be [heads, rows, head_dim]")
        hk = _check_rows("k", k, (k.shape[0], rows, D), q.dtype, dev)
    elif k_out is not None or k_weight is not None:
        raise ValueError("k_out or k_weight without k")
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) != (rows,) or \
            positions.device != dev or not positions.is_contiguous():
        raise ValueError(f"positions must be a contiguous int32 or int64 [{rows}] tensor on {dev}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (D,) or w.dtype != q.dtype or w.device != dev or
                              not w.is_contiguous() or w.data_ptr() % 16):
            raise ValueError(f"{name} must be a contiguous, 16-byte aligned [{D}] {q.dtype} tensor on {dev}")
    if q_out is not None or k_out is not None:
        _check_apart("q_out", q_out, "k_out", k_out)
        _check_apart("q_out", q_out, "k", k)
        _check_apart("k_out", k_out, "q", q)
    outs, structs = [], []
    for name, x, o, h in (("q_out", q, q_out, hq), ("k_out", k, k_out, hk)):
        if o is None:
            if x is not None:
                o = torch.empty_like(x) if stream is None else _allocate(stream, torch.empty_like, x)
            h = _heads(o)
        else:
            if o is not x:
                h = _check_rows(name, o, tuple(x.shape), q.dtype, dev)
            _check_writable(name, o)
        outs.append(o)
        structs.append(h)
    _launch(dev, stream, _capi.lib().pcp_qk_norm_rope, _DTYPES[q.dtype], rows, D, rotary.rotary_dim,
            _LAYOUTS[rotary.layout], hq, hk, *structs, positions.data_ptr(),
            int(positions.dtype == torch.int64), rotary.turns(dev, stream).data_ptr(), rotary.magnitude,
            0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(), eps)
    return outs[0], outs[1]
