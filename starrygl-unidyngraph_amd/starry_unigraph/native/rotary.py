"""Rotary positions for the attention over windows of events
(``history.cross_attention``): pairs of a head's channels of queries and keys
turned by an angle that grows with the event's time or index, so that their
scores depend on the distance of the two. A fused HIP kernel with its gradient
(float32, bfloat16 or float16 tensors on a GPU).

Work is enqueued on the current stream of the tensors' device. Gradients are of
reverse mode and first order; a tangent (forward mode) is refused. The reference
has no counterpart: its attention sees a neighbour's age through a learned
cosine encoding (runtime/modules/time_encode.py:41-58).
"""
from __future__ import annotations

import ctypes
import math

import torch

from starry_unigraph.lib import _capi
from starry_unigraph.native.history import (_first, _first_order, _guard, _no_tangents, _number, _rows, _tensor,
                                            _tracked)


def frequencies(dims: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                trained: int | None = None, low: float = 1.0, high: float = 32.0,
                device: torch.device | str = "cuda") -> torch.Tensor:
    """The angles a unit of position of ``dims`` rotated channels, one a pair:
    ``base ** (-2 i / dims)``, float64 [dims / 2]. ``scaling`` fits them to
    positions ``factor`` times as long (or to another unit of time):

    * "linear": every angle divided by ``factor``;
    * "base": the base raised so that the longest wave is ``factor`` times as
      long and the shortest stays;
    * "wavelength": waves that turn more than ``high`` times over ``trained``
      positions stay, those of less than ``low`` are divided by ``factor``, and
      those between blend."""
    if dims < 0 or dims % 2:
        raise ValueError(f"dims: {dims}, expected an even number")
    if not (base > 0 and math.isfinite(base)) or not (factor > 0 and math.isfinite(factor)):
        raise ValueError(f"base {base}, factor {factor}: expected positive numbers")
    if scaling == "base" and dims > 2:
        log = math.log(base) + math.log(factor) * (dims / (dims - 2))
        if not abs(log) < 708.0:   # (float64's range)
            raise ValueError(f"base {base} raised for a factor of {factor} is out of range")
        base = base * factor ** (dims / (dims - 2))
    f = base ** (torch.arange(0, dims, 2, dtype=torch.float64) * (-1.0 / max(dims, 1)))
    if scaling == "linear":
        f = f / factor
    elif scaling == "wavelength":
        if trained is None or not 1 <= trained < math.inf or not -math.inf < low < high:
            raise ValueError(f"wavelength scaling: trained {trained}, low {low}, high {high}")
        keep = ((f * (trained / (2.0 * math.pi)) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    elif scaling not in ("none", "base"):
        raise ValueError(f"scaling: {scaling!r}, expected 'none', 'linear', 'base' or 'wavelength'")
    return f.to(device)


def rotate(q: torch.Tensor, k: torch.Tensor | None, q_pos: torch.Tensor, k_pos: torch.Tensor | None,
           freqs: torch.Tensor, *, interleaved: bool = False,
           gain: float = 1.0) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``q`` [N, Lq, Hq, dh] and ``k`` [N, Lk, Hkv, dh] with the pairs of their
    first 2 P channels turned by ``position * freqs`` and scaled by ``gain``; the
    other channels as they are. ``k`` and ``k_pos`` may both be None.

    ``q_pos``, ``k_pos``: int64 [N, Lq], [N, Lk] (any values: an angle is within
    2^-32 of a turn at every one). ``freqs``: float64 [P], 2 P <= dh, the angle a
    unit of position of each pair (``frequencies``), under 2^128 (another, as one
    that is not finite, makes its pair NaN); no gradient. Pairs are channels
    (i, i + P), or with ``interleaved`` (2 i, 2 i + 1). Differentiable in q and
    k. One new event per sequence is L = 1."""
    _first("q", q, 4)
    N, Lq, Hq, dh = q.shape
    if dh == 0:
        raise ValueError("q: heads of 0 channels")
    if (k is None) != (k_pos is None):
        raise ValueError("k and k_pos: give both or neither")
    _tensor("q_pos", q_pos, q, (N, Lq), torch.int64)
    if k is not None:
        if k.dim() != 4:
            raise ValueError(f"k: {k.dim()} dimensions, expected 4")
        _tensor("k", k, q, (N, k.shape[1], k.shape[2], dh))
        _tensor("k_pos", k_pos, q, (N, k.shape[1]), torch.int64)
    if freqs.dim() != 1 or 2 * freqs.shape[0] > dh:
        raise ValueError(f"freqs: shape {tuple(freqs.shape)}, expected [pairs] of at most {dh // 2} pairs")
    _tensor("freqs", freqs, q, freqs.shape, torch.float64)
    if freqs.requires_grad:
        raise ValueError("freqs: has no gradient here (detach it)")
    gain = _number("gain", gain)
    if not abs(gain) <= torch.finfo(torch.float32).max:
        raise ValueError(f"gain: {gain}, expected a number in float32's range")
    _no_tangents(q, k, freqs)
    args = (q, k, q_pos, k_pos, freqs.contiguous(), bool(interleaved), gain)
    if _tracked(q, k):
        return _Rotate.apply(*args)
    return _Rotate.run(*args, False)


def _side(x, y, pos):
    """The C struct of ``x`` (its last dimension contiguous), ``y`` and their positions."""
    sn, st, sh, _ = x.stride()
    pn, pt = pos.stride()
    return ctypes.byref(_capi.RotarySide(x.data_ptr(), y.data_ptr(), pos.data_ptr(), x.shape[1], sn, st, sh, pn, pt,
                                         x.shape[2]))


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_pos, k_pos, freqs, interleaved, gain):
        ctx.save_for_backward(q_pos, k_pos, freqs)
        ctx.form = (interleaved, gain)
        ctx.set_materialize_grads(False)
        return _Rotate.run(q, k, q_pos, k_pos, freqs, interleaved, gain, False)

    @staticmethod
    def run(q, k, q_pos, k_pos, freqs, interleaved, gain, inverse):
        """(q, k) turned (None stays None)."""
        one = q if q is not None else k
        dev, new_q, new_k, sides = one.device, None, None, []
        if q is not None:
            q = _rows(q)
            new_q = q.new_empty(q.shape)
            sides.append(_side(q, new_q, q_pos))
        if k is not None:
            k = _rows(k)
            new_k = k.new_empty(k.shape)
            sides.append(_side(k, new_k, k_pos))
        with _guard(dev):
            _capi.check(_capi.lib().sgl_rotary(
                _capi.DTYPES[one.dtype], one.shape[0], one.shape[3], 2 * freqs.shape[0], sides[0],
                sides[1] if len(sides) == 2 else None, freqs.data_ptr(), interleaved, gain, inverse,
                _capi.stream_of(dev)), "rotate")
        return new_q, new_k

    @staticmethod
    @_first_order
    def backward(ctx, gq, gk):
        if gq is None and gk is None:
            return (None,) * 7
        q_pos, k_pos, freqs = ctx.saved_tensors
        dq, dk = _Rotate.run(gq, gk, q_pos, k_pos, freqs, *ctx.form, True)
        return dq, dk, None, None, None, None, None
