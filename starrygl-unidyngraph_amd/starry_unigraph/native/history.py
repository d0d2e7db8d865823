"""Operators of a sequence encoder over windows of events, each a fused HIP
kernel with its gradient (float32, bfloat16 or float16 tensors on a GPU):

* ``gated_scan``: a gated linear recurrence along each sequence, its gate
  decaying with the time between events;
* ``cross_attention``: attention of query events over another sequence's
  events with a bias learned by time distance;
* ``gated_norm``: the residual that a block's normalised, gated output is
  added to, and the norm before the next block.

A sequence is a row of a padded tensor and a count, as the sampler returns its
windows (``PaddedHop``: ``cnt`` and ``[rows, fanout]`` entries). Nothing past a
count is read, and outputs and gradients there are zero. Work is enqueued on
the current stream of the tensors' device; gradients are the same from run to
run. Gradients are of reverse mode and first order; a tangent (forward mode) is
refused. The reference has no counterpart: its embedding attends with one query
row over the window (backends/ctdg/runtime/models.py:77-137) and its memory
runs a GRU over the mailbox slots (models.py:214-254).
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from starry_unigraph.lib import _capi

_NO_GUARD = contextlib.nullcontext()


def _guard(dev: torch.device):
    """The device's context, where it is not the current one already."""
    return _NO_GUARD if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _tensor(name: str, t, like: torch.Tensor, shape: tuple, dtype=None) -> torch.Tensor:
    """``t`` as an operand: its type, shape and device checked."""
    want = like.dtype if dtype is None else dtype
    if t.dtype != want:
        raise ValueError(f"{name}: {t.dtype}, expected {want}")
    if t.device != like.device:
        raise ValueError(f"{name}: on {t.device}, expected {like.device}")
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def _no_tangents(*tensors) -> None:
    """Refuses forward-mode derivatives (the operators have none; a call that
    autograd does not see would drop them)."""
    if getattr(forward_ad, "_current_level", 0) < 0:   # no dual level is open
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("no forward-mode derivative: a tensor carries a tangent")


def _tracked(*tensors) -> bool:
    """Whether autograd has to know of a call (without it nothing is kept)."""
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with a contiguous last dimension (strides before it as they are)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _first(name: str, t: torch.Tensor, dims: int) -> None:
    if t.dtype not in _capi.DTYPES:
        raise ValueError(f"{name}: {t.dtype}, expected float32, bfloat16 or float16")
    if t.dim() != dims:
        raise ValueError(f"{name}: {t.dim()} dimensions, expected {dims}")
    if t.device.type != "cuda":
        _capi.require_gpu(t.device)


def _lens(name: str, lens, like: torch.Tensor, n: int):
    return None if lens is None else _tensor(name, lens, like, (n,), torch.int32).contiguous()


def _no_grad(name: str, t) -> None:
    if t is not None and t.requires_grad:
        raise ValueError(f"{name}: has no gradient here (detach it)")


# ------------------------------------------------------------------ gated scan
def gated_scan(gate: torch.Tensor, value: torch.Tensor, *, lens: torch.Tensor | None = None,
               state: torch.Tensor | None = None, gaps: torch.Tensor | None = None,
               decay: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The recurrence ``h_t = a_t h_(t-1) + (1 - a_t) value_t`` along every
    sequence, ``a_t = sigmoid(gate_t) exp(-decay * gaps_t)`` (without ``gaps``
    and ``decay``: ``sigmoid(gate_t)``), from ``state`` (default 0).

    ``gate``, ``value``: [N, L, D] of one type. ``lens``: int32 [N], the events
    of each sequence (default L; clamped to 0..L). ``state``: float32 [N, D].
    ``gaps``: float32 [N, L], the time before each event; ``decay``: float32
    [D], a rate a channel (both non-negative in use). Returns ``h`` [N, L, D]
    and the state after each sequence's last event, float32 [N, D] (``state``
    itself for an empty sequence). Differentiable in gate, value, state and
    decay. One new event per sequence is L = 1."""
    _first("gate", gate, 3)
    N, L, D = gate.shape
    _tensor("value", value, gate, gate.shape)
    lens = _lens("lens", lens, gate, N)
    if state is not None:
        _tensor("state", state, gate, (N, D), torch.float32)
    if (gaps is None) != (decay is None):
        raise ValueError("gaps and decay: give both or neither")
    if gaps is not None:
        _no_grad("gaps", gaps)
        _tensor("gaps", gaps, gate, (N, L), torch.float32)
        _tensor("decay", decay, gate, (D,), torch.float32)
    if D == 0:
        raise ValueError("gate: no channels")
    if N == 0 or L == 0:   # nothing to run: empty rows, the states as they are
        last = state + 0.0 if state is not None else torch.zeros(N, D, device=gate.device)
        return gate + value, last if decay is None else last + 0.0 * decay
    _no_tangents(gate, value, state, gaps, decay)
    if not _tracked(gate, value, state, decay):
        return _Scan.run(gate, value, state, decay, lens, gaps, False)[:2]
    return _Scan.apply(gate, value, state, decay, lens, gaps)


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        h, last, saved = _Scan.run(*args, True)
        ctx.save_for_backward(*saved)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    def run(gate, value, state, decay, lens, gaps, need):
        lib, P, dev = _capi.lib(), _capi.ptr, gate.device
        gate, value = _rows(gate), _rows(value)
        state = None if state is None else state.contiguous()
        decay = None if decay is None else decay.contiguous()
        N, L, D = gate.shape
        dt = _capi.DTYPES[gate.dtype]
        h = torch.empty(N, L, D, dtype=gate.dtype, device=dev)
        last = torch.empty(N, D, dtype=torch.float32, device=dev)
        keep = None
        if need:
            keep = torch.empty(lib.sgl_gated_scan_keep_elems(N, L, D), dtype=torch.float32, device=dev)
        nb = lib.sgl_gated_scan_workspace_bytes(dt, N, L, D, 0, 0)
        ws = _capi.workspace(nb, dev) if nb else None
        with _guard(dev):
            _capi.check(lib.sgl_gated_scan_forward(
                dt, N, L, D, *_Scan.inputs(gate, value, lens, state, gaps, decay), P(h), P(last), P(keep), P(ws), nb,
                _capi.stream_of(dev)), "gated_scan")
        return h, last, (gate, value, state, decay, lens, gaps, keep)

    @staticmethod
    def inputs(gate, value, lens, state, gaps, decay) -> tuple:
        P = _capi.ptr
        gn, gt = gaps.stride() if gaps is not None else (0, 0)
        return (P(gate), gate.stride(0), gate.stride(1), P(value), value.stride(0), value.stride(1), P(lens), P(state),
                P(gaps), gn, gt, P(decay))

    @staticmethod
    @once_differentiable
    def backward(ctx, gh, glast):
        gate, value, state, decay, lens, gaps, keep = ctx.saved_tensors
        if gh is None and glast is None:
            return (None,) * 6
        lib, P, dev = _capi.lib(), _capi.ptr, gate.device
        N, L, D = gate.shape
        dt = _capi.DTYPES[gate.dtype]
        gh = None if gh is None else gh.contiguous()
        glast = None if glast is None else glast.contiguous()
        dgate = torch.empty(N, L, D, dtype=gate.dtype, device=dev)
        dvalue = torch.empty_like(dgate)
        dstate = torch.empty(N, D, dtype=torch.float32, device=dev) if state is not None else None
        ddecay = torch.empty(D, dtype=torch.float32, device=dev) if decay is not None else None
        nb = lib.sgl_gated_scan_workspace_bytes(dt, N, L, D, 1, decay is not None)
        ws = _capi.workspace(nb, dev) if nb else None
        with _guard(dev):
            _capi.check(lib.sgl_gated_scan_backward(
                dt, N, L, D, *_Scan.inputs(gate, value, lens, state, gaps, decay), P(keep), P(gh), P(glast), P(dgate),
                P(dvalue), P(dstate), P(ddecay), P(ws), nb, _capi.stream_of(dev)), "gated_scan backward")
        return dgate, dvalue, dstate, ddecay, None, None


# ------------------------------------------------------------------ cross attention
def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, q_lens: torch.Tensor | None = None,
                    k_lens: torch.Tensor | None = None, key_mask: torch.Tensor | None = None,
                    bias: torch.Tensor | None = None, q_pos: torch.Tensor | None = None,
                    k_pos: torch.Tensor | None = None, resolution: int = 0, two_sided: bool = False,
                    scale: float | None = None) -> torch.Tensor:
    """Attention of ``q`` [N, Lq, Hq, dh] over the states ``k``, ``v``
    [N, Lk, Hkv, dh] of another length (Hq a multiple of Hkv, at most 64 times:
    consecutive query heads share a key head; dh up to 128): softmax over the
    live keys of ``scale * <q, k> + bias``, ``scale`` dh**-0.5 by default.

    ``q_lens``, ``k_lens``: int32 [N], the events of each sequence (default
    all; clamped). ``key_mask``: bool [N, Lk], False a key that is left out.
    ``bias``: float32 [Hq, C], C at most 64: a learned value for each head and
    bucket of the distance ``q_pos - k_pos`` (int64 event times or indexes,
    [N, Lq] and [N, Lk], whose differences are int64 too). ``two_sided``: C is
    twice the buckets, the second half for keys after the query; else such keys
    count as distance 0. The buckets are ``distance_bucket``'s, 2**resolution an
    octave. Returns [N, Lq, Hq, dh], zero in rows without a live key (or with
    -inf in the table for all of them). Differentiable in q, k, v
    and bias. One new event per sequence is Lq = 1."""
    _first("q", q, 4)
    N, Lq, Hq, dh = q.shape
    if k.dim() != 4:
        raise ValueError(f"k: {k.dim()} dimensions, expected 4")
    Lk, Hkv = k.shape[1], k.shape[2]
    _tensor("k", k, q, (N, Lk, Hkv, dh))
    _tensor("v", v, q, (N, Lk, Hkv, dh))
    if Hq == 0 or Hkv == 0 or Hq % Hkv:
        raise ValueError(f"q: {Hq} heads over {Hkv} key heads, expected a multiple")
    if Hq // Hkv > 64:
        raise ValueError(f"q: {Hq} heads over {Hkv} key heads, at most 64 to one")
    if not 1 <= dh <= 128:
        raise ValueError(f"q: heads of {dh}, expected 1 to 128")
    q_lens, k_lens = _lens("q_lens", q_lens, q, N), _lens("k_lens", k_lens, q, N)
    if key_mask is not None:
        _tensor("key_mask", key_mask, q, (N, Lk), torch.bool)
    if bias is not None:
        if q_pos is None or k_pos is None:
            raise ValueError("bias: needs q_pos and k_pos")
        if bias.dim() != 2 or not 1 <= bias.shape[1] <= 64 or (two_sided and bias.shape[1] % 2):
            raise ValueError(f"bias: shape {tuple(bias.shape)}, expected [{Hq}, buckets] of at most 64 columns "
                             "(an even number when two_sided)")
        _tensor("bias", bias, q, (Hq, bias.shape[1]), torch.float32)
        if not 0 <= int(resolution) <= 4:
            raise ValueError(f"resolution: {resolution}, expected 0 to 4")
        _tensor("q_pos", q_pos, q, (N, Lq), torch.int64)
        _tensor("k_pos", k_pos, q, (N, Lk), torch.int64)
    scale = dh ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale: {scale}")
    _no_tangents(q, k, v, bias)
    least = 16 // q.element_size()
    if dh < least:   # the kernels read 16 bytes of a head at a time: zeros add nothing to the products
        q, k, v = (torch.nn.functional.pad(t, (0, least - dh)) for t in (q, k, v))
    fixed = (q_lens, k_lens, key_mask) + ((q_pos, k_pos) if bias is not None else (None, None))
    if _tracked(q, k, v, bias):
        o = _Attend.apply(q, k, v, bias, fixed, int(resolution), bool(two_sided), scale)
    else:
        o = _Attend.run(q, k, v, bias, fixed, int(resolution), bool(two_sided), scale, False)[0]
    return o if dh >= least else o[..., :dh]


def distance_bucket(distance: torch.Tensor, buckets: int, resolution: int = 0) -> torch.Tensor:
    """The bucket of each int64 ``distance`` (its absolute value; at least 0):
    distances under 2**resolution are buckets of their own, and above them each
    octave has 2**resolution; the last of the ``buckets`` takes everything
    beyond it. A two-sided table adds ``buckets`` where the distance is
    negative. The kernels compute the same from integers."""
    d = distance.clamp(-0xFFFFFFFF, 0xFFFFFFFF).abs()   # (int64's lowest value has no absolute value)
    e = torch.full_like(d, resolution)
    for b in range(resolution + 1, 32):
        e = e + (d >= (1 << b))
    return ((d >> (e - resolution)) + ((e - resolution) << resolution)).clamp(max=buckets - 1)


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        o, saved = _Attend.run(*args, True)
        ctx.save_for_backward(*saved)
        ctx.form = args[5:]
        return o

    @staticmethod
    def run(q, k, v, bias, fixed, resolution, two_sided, scale, need):
        """(o, the backward's tensors)."""
        lib, P, dev = _capi.lib(), _capi.ptr, q.device
        q, k, v = _rows(q), _rows(k), _rows(v)
        bias = None if bias is None else bias.contiguous()
        a = _Attend.problem(q, k, v, bias, fixed, resolution, two_sided, scale)
        ref = ctypes.byref(a)
        N, Lq, Hq, dh = q.shape
        o = torch.empty(N, Lq, Hq, dh, dtype=q.dtype, device=dev)
        saves = lib.sgl_cross_attention_saves(ref) if need else 0
        lse = torch.empty(N, Lq * Hq, 2, dtype=torch.float32, device=dev) if saves & 1 else None
        rest = torch.empty_like(o) if saves & 2 else None
        nb = lib.sgl_cross_attention_workspace_bytes(ref, 0)
        ws = _capi.workspace(nb, dev) if nb else None
        with _guard(dev):
            _capi.check(lib.sgl_cross_attention_forward(ref, P(o), P(rest), P(lse), P(ws), nb, _capi.stream_of(dev)),
                        "cross_attention")
        return o, (q, k, v, bias, o if saves & 1 else None, rest, lse, *fixed)

    @staticmethod
    def problem(q, k, v, bias, fixed, resolution, two_sided, scale):
        P = _capi.ptr
        q_lens, k_lens, mask, q_pos, k_pos = fixed
        N, Lq, Hq, dh = q.shape
        Lk, Hkv = k.shape[1], k.shape[2]
        ms = mask.stride() if mask is not None else (0, 0)
        qs, ks = (q_pos.stride(), k_pos.stride()) if q_pos is not None else ((0, 0), (0, 0))
        cols = bias.shape[1] if bias is not None else 0
        return _capi.Attention(
            _capi.DTYPES[q.dtype], Hq, Hkv, dh, N, Lq, Lk, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], P(q),
            P(k), P(v), P(q_lens), P(k_lens), P(mask), *ms, P(bias), cols // 2 if two_sided else cols, resolution,
            two_sided, scale, P(q_pos), P(k_pos), *qs, *ks)

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, bias, o, rest, lse, *fixed = ctx.saved_tensors
        lib, P, dev = _capi.lib(), _capi.ptr, q.device
        # (from the tensors as they are now: a hook on saved tensors may bring them back elsewhere)
        a = ctypes.byref(_Attend.problem(q, k, v, bias, fixed, *ctx.form))
        go = go.contiguous()
        dq = torch.empty_like(go)
        dk = torch.empty(k.shape, dtype=k.dtype, device=dev)
        dv = torch.empty(v.shape, dtype=v.dtype, device=dev)
        db = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[3] else None
        nb = lib.sgl_cross_attention_workspace_bytes(a, 1)
        ws = _capi.workspace(nb, dev) if nb else None
        with _guard(dev):
            _capi.check(lib.sgl_cross_attention_backward(
                a, P(o), P(rest), P(lse), P(go), P(dq), P(dk), P(dv), P(db), P(ws), nb, _capi.stream_of(dev)),
                "cross_attention backward")
        return dq, dk, dv, db, None, None, None, None


# ------------------------------------------------------------------ gated norm
def gated_norm(x: torch.Tensor, z: torch.Tensor, gate: torch.Tensor, scale: torch.Tensor, *,
               post_weight: torch.Tensor, post_bias: torch.Tensor | None = None, pre_weight: torch.Tensor,
               pre_bias: torch.Tensor | None = None, eps: float = 1e-5,
               rms: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``y = x + scale * sigmoid(gate) * norm(z)`` and the next block's input
    ``norm(y)``: a block's output ``z`` normalised (post), gated and scaled onto
    the residual ``x``, and the norm before the next block (pre) of the sum.

    ``x``, ``z``, ``gate``: [..., D] of one type and shape, D up to 8192;
    ``scale``, the weights and biases: float32 [D] (biases both or neither).
    The norms are layer norms over D, or with ``rms`` divide by the root mean
    square alone. Returns (y, norm(y)); the norm is of the unrounded sum.
    Differentiable in every tensor."""
    _first("x", x, max(x.dim(), 1))
    D = x.shape[-1]
    if not 1 <= D <= 8192:
        raise ValueError(f"x: rows of {D}, expected 1 to 8192")
    _tensor("z", z, x, x.shape)
    _tensor("gate", gate, x, x.shape)
    if (post_bias is None) != (pre_bias is None):
        raise ValueError("post_bias and pre_bias: give both or neither")
    for name, t in (("scale", scale), ("post_weight", post_weight), ("post_bias", post_bias),
                    ("pre_weight", pre_weight), ("pre_bias", pre_bias)):
        if t is not None:
            _tensor(name, t, x, (D,), torch.float32)
    args = (x, z, gate, scale, post_weight, pre_weight, post_bias, pre_bias)
    _no_tangents(*args)
    if _tracked(*args):
        return _Norm.apply(*args, float(eps), bool(rms))
    return _Norm.run(*args, float(eps), bool(rms))[:2]


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows of its last dimension at one stride (a view where it is
    one, else a copy)."""
    t = _rows(t)
    if t.dim() == 2:
        return t
    try:
        return t.view(-1, t.shape[-1])
    except RuntimeError:
        return t.contiguous().view(-1, t.shape[-1])


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        y, n, saved = _Norm.run(*args)
        ctx.save_for_backward(*saved)
        ctx.form = (y.shape, *args[-2:])
        ctx.set_materialize_grads(False)
        return y, n

    @staticmethod
    def run(x, z, gate, scale, post_w, pre_w, post_b, pre_b, eps, rms):
        lib, P, dev = _capi.lib(), _capi.ptr, x.device
        shape = x.shape
        x, z, gate = _as_rows(x), _as_rows(z), _as_rows(gate)
        vecs = [None if t is None else t.contiguous() for t in (scale, post_w, post_b, pre_w, pre_b)]
        rows, D = x.shape
        y = torch.empty(shape, dtype=x.dtype, device=dev)
        n = torch.empty_like(y)
        dt = _capi.DTYPES[x.dtype]
        with _guard(dev):
            _capi.check(lib.sgl_gated_norm_forward(dt, rows, D, *_Norm.inputs(x, z, gate, vecs), eps, rms, P(y), P(n),
                                                   _capi.stream_of(dev)), "gated_norm")
        return y, n, (x, z, gate, *vecs)

    @staticmethod
    def inputs(x, z, gate, vecs) -> tuple:
        P = _capi.ptr
        return (P(x), x.stride(0), P(z), z.stride(0), P(gate), gate.stride(0), *[P(t) for t in vecs])

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gn):
        if gy is None and gn is None:
            return (None,) * 10
        x, z, gate, *vecs = ctx.saved_tensors
        shape, eps, rms = ctx.form
        lib, P, dev = _capi.lib(), _capi.ptr, x.device
        rows, D = x.shape
        gy = None if gy is None else gy.contiguous()
        gn = None if gn is None else gn.contiguous()
        dx = torch.empty(shape, dtype=x.dtype, device=dev)
        dz, dg = torch.empty_like(dx), torch.empty_like(dx)
        nsum = 5 if vecs[2] is not None else 3
        dp = torch.empty(nsum, D, dtype=torch.float32, device=dev)
        nb = lib.sgl_gated_norm_workspace_bytes(rows, D)
        ws = _capi.workspace(nb, dev) if nb else None
        with _guard(dev):
            _capi.check(lib.sgl_gated_norm_backward(
                _capi.DTYPES[x.dtype], rows, D, *_Norm.inputs(x, z, gate, vecs), eps, rms, P(gy), P(gn), P(dx), P(dz),
                P(dg), P(dp), nsum, P(ws), nb, _capi.stream_of(dev)), "gated_norm backward")
        d = dp.unbind(0)
        return dx, dz, dg, d[0], d[1], d[2], d[3] if nsum == 5 else None, d[4] if nsum == 5 else None, None, None
