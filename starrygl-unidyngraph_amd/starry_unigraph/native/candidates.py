"""Losses over every candidate node, each a set of fused HIP kernels with its
gradient (float32, bfloat16 or float16 tensors on a GPU):

* ``cross_entropy``: the softmax cross entropy of rows over all rows of a table
  (which node comes next, out of all of them);
* ``distillation``: the divergence of that softmax from a teacher's, given the
  teacher's top candidates and their logits.

The scores [rows, candidates] are never stored: the table is walked in pieces
with a running softmax, and the gradient of the table forms them again. Work is
enqueued on the current stream of the tensors' device; results and gradients
are the same from run to run. Gradients are of reverse mode and first order; a
tangent (forward mode) is refused. The reference has no counterpart: it scores
an event against one drawn negative
(backends/ctdg/runtime/models.py:313-324, runtime.py:124-136).
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from starry_unigraph.lib import _capi
from starry_unigraph.native.history import (_as_rows, _first, _first_order, _guard, _no_grad, _no_tangents, _number,
                                            _rows, _tensor, _tracked)

MAX_DIM = 256       # channels of a row
MAX_TARGETS = 1024  # a teacher's entries of a row
MAX_STRIDE = 1 << 22   # elements from row to row that the kernels take


def cross_entropy(h: torch.Tensor, table: torch.Tensor, target: torch.Tensor, *, bias: torch.Tensor | None = None,
                  scale: float = 1.0) -> torch.Tensor:
    """``logsumexp_v(s_v) - s_target`` of each row over all candidates, ``s_v =
    scale * <h, table_v> + bias_v``: float32, like ``target``.

    ``h``: [..., D]; ``table``: [V, D] of the same type, D up to 256; ``target``:
    int64 [...], the candidate that came: a row with a negative one (padding) is
    left out, its loss 0 (``h`` may hold anything there); with one of V or more
    the loss is NaN and has no gradient. ``bias``: float32 [V], a learned
    value of each candidate, or -inf for those that are left out: their rows of
    the table may hold anything and have gradients of 0 (a target that is left
    out: the loss is inf and the row has no gradient; if all are, 0).
    Differentiable in h, table and bias. One new event is one row."""
    scale = _number("scale", scale)
    rows = _check(h, table, bias, scale)
    if target.dtype != torch.int64 or target.shape != h.shape[:-1] or target.device != h.device:
        raise ValueError(f"target: {target.dtype} {tuple(target.shape)} on {target.device}, expected int64 "
                         f"{tuple(h.shape[:-1])} on {h.device}")
    _no_tangents(h, table, bias)
    return _shaped(_call(rows, table, bias, target.reshape(-1).contiguous(), None, scale, 1.0), h)


def distillation(h: torch.Tensor, table: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor, *,
                 bias: torch.Tensor | None = None, scale: float = 1.0, temperature: float = 1.0) -> torch.Tensor:
    """``T^2 * sum_k q_k (log q_k - log p_ids_k)`` of each row: the divergence of
    the row's softmax over all candidates, ``p = softmax((scale * <h, table_v>
    + bias_v) / T)``, from a teacher's over its top ones, ``q = softmax(logits /
    T)`` over the row's live entries. float32 [...].

    ``h``, ``table``, ``bias`` and ``scale`` as in :func:`cross_entropy`.
    ``ids``: int64 [..., K], K up to 1024, the teacher's candidates in any order
    (negative: no entry; the same one twice: two entries, with which the sum may
    be negative); ``logits``: float32 [..., K], without gradient (-inf: no entry,
    whatever its id). A row without an entry has
    loss 0 and no gradient; one with an id of V or more NaN and none; one that
    wants a candidate that is left out inf and none. Differentiable in h, table and
    bias."""
    scale, temperature = _number("scale", scale), _number("temperature", temperature)
    rows = _check(h, table, bias, scale)
    check_temperature(temperature, scale)
    if ids.dtype != torch.int64 or ids.dim() != h.dim() or ids.shape[:-1] != h.shape[:-1] or ids.device != h.device:
        raise ValueError(f"ids: {ids.dtype} {tuple(ids.shape)} on {ids.device}, expected int64 "
                         f"[{', '.join(str(n) for n in h.shape[:-1])}, K] on {h.device}")
    K = ids.shape[-1]
    if not 1 <= K <= MAX_TARGETS:
        raise ValueError(f"ids: {K} entries a row, expected 1 to {MAX_TARGETS}")
    _tensor("logits", logits, h, ids.shape, torch.float32)
    _no_grad("logits", logits)
    _no_tangents(h, table, bias, logits)
    entries = (ids.reshape(-1, K).contiguous(), logits.reshape(-1, K).contiguous())
    return _shaped(_call(rows, table, bias, None, entries, scale, temperature), h)


def check_temperature(temperature: float, scale: float = 1.0) -> None:
    """Refuses a temperature that :func:`distillation` does not take."""
    if not (0.0 < temperature < math.inf):
        raise ValueError(f"temperature: {temperature}, expected a positive number")
    if not max(abs(scale), 1.0) / temperature < 2e38 or not temperature < 1e19:
        raise ValueError(f"temperature: {temperature} with a scale of {scale} is out of float32's range")


def _check(h, table, bias, scale) -> torch.Tensor:
    """``h`` as rows, its and the table's types, shapes and device checked."""
    _first("h", h, max(h.dim(), 1))
    D = h.shape[-1]
    if not 1 <= D <= MAX_DIM:
        raise ValueError(f"h: rows of {D}, expected 1 to {MAX_DIM}")
    if table.dim() != 2:
        raise ValueError(f"table: {table.dim()} dimensions, expected 2")
    V = table.shape[0]
    _tensor("table", table, h, (V, D))
    if V == 0:
        raise ValueError("table: no candidates")
    if bias is not None:
        _tensor("bias", bias, h, (V,), torch.float32)
    if not abs(scale) < 2e38:   # (float32's range, with log2 e)
        raise ValueError(f"scale: {scale}")
    return _as_rows(h) if h.dim() != 1 else h.unsqueeze(0)


def _call(h, table, bias, target, entries, scale, temperature) -> torch.Tensor:
    if h.shape[0] == 0:   # no rows: an empty loss that every operand gets a gradient of 0 from
        zero = (h.sum() + table[:0].sum()).float()
        return h.new_zeros(0, dtype=torch.float32) + (zero if bias is None else zero + bias[:0].sum())
    least = 16 // h.element_size()
    if h.shape[1] < least:   # the kernels read 16 bytes of a row at a time: zeros add nothing to the products
        h, table = (torch.nn.functional.pad(t, (0, least - t.shape[1])) for t in (h, table))
    if _tracked(h, table, bias):
        return _Loss.apply(h, table, bias, target, entries, scale, temperature)
    return _Loss.run(h, table, bias, target, entries, scale, temperature, 0)[0]


def _shaped(loss: torch.Tensor, h: torch.Tensor) -> torch.Tensor:
    """``loss`` [rows] like ``h``'s rows (rows in a line stay: a view is a step of autograd's)."""
    return loss if h.dim() == 2 else loss.view(h.shape[:-1])


def _near(t: torch.Tensor) -> torch.Tensor:
    """``t`` with a contiguous last dimension and rows at most MAX_STRIDE apart."""
    t = _rows(t)
    return t if t.stride(0) <= MAX_STRIDE else t.contiguous()


@functools.lru_cache(maxsize=256)
def _bytes(dtype: int, dim: int, n: int, v: int, K: int, teacher: bool, need: int) -> tuple[int, int, int]:
    """What the forward keeps for the backward, its workspace, the backward's."""
    lib = _capi.lib()
    a = ctypes.byref(_capi.Candidates(dtype, dim, n, v, 16, 16, dim, dim, None, 1.0, 1.0))   # (never read)
    return (lib.sgl_candidates_keep_bytes(a, K, teacher, need),
            lib.sgl_candidates_workspace_bytes(a, K, teacher, need, 0),
            lib.sgl_candidates_workspace_bytes(a, K, teacher, need, 1) if need else 0)


# (Few steps of Python from here: they bound a training call of a small batch, and
# take twice as long on the thread that autograd runs the backward on.)
def _at(h, table, bias) -> tuple:
    return h.data_ptr(), table.data_ptr(), h.stride(0), table.stride(0), None if bias is None else bias.data_ptr()


def _problem(h, table, at, scale, temperature):
    return ctypes.byref(_capi.Candidates(_capi.DTYPES[h.dtype], h.shape[1], h.shape[0], table.shape[0], *at, scale,
                                         temperature))


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, table, bias, target, entries, scale, temperature):
        # the gradients that will be asked for: 1 of the rows, 2 of the table and bias
        need = int(h.requires_grad) + 2 * int(table.requires_grad or (bias is not None and bias.requires_grad))
        loss, saved, ctx.form = _Loss.run(h, table, bias, target, entries, scale, temperature, need)
        ctx.save_for_backward(*saved)
        return loss

    @staticmethod
    def run(h, table, bias, target, entries, scale, temperature, need):
        """(loss, the backward's tensors, its other values)."""
        dev = h.device
        h, table = _near(h), _near(table)
        if bias is not None:
            bias = bias.contiguous()
        teacher = entries is not None
        K, ids, logits = 1, None, None
        if teacher:
            K, ids, logits = entries[0].shape[1], entries[0].data_ptr(), entries[1].data_ptr()
        kept, room, back = _bytes(_capi.DTYPES[h.dtype], h.shape[1], h.shape[0], table.shape[0], K, teacher, need)
        at = _at(h, table, bias)
        a = _problem(h, table, at, scale, temperature)
        loss = torch.empty(h.shape[0], dtype=torch.float32, device=dev)
        keep = _capi.workspace(kept, dev) if kept else None
        ws = _capi.workspace(room, dev)
        with _guard(dev):
            _capi.check(_capi.lib().sgl_candidates_forward(
                a, None if teacher else target.data_ptr(), ids, logits, K, need, loss.data_ptr(),
                keep.data_ptr() if kept else None, kept, ws.data_ptr(), room, _capi.stream_of(dev)),
                "distillation" if teacher else "cross_entropy")
        return loss, (h, table, bias, keep), (a, at, scale, temperature, K, teacher, need, kept, back)

    @staticmethod
    @_first_order
    def backward(ctx, g):
        h, table, bias, keep = ctx.saved_tensors
        a, at, scale, temperature, K, teacher, need, kept, room = ctx.form
        now = _at(h, table, bias)
        if now != at:   # (a hook on saved tensors has brought them back elsewhere)
            a = _problem(h, table, now, scale, temperature)
        g = g.contiguous()
        rows, candidates, values, *_ = ctx.needs_input_grad
        dh = h.new_empty(h.shape) if rows else None
        dt = db = ws = None
        if candidates or values:
            dt, ws = table.new_empty(table.shape), _capi.workspace(room, h.device)
            db = bias.new_empty(bias.shape) if values else None
        with _guard(h.device):
            _capi.check(_capi.lib().sgl_candidates_backward(
                a, K, teacher, need, keep.data_ptr(), kept, g.data_ptr(), dh.data_ptr() if rows else None,
                None if dt is None else dt.data_ptr(), db.data_ptr() if values else None,
                None if ws is None else ws.data_ptr(), 0 if ws is None else room, _capi.stream_of(h.device)),
                "candidates backward")
        return dh, dt if candidates else None, db, None, None, None, None
