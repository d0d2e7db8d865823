"""What the losses over all candidates and the rotary positions refuse, without
a GPU: their checks come before any launch (tensors here live on the CPU), the
C entries' before any access."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

from starry_unigraph.lib import _capi
from starry_unigraph.native import candidates, rotary


@pytest.fixture
def anywhere(monkeypatch):
    """The operators' argument checks on CPU tensors."""
    monkeypatch.setattr(_capi, "require_gpu", lambda device=None: torch.device("cpu"))


def _f(*s, dtype=torch.float32):
    return torch.zeros(s, dtype=dtype)


def _i(*s, dtype=torch.int64):
    return torch.zeros(s, dtype=dtype)


def test_cpu_tensors_are_refused():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        candidates.cross_entropy(_f(2, 8), _f(5, 8), _i(2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        candidates.distillation(_f(2, 8), _f(5, 8), _i(2, 3), _f(2, 3))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rotary.rotate(_f(1, 2, 1, 4), None, _i(1, 2), None, _f(2, dtype=torch.float64))


@pytest.mark.parametrize("kw, match", [
    (dict(h=_f(2, 8, dtype=torch.float64)), "h: torch.float64"),
    (dict(h=torch.tensor(1.0)), "h: 0 dimensions"),
    (dict(h=_f(2, 0), table=_f(5, 0)), "h: rows of 0"),
    (dict(h=_f(2, 257), table=_f(5, 257)), "h: rows of 257"),
    (dict(table=_f(5, 8, dtype=torch.bfloat16)), "table: torch.bfloat16"),
    (dict(table=_f(5, 9)), "table: shape"),
    (dict(table=_f(5, 8, 1)), "table: 3 dimensions"),
    (dict(table=_f(0, 8)), "no candidates"),
    (dict(bias=_f(4)), "bias: shape"),
    (dict(bias=_f(5, dtype=torch.float16)), "bias: torch.float16"),
    (dict(scale=float("nan")), "scale"),
])
def test_shared_refusals(anywhere, kw, match):
    args = dict(h=_f(2, 8), table=_f(5, 8))
    args.update(kw)
    h, table = args.pop("h"), args.pop("table")
    n = h.shape[:-1]
    with pytest.raises(ValueError, match=match):
        candidates.cross_entropy(h, table, _i(*n), **args)
    with pytest.raises(ValueError, match=match):
        candidates.distillation(h, table, _i(*n, 3), _f(*n, 3), **args)


@pytest.mark.parametrize("target", [_i(3), _i(2, 1), _i(2, dtype=torch.int32), _f(2)])
def test_label_refusals(anywhere, target):
    with pytest.raises(ValueError, match="target"):
        candidates.cross_entropy(_f(2, 8), _f(5, 8), target)


@pytest.mark.parametrize("kw, match", [
    (dict(ids=_i(2)), "ids"),
    (dict(ids=_i(3, 4)), "ids"),
    (dict(ids=_i(2, 4, dtype=torch.int32)), "ids: torch.int32"),
    (dict(ids=_i(2, 0), logits=_f(2, 0)), "0 entries"),
    (dict(ids=_i(2, 1025), logits=_f(2, 1025)), "1025 entries"),
    (dict(logits=_f(2, 5)), "logits: shape"),
    (dict(logits=_f(2, 4, dtype=torch.bfloat16)), "logits: torch.bfloat16"),
    (dict(logits=_f(2, 4).requires_grad_()), "logits: has no gradient"),
    (dict(temperature=0.0), "temperature"),
    (dict(temperature=float("inf")), "temperature"),
    (dict(temperature=float("nan")), "temperature"),
])
def test_teacher_refusals(anywhere, kw, match):
    args = dict(ids=_i(2, 4), logits=_f(2, 4))
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        candidates.distillation(_f(2, 8), _f(5, 8), args.pop("ids"), args.pop("logits"), **args)


@pytest.mark.parametrize("kw, match", [
    (dict(q=_f(2, 3, 4)), "q: 3 dimensions"),
    (dict(q=_f(2, 3, 1, 8, dtype=torch.float64)), "q: torch.float64"),
    (dict(q=_f(2, 3, 1, 0)), "heads of 0"),
    (dict(k=None), "both or neither"),
    (dict(k=_f(2, 4, 8)), "k: 3 dimensions"),
    (dict(k=_f(2, 4, 1, 7)), "k: shape"),
    (dict(k=_f(2, 4, 1, 8, dtype=torch.float16)), "k: torch.float16"),
    (dict(q_pos=_i(2, 4)), "q_pos: shape"),
    (dict(q_pos=_f(2, 3)), "q_pos: torch.float32"),
    (dict(k_pos=_i(2, 3)), "k_pos: shape"),
    (dict(freqs=_f(5, dtype=torch.float64)), "at most 4 pairs"),
    (dict(freqs=_f(4)), "freqs: torch.float32"),
    (dict(freqs=_f(2, 2, dtype=torch.float64)), "freqs: shape"),
    (dict(freqs=_f(4, dtype=torch.float64).requires_grad_()), "freqs: has no gradient"),
    (dict(gain=float("inf")), "gain"),
])
def test_rotation_refusals(anywhere, kw, match):
    args = dict(q=_f(2, 3, 1, 8), k=_f(2, 4, 1, 8), q_pos=_i(2, 3), k_pos=_i(2, 4), freqs=_f(4, dtype=torch.float64))
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        rotary.rotate(*[args.pop(n) for n in ("q", "k", "q_pos", "k_pos", "freqs")], **args)


def test_tangents_are_refused(anywhere):
    with fwd.dual_level():
        t = fwd.make_dual(_f(2, 8), _f(2, 8))
        with pytest.raises(NotImplementedError):
            candidates.cross_entropy(t, _f(5, 8), _i(2))
        with pytest.raises(NotImplementedError):
            candidates.distillation(t, _f(5, 8), _i(2, 3), _f(2, 3))
        with pytest.raises(NotImplementedError):
            rotary.rotate(t.view(1, 2, 1, 8), None, _i(1, 2), None, _f(2, dtype=torch.float64))


def test_frequencies():
    f = rotary.frequencies(8, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, 10000.0 ** -torch.tensor([0, 0.25, 0.5, 0.75]).double())
    assert torch.allclose(rotary.frequencies(8, scaling="linear", factor=4.0, device="cpu"), f / 4)
    raised = rotary.frequencies(8, scaling="base", factor=4.0, device="cpu")
    assert raised[0] == 1 and torch.allclose(raised[-1], f[-1] / 4)
    long = rotary.frequencies(64, scaling="wavelength", factor=16.0, trained=8192, device="cpu")
    short = rotary.frequencies(64, device="cpu")
    turns = short * 8192 / (2 * torch.pi)
    assert torch.equal(long[turns > 32], short[turns > 32])
    assert torch.allclose(long[turns < 1], short[turns < 1] / 16)
    between = (turns > 1) & (turns < 32)
    assert ((long < short) & (long > short / 16))[between].all() and between.any()
    assert rotary.frequencies(0, device="cpu").shape == (0,) and rotary.frequencies(2, scaling="base", device="cpu") == 1
    for kw in (dict(dims=3), dict(dims=-2), dict(dims=4, base=0.0), dict(dims=4, factor=float("inf")),
               dict(dims=4, scaling="other"), dict(dims=4, scaling="wavelength"),
               dict(dims=4, scaling="wavelength", trained=8, low=2.0, high=2.0)):
        with pytest.raises(ValueError):
            rotary.frequencies(device="cpu", **kw)


def _problem(**kw):
    a = dict(dtype=1, dim=100, n=10, v=20, h=4096, table=4096, h_stride=100, table_stride=100, bias=None, scale=1.0,
             temperature=1.0)
    a.update(kw)
    return _capi.Candidates(*a.values())


@pytest.mark.parametrize("kw, match", [
    (dict(dtype=3), b"element type"),
    (dict(dim=7), b"rows of 7"),
    (dict(dim=257), b"rows of 257"),
    (dict(dim=3, dtype=0), b"rows of 3"),
    (dict(n=-1), b"too many"),
    (dict(n=1 << 24), b"too many"),
    (dict(v=0), b"too many"),
    (dict(v=1 << 31), b"too many"),
    (dict(h_stride=-1), b"stride"),
    (dict(table_stride=(1 << 22) + 1), b"stride"),
    (dict(table=None), b"NULL"),
    (dict(scale=float("inf")), b"scale"),
    (dict(temperature=0.0), b"temperature"),
])
def test_entry_points_refuse(kw, match):
    lib, ref = _capi.lib(), ctypes.byref(_problem(**kw))
    assert lib.sgl_candidates_workspace_bytes(ref, 1, 0, 3, 0) == 0 and lib.sgl_candidates_keep_bytes(ref, 1, 0, 3) == 0
    big = 1 << 40
    assert lib.sgl_candidates_forward(ref, 4096, None, None, 1, 3, 4096, 4096, big, 4096, big, None) != 0
    assert match in lib.sgl_last_error()
    assert lib.sgl_candidates_backward(ref, 1, 0, 3, 4096, big, 4096, 4096, 4096, None, 4096, big, None) != 0
    assert match in lib.sgl_last_error()


def test_entry_points_refuse_their_arrays():
    lib, ref, big = _capi.lib(), ctypes.byref(_problem()), 1 << 40
    good = dict(target=4096, ids=None, logits=None, k=1, need=3, loss=4096, keep=4096, nk=big, ws=4096, nb=big)
    for kw, what in (
            (dict(k=2), b"2 targets"), (dict(k=0), b"0 targets"),
            (dict(target=None, ids=4096, logits=4096, k=1025), b"1025 targets"),
            (dict(target=None, ids=4096, k=3), b"NULL array"), (dict(target=None), b"NULL array"),
            (dict(ids=4096), b"at once"), (dict(logits=4096), b"at once"), (dict(loss=None), b"NULL array"),
            (dict(need=4), b"need 4"), (dict(need=-1), b"need -1"), (dict(keep=None), b"for the backward"),
            (dict(nk=16), b"for the backward"), (dict(ws=None), b"workspace"), (dict(nb=16), b"workspace")):
        args = {**good, **kw}
        assert lib.sgl_candidates_forward(ref, *args.values(), None) != 0, kw
        assert what in lib.sgl_last_error(), kw
    good = dict(k=1, teacher=0, need=3, keep=4096, nk=big, g=4096, dh=4096, dtable=4096, dbias=None, ws=4096, nb=big)
    for kw, what in (
            (dict(k=2), b"2 targets"), (dict(k=0, teacher=1), b"0 targets"), (dict(need=0), b"need 0"),
            (dict(g=None), b"did not prepare"), (dict(need=1), b"did not prepare"), (dict(need=2), b"did not prepare"),
            (dict(dtable=None, dbias=4096), b"did not prepare"), (dict(keep=None), b"for the backward"),
            (dict(nk=16), b"for the backward"), (dict(ws=None), b"workspace"), (dict(nb=16), b"workspace")):
        args = {**good, **kw}
        assert lib.sgl_candidates_backward(ref, *args.values(), None) != 0, kw
        assert what in lib.sgl_last_error(), kw
    none = ctypes.byref(_problem(n=0))
    assert lib.sgl_candidates_backward(none, *good.values(), None) != 0
    side = _capi.RotarySide(4096, 4096, 4096, 5, 40, 8, 8, 5, 1, 1)
    s = ctypes.byref(side)
    for args in ((3, 2, 8, 8, s, s, 4096, 0, 1.0, 0), (0, -1, 8, 8, s, s, 4096, 0, 1.0, 0),
                 (0, 2, 8, 7, s, s, 4096, 0, 1.0, 0), (0, 2, 8, 10, s, s, 4096, 0, 1.0, 0),
                 (0, 2, 8, 8, s, s, None, 0, 1.0, 0), (0, 2, 8, 8, None, s, 4096, 0, 1.0, 0),
                 (0, 1 << 40, 8, 8, s, s, 4096, 0, 1.0, 0), (0, 1 << 31, 8, 8, s, s, 4096, 0, 1.0, 0)):
        assert lib.sgl_rotary(*args, None) != 0, args
    side.y = None
    assert lib.sgl_rotary(0, 2, 8, 8, s, None, 4096, 0, 1.0, 0, None) != 0


@pytest.mark.parametrize("scale, temperature", [(1.0, 1e-39), (1e30, 1e-20), (1.0, 1e20), (3e38, 1.0)])
def test_factors_beyond_float32_are_refused(anywhere, scale, temperature):
    with pytest.raises(ValueError, match="temperature|scale"):
        candidates.distillation(_f(2, 8), _f(5, 8), _i(2, 4), _f(2, 4), scale=scale, temperature=temperature)
    lib, ref = _capi.lib(), ctypes.byref(_problem(scale=scale, temperature=temperature))
    assert lib.sgl_candidates_forward(ref, 4096, None, None, 1, 3, 4096, 4096, 1 << 40, 4096, 1 << 40, None) != 0
    assert b"temperature" in lib.sgl_last_error()
