"""The history operators' calls on the way to their kernels, without a GPU:
what autograd asks of them, and refusals that come before any launch."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from starry_unigraph.lib import _capi
from starry_unigraph.native import history


@pytest.fixture
def anywhere(monkeypatch):
    """Argument checks on CPU tensors; a call that passes them all stops where
    its kernels would be launched."""
    class Reached(Exception):
        pass

    def stop(*a):
        raise Reached

    monkeypatch.setattr(_capi, "require_gpu", lambda device=None: torch.device("cpu"))
    for op in (history._Scan, history._Attend, history._Norm):
        monkeypatch.setattr(op, "run", stop)
        monkeypatch.setattr(op, "apply", stop)
    return Reached


def _f(*s):
    return torch.zeros(*s)


def _scan(**kw):
    t = dict(gate=_f(2, 3, 4), value=_f(2, 3, 4), state=_f(2, 4), gaps=_f(2, 3), decay=_f(4))
    t.update(kw)
    return history.gated_scan(t.pop("gate"), t.pop("value"), **t)


def _attend(**kw):
    t = dict(q=_f(2, 3, 4, 8), k=_f(2, 5, 2, 8), v=_f(2, 5, 2, 8), bias=_f(4, 6),
             q_pos=torch.zeros(2, 3, dtype=torch.int64), k_pos=torch.zeros(2, 5, dtype=torch.int64))
    t.update(kw)
    return history.cross_attention(t.pop("q"), t.pop("k"), t.pop("v"), **t)


def _norm(**kw):
    t = dict(x=_f(2, 4), z=_f(2, 4), gate=_f(2, 4), scale=_f(4), post_weight=_f(4), pre_weight=_f(4),
             post_bias=_f(4), pre_bias=_f(4))
    t.update(kw)
    return history.gated_norm(*[t.pop(k) for k in ("x", "z", "gate", "scale")], **t)


@pytest.mark.parametrize("call, shapes", [
    (_scan, dict(gate=(2, 3, 4), value=(2, 3, 4), state=(2, 4), gaps=(2, 3), decay=(4,))),
    (_attend, dict(q=(2, 3, 4, 8), k=(2, 5, 2, 8), v=(2, 5, 2, 8), bias=(4, 6))),
    (_norm, dict(x=(2, 4), z=(2, 4), gate=(2, 4), scale=(4,), post_weight=(4,), post_bias=(4,), pre_weight=(4,),
                 pre_bias=(4,))),
], ids=["scan", "attention", "norm"])
def test_forward_mode_tangents_are_refused(anywhere, call, shapes):
    """Not dropped without an error: with gradients on, off, and through
    torch.func; beside a dual level that none of the tensors is in, the call
    goes on."""
    for name, shape in shapes.items():
        with fwd.dual_level():
            dual = fwd.make_dual(_f(*shape), torch.ones(shape))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(**{name: dual})
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(**{name: dual})
            with pytest.raises(anywhere):
                call()
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda t: call(**{name: t}), (_f(*shape),), (torch.ones(shape),))
    with pytest.raises(anywhere):
        call()


def test_more_query_heads_than_a_key_head_takes(anywhere):
    with pytest.raises(anywhere):
        _attend(q=_f(2, 3, 128, 8), bias=None)
    with pytest.raises(ValueError, match="at most 64"):
        _attend(q=_f(2, 3, 130, 8), bias=None)


def test_norm_backward_with_biases_gives_their_gradients():
    """The C entry's form of three parameter gradients forms y without biases."""
    L = _capi.load_library()
    one = 4096   # (never read: the checks come first)
    back = lambda post_b, pre_b, nsum: L.sgl_gated_norm_backward(
        0, 2, 8, one, 8, one, 8, one, 8, one, one, post_b, one, pre_b, 1e-5, 0, one, one, one, one, one, one, nsum, None,
        0, None)
    for biases in ((one, None), (None, one), (one, one)):
        assert back(*biases, 3) == 1 and b"biases need 5" in L.sgl_last_error()
        assert back(*biases, 5) == 3   # (no workspace given)
    assert back(None, None, 3) == 3


def test_distance_bucket_of_the_farthest_distances():
    """int64's ends fall into the last bucket, as the kernels have them."""
    ends = torch.tensor([torch.iinfo(torch.int64).min, torch.iinfo(torch.int64).min + 1, torch.iinfo(torch.int64).max,
                         -(1 << 32), 1 << 32])
    for buckets, resolution in ((1, 0), (20, 0), (64, 1)):
        assert history.distance_bucket(ends, buckets, resolution).tolist() == [buckets - 1] * 5
