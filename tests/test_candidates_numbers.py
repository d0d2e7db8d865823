"""Factors of the losses over all candidates and of the rotation are numbers: a
tensor that asks for a gradient is refused, not read and dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from starry_unigraph.native import candidates, rotary
from test_candidates_refusals import _f, _i, anywhere  # noqa: F401


def _calls():
    return {"scale": [lambda x: candidates.cross_entropy(_f(2, 8), _f(5, 8), _i(2), scale=x),
                      lambda x: candidates.distillation(_f(2, 8), _f(5, 8), _i(2, 3), _f(2, 3), scale=x)],
            "temperature": [lambda x: candidates.distillation(_f(2, 8), _f(5, 8), _i(2, 3), _f(2, 3), temperature=x)],
            "gain": [lambda x: rotary.rotate(_f(1, 2, 1, 8), None, _i(1, 2), None, _f(4, dtype=torch.float64), gain=x)]}


@pytest.mark.parametrize("name", ["scale", "temperature", "gain"])
def test_gradients_are_refused(anywhere, name):  # noqa: F811
    for call in _calls()[name]:
        for x in (torch.ones(()).requires_grad_(), torch.nn.Parameter(torch.ones(1))):
            with pytest.raises(ValueError, match=f"{name}: has no gradient"):
                call(x)
        with fwd.dual_level(), pytest.raises(NotImplementedError):
            call(fwd.make_dual(torch.ones(()), torch.ones(())))


@pytest.mark.parametrize("gain", [1e39, -1e300, float("nan"), float("-inf")])
def test_gains_beyond_float32_are_refused(anywhere, gain):  # noqa: F811
    with pytest.raises(ValueError, match="gain"):
        _calls()["gain"][0](gain)


def test_a_tangent_of_the_frequencies_is_refused(anywhere):  # noqa: F811
    f = _f(4, dtype=torch.float64)
    with fwd.dual_level(), pytest.raises(NotImplementedError):
        rotary.rotate(_f(1, 2, 1, 8), None, _i(1, 2), None, fwd.make_dual(f, f))


@pytest.mark.parametrize("kw", [
    dict(scaling="base", factor=1e300), dict(scaling="base", base=1e-300, factor=1e-10),
    dict(scaling="wavelength", trained=float("nan")), dict(scaling="wavelength", trained=float("inf")),
    dict(scaling="wavelength", trained=8192, low=float("-inf")),
    dict(scaling="wavelength", trained=8192, low=float("nan")),
    dict(scaling="wavelength", trained=8192, high=float("nan"))])
def test_frequencies_without_angles_are_refused(kw):
    with pytest.raises(ValueError):
        rotary.frequencies(8, device="cpu", **kw)
