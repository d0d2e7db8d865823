"""fp16 cross attention: the gradients keep their digits whatever the
magnitudes of v, do and p, as long as they are fp16 numbers themselves."""
import pytest
import torch

import history_oracle as ho

pytestmark = pytest.mark.gpu
FP16 = torch.float16


@pytest.fixture(scope="module")
def ops(gpu):
    from starry_unigraph.native import history
    return history


def _grads(ops, t, dev, **kw):
    d = {k: x.to(dev) for k, x in t.items()}
    leaves = [d[k].requires_grad_() for k in ("q", "k", "v")]
    o = ops.cross_attention(*leaves, **kw)
    return dict(zip(("dq", "dk", "dv"), (g.cpu().double() for g in torch.autograd.grad(o, leaves, d["go"]))))


@pytest.mark.parametrize("value, grad", [(2.0 ** -20, 2.0 ** 14), (2.0 ** -10, 2.0 ** 4), (1.0, 1.0), (2.0 ** 15, 2.0 ** -12)])
@pytest.mark.parametrize("form", [  # N, Lq, Lk, Hq, Hkv
    (3, 8, 64, 4, 2),         # one wave a sequence
    (3, 8, 2, 4, 2),
    (2, 64, 2, 4, 2),         # all keys in one tile
    (2, 64, 2048, 4, 2),
    (96, 128, 128, 4, 2),     # eight waves a workgroup, two heads of the same queries
    (64, 128, 128, 3, 1),
], ids=str)
def test_exact_gradients_of_any_magnitude(ops, gpu, form, value, grad):
    """q is orthogonal to every k: each key weighs 1 / Lk. Values are +value
    and -value in eight elements, as many of each, so D is 0 and ds = +-8 value
    grad / Lk; k has the same signs, so dq is 8 value grad, and dk of a key the
    sum of ds over its rows. All are powers of two times the heads."""
    N, Lq, Lk, Hq, Hkv = form
    G = Hq // Hkv
    sign = 1.0 - 2.0 * (torch.arange(Lk) % 2)
    t = dict(q=torch.zeros(N, Lq, Hq, 16), k=torch.zeros(N, Lk, Hkv, 16), v=torch.zeros(N, Lk, Hkv, 16),
             go=torch.zeros(N, Lq, Hq, 16))
    t["q"][..., 5], t["k"][..., 3] = 1.0, sign[None, :, None]
    t["v"][..., 8:] = value * sign[None, :, None, None]
    t["go"][..., 8:] = grad
    t = {k: x.to(FP16) for k, x in t.items()}
    assert float(t["v"].abs().max()) == value and float(t["go"].max()) == grad
    got = _grads(ops, t, gpu, scale=1.0)
    ds = 8 * value * grad / Lk
    want = {k: torch.zeros(x.shape, dtype=torch.float64) for k, x in got.items()}
    want["dq"][..., 3] = 8 * value * grad
    want["dk"][..., 5] = (sign * ds * Lq * G)[None, :, None]
    want["dv"][..., 8:] = grad * Lq * G / Lk
    for k in want:
        if float(want[k].abs().max()) > 65504:   # no fp16 number itself (dv of two keys, where do is large)
            assert k == "dv"
            continue
        # p is off by the logarithm's and the exponential's last places (2^-19 of it), a term and the result round once
        tol = (2 * ho.unit(FP16) + 2.0 ** -19) * want[k].abs() + 2.0 ** -25
        assert ((got[k] - want[k]).abs() <= tol).all(), (k, got[k].abs().max(), want[k].abs().max())


@pytest.mark.parametrize("std", [1e-5, 1e-4, 1e-3, 1.0, 1e3, 1.2e4])
@pytest.mark.parametrize("case", [(5, 6, 40, 4, 2, 24), (3, 70, 250, 4, 2, 24), (30, 128, 130, 4, 1, 64)], ids=str)
def test_random_gradients_of_any_magnitude(ops, gpu, case, std):
    N, Lq, Lk, Hq, Hkv, dh = case
    g = torch.Generator().manual_seed(Lk)
    r = lambda *s: torch.randn(*s, generator=g)
    t = dict(q=r(N, Lq, Hq, dh), k=r(N, Lk, Hkv, dh), v=r(N, Lk, Hkv, dh) * std,
             go=r(N, Lq, Hq, dh) * min(0.5 / std, 1e4))
    t = {k: x.to(FP16) for k, x in t.items()}
    want, bound = ho.attend(**t)
    for k, got in _grads(ops, t, gpu).items():
        bad = ~((got - want[k]).abs() <= bound[k])
        assert not bad.any(), (k, float(((got - want[k]).abs() / bound[k]).max()))


def test_the_scale_follows_terms_that_grow_along_a_sequence(ops, gpu):
    """Values (and with them ds) 2^24 times larger in the last keys than in the
    first: what was summed before is rescaled, nothing overflows."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)
    N, Lq, Lk = 2, 70, 400
    t = dict(q=r(N, Lq, 4, 32) * 0.1, k=r(N, Lk, 2, 32), v=r(N, Lk, 2, 32) * 2.0 ** torch.linspace(-12, 12, Lk)[None, :, None, None],
             go=r(N, Lq, 4, 32) * 2.0 ** torch.linspace(4, -12, Lq)[None, :, None, None])
    t = {k: x.to(FP16) for k, x in t.items()}
    want, bound = ho.attend(**t)
    for k, got in _grads(ops, t, gpu).items():
        assert ((got - want[k]).abs() <= bound[k]).all(), k
