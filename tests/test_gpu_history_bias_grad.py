"""The bias table's gradient over the whole range of magnitudes of values and
gradients: sums that are exact by construction, and random ones against
float64."""
import math

import pytest
import torch

import history_oracle as ho

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops(gpu):
    from starry_unigraph.native import history
    return history


FORMS = [  # N, Lq, Lk, Hq, Hkv
    (3, 8, 16, 4, 2),        # one wave a sequence
    (1500, 3, 64, 4, 2),     # the same, several sequences a wave
    (2, 64, 64, 4, 2),       # all keys in one tile
    (2, 64, 128, 4, 2),
    (96, 128, 128, 4, 2),    # eight waves a workgroup, two heads of the same queries
    (64, 128, 128, 3, 1),    # three heads: rows in order
]


def _even(form, dtype, value, grads):
    """q = 0: every key of a row weighs 1 / Lk, a power of two. Values are
    +value at distance 1 and -value at distance 0, as many of each, in one
    element; so a row's D is 0, ds = +-grads[i] value / Lk, and each column's
    sum is sum(grads) value / 2 a sequence and head."""
    N, Lq, Lk, Hq, Hkv = form
    t = dict(q=torch.zeros(N, Lq, Hq, 8), k=torch.ones(N, Lk, Hkv, 8), v=torch.zeros(N, Lk, Hkv, 8),
             go=torch.zeros(N, Lq, Hq, 8))
    near = torch.arange(Lk) % 2
    t["v"][..., 3] = (value * (2.0 * near - 1))[None, :, None]
    t["go"][..., 3] = grads[None, :, None]
    t = {k: x.to(dtype) for k, x in t.items()}
    t["bias"] = torch.zeros(Hq, 4)
    t["q_pos"], t["k_pos"] = torch.full((N, Lq), 10), (10 - near).expand(N, Lk).contiguous()
    want = torch.zeros(Hq, 4, dtype=torch.float64)
    want[:, 1] = N * float(grads.double().sum()) * value / 2
    want[:, 0] = -want[:, 1]
    return t, want


def _dbias(ops, t, dev, resolution=0):
    d = {k: x.to(dev) for k, x in t.items()}
    d["bias"].requires_grad_()
    o = ops.cross_attention(d["q"], d["k"], d["v"], bias=d["bias"], q_pos=d["q_pos"], k_pos=d["k_pos"],
                            resolution=resolution)
    return torch.autograd.grad(o, d["bias"], d["go"])[0].cpu().double()


# p = exp2(x - log2(Lk)) is off by the logarithm's and the exponential's last places: 2^-21 of 6 or 7, times ln 2, and
# a rounding each; all p alike, so D stays 0. The sums are exact, the result rounds once, the sum over rows once.
TOL = 2.0 ** -19


@pytest.mark.parametrize("value", [2.0 ** -24, 2.0 ** -22, 2.0 ** -18, 2.0 ** -10, 1.0])
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_small_negative_terms_count_as_positive_ones_do(ops, gpu, form, dtype, value):
    """Column 0 gets the negatives of column 1's terms, none of them lost."""
    t, want = _even(form, dtype, value, torch.ones(form[1]))
    got = _dbias(ops, t, gpu)
    assert ((got - want).abs() <= TOL * want.abs()).all(), (got, want)


@pytest.mark.parametrize("value, grad", [(2.0 ** -40, 1.0), (2.0 ** -100, 1.0), (2.0 ** -30, 2.0 ** -50),
                                         (2.0 ** 26, 1.0), (2.0 ** 28, 1.0), (2.0 ** 60, 2.0 ** 30), (2.0 ** 30, 2.0 ** -60)])
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_sums_of_any_magnitude(ops, gpu, form, dtype, value, grad):
    """Neither lost below the cells' last place nor wrapped above their first:
    a cell is shared by many lanes and waves, and all of them add to one here."""
    t, want = _even(form, dtype, value, torch.full((form[1],), grad))
    got = _dbias(ops, t, gpu)
    assert ((got - want).abs() <= TOL * want.abs()).all(), (got, want)


@pytest.mark.parametrize("big", [2.0 ** 10, 2.0 ** 20])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_one_rows_large_gradient_leaves_the_others(ops, gpu, form, dtype, big):
    """Row 0's gradient is far larger and its distances have columns of their
    own: the other columns are as exact beside it as alone."""
    if dtype == FP16:
        big = min(big, 2.0 ** 15)
    grads = torch.ones(form[1])
    grads[0] = big
    t, want = _even(form, dtype, 2.0 ** -6, grads)
    t["q_pos"][:, 0] = 12   # distances 2 and 3, with two buckets an octave columns 2 and 3
    far = want[:, :2] * big / float(grads.double().sum())
    want[:, :2] -= far
    want[:, 2:] = far
    got = _dbias(ops, t, gpu, resolution=1)
    assert ((got - want).abs() <= TOL * want.abs()).all(), (got, want)


@pytest.mark.parametrize("std", [1e-6, 1e-4, 1e-2, 1.0, 1e3, 1e6])
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("case", [(5, 6, 40, 4, 2, 24), (3, 70, 150, 4, 2, 24), (30, 128, 130, 4, 1, 24)], ids=str)
def test_values_of_any_deviation(ops, gpu, case, dtype, std):
    """Random inputs, values scaled: within the bounds of float32 products and
    sums, as at a deviation of one."""
    N, Lq, Lk, Hq, Hkv, dh = case
    g = torch.Generator().manual_seed(Lk)
    r = lambda *s: torch.randn(*s, generator=g)
    t = dict(q=r(N, Lq, Hq, dh), k=r(N, Lk, Hkv, dh), v=r(N, Lk, Hkv, dh) * std, go=r(N, Lq, Hq, dh))
    t = {k: x.to(dtype) for k, x in t.items()}
    t["bias"] = r(Hq, 12)
    t["q_pos"], t["k_pos"] = (torch.randint(0, 3000, (N, L), generator=g) for L in (Lq, Lk))
    cols = ho.columns(t["q_pos"], t["k_pos"], 12, 0, False)
    wide = {k: x.float() if k in ("q", "k", "v", "go") else x for k, x in t.items() if k not in ("q_pos", "k_pos")}
    want, bound = ho.attend(**wide, cols=cols)
    got = _dbias(ops, t, gpu)
    bad = ~((got - want["dbias"]).abs() <= bound["dbias"])
    assert not bad.any(), float(((got - want["dbias"]).abs() / bound["dbias"]).max())
