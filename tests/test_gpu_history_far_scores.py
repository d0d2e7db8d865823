"""Cross attention with scores far from zero: the softmax does not change when
all scores of a row move together."""
import math

import pytest
import torch

import history_oracle as ho
from test_gpu_history import _rand

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16

FORMS = [  # N, Lq, Lk, Hq, Hkv
    (3, 8, 16, 4, 2),        # one wave a sequence
    (3, 40, 50, 4, 2),       # all keys in one tile
    (3, 40, 200, 4, 2),
    (3, 1, 900, 4, 2),       # a long history in parts
    (96, 128, 130, 4, 2),    # eight waves a workgroup, two heads of the same queries
    (70, 128, 130, 3, 1),
]


@pytest.fixture(scope="module")
def ops(gpu):
    from starry_unigraph.native import history
    return history


def _run(ops, t, dev):
    d = {k: x.to(dev) for k, x in t.items()}
    leaves = [d[k].requires_grad_() for k in ("q", "k", "v", "bias")]
    o = ops.cross_attention(d["q"], d["k"], d["v"], bias=d["bias"], q_pos=d["q_pos"], k_pos=d["k_pos"], two_sided=True)
    return [x.detach().cpu() for x in (o, *torch.autograd.grad(o, leaves, d["go"]))]


def _inputs(form, dtype, std=1.0):
    N, Lq, Lk, Hq, Hkv = form
    g = torch.Generator().manual_seed(Lk)
    t = dict(q=_rand(g, N, Lq, Hq, 16, dtype=dtype, std=std), k=_rand(g, N, Lk, Hkv, 16, dtype=dtype, std=std),
             v=_rand(g, N, Lk, Hkv, 16, dtype=dtype), go=_rand(g, N, Lq, Hq, 16, dtype=dtype), bias=torch.zeros(Hq, 4))
    t["q_pos"], t["k_pos"] = (torch.randint(0, 9, (N, L), generator=g) for L in (Lq, Lk))
    return t


@pytest.mark.parametrize("shift", [-1e9, 1e9, -1e4, -2e38])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_a_bias_of_one_value_changes_nothing(ops, gpu, form, dtype, shift):
    """q = 0 and every bucket at the same far value: the scores are equal, each
    key weighs one part in Lk, and every result has the bits of a table of 0."""
    t = _inputs(form, dtype)
    t["q"].zero_()
    want = _run(ops, t, gpu)
    t["bias"].fill_(shift)
    for got, w in zip(_run(ops, t, gpu), want):
        assert torch.equal(got, w)


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_a_rows_weights_sum_to_one_at_large_scores(ops, gpu, form):
    """Scores of thousands: what dv of all keys add up to is what do of all
    rows add up to, within the roundings of sums of Lk weights of a row."""
    N, Lq, Lk, Hq, Hkv = form
    t = _inputs(form, FP32, std=40.0)
    _, _, _, dv, _ = _run(ops, t, gpu)
    go = t["go"].double().unflatten(2, (Hkv, Hq // Hkv))
    want, size = go.sum((1, 3)), go.abs().sum((1, 3))
    # p: a sum of Lk, two exponentials, a logarithm of at most 10 (2^-21 of it, times ln 2); dv: sums over the rows
    tol = ((Lk + Lq * Hq // Hkv + 16) * ho.F + 2.0 ** -20) * size
    assert ((dv.double().sum(1) - want).abs() <= tol).all(), ((dv.double().sum(1) - want).abs() / size).max()


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_buckets_at_the_types_lowest_value(ops, gpu, form, dtype):
    """Keys after the query in buckets of float32's lowest value, a mask in the
    table. Rows with an earlier key ignore them, to the bit as with -inf in the
    table; rows with none weigh their keys equally (their scores differ by less
    than the lowest value's last place), as a table of equal values over q = 0."""
    t = _inputs(form, dtype)
    t["q_pos"][1] = -1   # (sequence 1: every key lies after every query)
    low = torch.finfo(FP32).min
    t["bias"][:, :2], t["bias"][:, 2:] = torch.tensor([0.3, -0.2]), low
    got = _run(ops, t, gpu)
    t["bias"][:, 2:] = -math.inf
    cut = _run(ops, t, gpu)
    rest = torch.arange(form[0]) != 1
    behind = (t["q_pos"][:, :, None] < t["k_pos"][:, None, :]).all(2)   # rows without an earlier key
    keep = rest & ~behind.any(1)
    for g, c in zip(got[:4], cut):
        assert torch.equal(g[keep], c[keep])
    t["bias"].zero_()
    t["q"].zero_()
    flat = _run(ops, t, gpu)
    for i in (0, 3):   # o and dv: what does not depend on q itself
        assert torch.equal(got[i][1], flat[i][1])
    assert torch.isfinite(got[4]).all()


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_rows_of_minus_infinity_are_empty(ops, gpu, form):
    """A table of -inf leaves a row nothing: zeros, as by the key mask."""
    t = _inputs(form, FP32)
    t["bias"].fill_(-math.inf)
    for got in _run(ops, t, gpu):
        assert not got.any()
