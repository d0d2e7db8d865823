"""Infinities and NaN in live places of the cross attention: they reach what
the definition lets them reach, and nothing else."""
import math

import pytest
import torch

from test_gpu_history import _rand

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16

FORMS = [  # N, Lq, Lk, Hq, Hkv, dh
    (3, 8, 16, 4, 2, 16),      # one wave a sequence
    (3, 40, 50, 4, 2, 16),     # all keys in one tile
    (3, 40, 200, 4, 2, 16),
    (3, 1, 900, 4, 2, 16),     # a long history in parts
    (96, 128, 130, 4, 2, 16),  # eight waves a workgroup, two heads of the same queries
    (70, 128, 130, 3, 1, 16),
]


@pytest.fixture(scope="module")
def ops(gpu):
    from starry_unigraph.native import history
    return history


def _inputs(form, dtype, mask=False):
    N, Lq, Lk, Hq, Hkv, dh = form
    g = torch.Generator().manual_seed(Lk)
    t = dict(q=_rand(g, N, Lq, Hq, dh, dtype=dtype), k=_rand(g, N, Lk, Hkv, dh, dtype=dtype),
             v=_rand(g, N, Lk, Hkv, dh, dtype=dtype), go=_rand(g, N, Lq, Hq, dh, dtype=dtype), bias=_rand(g, Hq, 12))
    t["q_pos"], t["k_pos"] = (torch.randint(0, 500, (N, L), generator=g) for L in (Lq, Lk))
    t["key_mask"] = torch.rand(N, Lk, generator=g) < 0.7 if mask else None
    return t


def _run(ops, t, dev):
    d = {k: x.to(dev) if x is not None else None for k, x in t.items()}
    leaves = [d[k].requires_grad_() for k in ("q", "k", "v", "bias")]
    o = ops.cross_attention(d["q"], d["k"], d["v"], bias=d["bias"], q_pos=d["q_pos"], k_pos=d["k_pos"],
                            key_mask=d["key_mask"])
    return [x.detach().cpu() for x in (o, *torch.autograd.grad(o, leaves, d["go"]))]


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_a_nan_score_spoils_its_row_and_what_sums_over_it(ops, gpu, form, dtype):
    """One query row's NaN: its o and dq, and dk and dv of every key that it
    attends to; no other row, head or sequence."""
    t = _inputs(form, dtype)
    clean = _run(ops, t, gpu)
    n, i, h = 1, form[1] - 1, 1
    t["q"][n, i, h, 3] = math.nan
    o, dq, dk, dv, db = _run(ops, t, gpu)
    for got, want in ((o, clean[0]), (dq, clean[1])):
        assert torch.isnan(got[n, i, h]).all()
        got[n, i, h] = want[n, i, h]
        assert torch.equal(got, want)
    for got, want in ((dk, clean[2]), (dv, clean[3])):
        assert torch.isnan(got[n, :, 0]).all()   # (head 1's key head)
        got[n, :, 0] = want[n, :, 0]
        assert torch.equal(got, want)
    assert torch.isnan(db[h]).any()


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_one_nan_score_of_a_row_spoils_the_others(ops, gpu, form, dtype):
    """A live key's NaN: the softmax of every row of its key head is NaN at
    every key, so o, dq, dk and dv of that head are."""
    t = _inputs(form, dtype)
    clean = _run(ops, t, gpu)
    G = form[3] // form[4]
    t["k"][2, form[2] // 2, 0, 5] = math.nan
    out = _run(ops, t, gpu)
    for got, want, heads in zip(out[:4], clean, (G, G, 1, 1)):
        assert torch.isnan(got[2, :, :heads]).all()
        got[2, :, :heads] = want[2, :, :heads]
        assert torch.equal(got, want)
    assert torch.isnan(out[4][:G]).any(1).all()


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_masked_keys_have_no_gradient_beside_an_infinite_one(ops, gpu, form, dtype, bad):
    """A gradient of o that is not finite: keys left out by the mask, and rows
    whose mask leaves nothing, have zero gradients all the same."""
    t = _inputs(form, dtype, mask=True)
    t["key_mask"][0] = False
    clean = _run(ops, t, gpu)
    t["go"][0, 0, :, 2] = bad   # rows without a live key: nothing changes anywhere
    for got, want in zip(_run(ops, t, gpu), clean):
        assert torch.equal(got, want)
    t["go"][1, form[1] - 1, 0, 4] = bad
    _, dq, dk, dv, db = _run(ops, t, gpu)
    dead = ~t["key_mask"]
    assert not dk[dead].any() and not dv[dead].any()
    # (D = <do, o> is an infinity: ds is one too at keys whose dp has the other sign, and NaN elsewhere)
    assert not torch.isfinite(dk[1, ~dead[1], 0]).any()
    dq[1, form[1] - 1, 0] = clean[1][1, form[1] - 1, 0]
    assert torch.equal(dq, clean[1])
    for got, want in ((dk, clean[2]), (dv, clean[3])):
        got[1, :, 0] = want[1, :, 0]
        assert torch.equal(got, want)
    assert not torch.isfinite(db[0]).all()


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_masked_keys_have_no_gradient_beside_an_infinite_query(ops, gpu, form):
    t = _inputs(form, FP32, mask=True)
    t["q"][1, 0, 0, 4] = math.inf
    _, _, dk, dv, _ = _run(ops, t, gpu)
    dead = ~t["key_mask"]
    assert not dk[dead].any() and not dv[dead].any()
