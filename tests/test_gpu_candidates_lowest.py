"""A bias of float32's lowest value as a mask: a candidate that is in, with a
weight of 0 beside others; a row that wants it has a loss of that size."""
import math

import pytest
import torch

import candidates_oracle as co
from test_gpu_candidates import BF16, FP16, FP32, _close, _inputs, ops  # noqa: F401

pytestmark = pytest.mark.gpu
LOW = torch.finfo(FP32).min


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,V,D", [(5, 64, 32), (300, 700, 64), (1100, 300, 100), (4500, 90, 40)])
def test_labels(ops, gpu, N, V, D, dtype):  # noqa: F811
    g, h, w, b, go = _inputs(N + V, N, V, D, dtype, True)
    masked = torch.rand(V, generator=g) < 0.3
    masked[0], masked[1], masked[2] = True, False, True
    b[masked] = LOW
    b[2] = LOW * 0.75                 # in base 2 past the range as well
    t = torch.randint(0, V, (N,), generator=g)
    t[0], t[1], t[2] = 0, 1, 2
    # the score's own digits are lost beside the mask: half a step of it
    want, bound = co.loss(h, w, *co.labels(t), go, b)
    out = masked[t]
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu), bias=leaves[2])
    got = loss.detach().cpu().double()
    assert bool(((got - want["loss"]).abs()[out] <= 2.0 ** -23 * want["loss"].abs()[out]).all())
    # (the oracle's bounds are of the largest score of a row: those of the candidates that count)
    clean = b.clone()
    clean[masked] = -math.inf
    t_in = torch.where(out, -1, t)
    want, bound = co.loss(h, w, *co.labels(t_in), go, clean)
    _close(torch.where(out.to(gpu), 0.0, loss.detach()), want["loss"], bound["loss"], "loss")
    # gradients: p - q with q of the masked targets too
    dh, dw, db = torch.autograd.grad(loss, leaves, go.to(gpu))
    rows = ~out.to(gpu)
    _close(torch.where(rows[:, None], dh, 0.0), want["dh"], bound["dh"], "dh")
    p = torch.softmax((h.double() @ w.double().t() + clean.double()), 1)
    exact = (go.double()[:, None] * p).sum(0) - torch.zeros(V, dtype=torch.float64).index_add_(0, t, go.double())
    size = (go.double()[:, None] * p).sum(0) + torch.zeros(V, dtype=torch.float64).index_add_(0, t, go.double())
    # weights of 1e-5 of themselves (scores of 10 with 100 terms in float32), sums of N terms
    assert bool(((db.cpu().double() - exact).abs() <= (2e-5 + N * 2.0 ** -24) * size + 1e-30).all())


def test_every_candidate(ops, gpu):  # noqa: F811
    """Equal masks everywhere: equal weights, labels and teacher."""
    for N, V in ((3, 50), (300, 500)):
        h, w = torch.randn(N, 32, device=gpu), torch.randn(V, 32, device=gpu)
        b = torch.full((V,), LOW, device=gpu)
        t = torch.randint(0, V, (N, 2), device=gpu)
        t[:, 1] = (t[:, 0] + 1) % V
        assert (ops.cross_entropy(h, w, t[:, 0], bias=b) - math.log(V)).abs().max() < 1e-5
        loss = ops.distillation(h, w, t, torch.zeros(N, 2, device=gpu), bias=b)
        assert (loss - math.log(V / 2)).abs().max() < 1e-5


@pytest.mark.parametrize("T", [0.5, 1.0, 2.0])
def test_teacher(ops, gpu, T):  # noqa: F811
    """Half of a teacher's weight on a masked candidate: T times half the mask."""
    N, V, D = 40, 90, 32
    g, h, w, b, go = _inputs(5, N, V, D, FP32, True)
    b[7] = LOW
    ids = torch.tensor([[7, 3]]).expand(N, 2)
    with torch.no_grad():
        got = ops.distillation(h.to(gpu), w.to(gpu), ids.to(gpu), torch.zeros(N, 2, device=gpu), bias=b.to(gpu),
                               temperature=T).cpu().double()
    want = -T * 0.5 * LOW
    assert bool(((got - want).abs() <= 2.0 ** -22 * want).all())
