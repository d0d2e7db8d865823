"""Rows whose every score is -inf though candidates are in: no distribution, so
NaN, and nothing for the other rows."""
import math

import pytest
import torch

from test_gpu_candidates import BF16, FP16, FP32, _inputs, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,V,D", [(5, 64, 32), (300, 700, 64), (1100, 300, 100)])
@pytest.mark.parametrize("biased", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("taught", [False, True], ids=["labels", "teacher"])
def test_every_score_infinite(ops, gpu, N, V, D, dtype, biased, taught):  # noqa: F811
    g, h, w, b, go = _inputs(N + V, N, V, D, dtype, biased)
    w[:, 3] = w[:, 3].abs() + 0.5
    h[2, 3] = -math.inf               # every product with it is -inf
    t = torch.randint(0, V, (N, 1), generator=g)
    if biased:
        b[::7] = -math.inf
        t = t // 7 * 7 + 1            # (none of those)
        t[t >= V] = 1
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b) if x is not None]
    kw = dict(bias=leaves[2]) if biased else {}
    loss = (ops.distillation(leaves[0], leaves[1], t.to(gpu), torch.zeros(N, 1, device=gpu), **kw) if taught
            else ops.cross_entropy(leaves[0], leaves[1], t[:, 0].to(gpu), **kw))
    grads = torch.autograd.grad(loss, leaves, go.to(gpu))
    others = torch.arange(N, device=gpu) != 2
    assert torch.isnan(loss[2]) and torch.isfinite(loss[others]).all()
    assert torch.isnan(grads[0][2]).all() and torch.isfinite(grads[0][others]).all()
    with torch.no_grad():
        alone = (ops.distillation(h.to(gpu), w.to(gpu), t.to(gpu), torch.zeros(N, 1, device=gpu), **kw) if taught
                 else ops.cross_entropy(h.to(gpu), w.to(gpu), t[:, 0].to(gpu), **kw))
    assert torch.isnan(alone[2]) and torch.isfinite(alone[others]).all()


def test_finite_rows_whose_scores_overflow(ops, gpu):  # noqa: F811
    h = torch.zeros(3, 8, device=gpu)
    h[0], h[1] = -3e38, 1.0
    w = torch.full((40, 8), 10.0, device=gpu)
    loss = ops.cross_entropy(h.requires_grad_(), w, torch.tensor([3, 3, -1], device=gpu))
    dh = torch.autograd.grad(loss.sum(), h)[0]
    assert torch.isnan(loss[0]) and abs(float(loss[1]) - math.log(40)) < 1e-5 and loss[2] == 0
    assert torch.isnan(dh[0]).all() and torch.isfinite(dh[1:]).all()
