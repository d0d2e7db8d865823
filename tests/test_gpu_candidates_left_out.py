"""Candidates that are left out (bias -inf) have gradients of 0 whatever the
rows and their gradients hold."""
import math

import pytest
import torch

from test_gpu_candidates import BF16, FP16, FP32, _inputs, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,V,D", [(5, 70, 32), (40, 200, 64), (300, 20_011, 100), (1200, 300, 256)])
@pytest.mark.parametrize("what", [math.nan, math.inf, "gradient"], ids=["nan", "inf", "gradient"])
@pytest.mark.parametrize("taught", [False, True], ids=["labels", "teacher"])
def test_not_finite_rows_leave_them(ops, gpu, N, V, D, dtype, what, taught):  # noqa: F811
    g, h, w, b, go = _inputs(N + V, N, V, D, dtype, True)
    t = torch.randint(1, V // 2, (N, 1), generator=g) * 2   # (the odd ones are left out)
    b[1::2] = -math.inf
    w[1::2] = math.nan
    if what == "gradient":
        go[2] = math.inf
    else:
        h[2, 3] = what
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    loss = (ops.distillation(leaves[0], leaves[1], t.to(gpu), torch.zeros(N, 1, device=gpu), bias=leaves[2]) if taught
            else ops.cross_entropy(leaves[0], leaves[1], t[:, 0].to(gpu), bias=leaves[2]))
    dh, dw, db = torch.autograd.grad(loss, leaves, go.to(gpu))
    assert not dw[1::2].any() and not db[1::2].any()
    assert not torch.isfinite(dw[::2]).all() and not torch.isfinite(db[::2]).all()
    others = torch.arange(N, device=gpu) != 2
    assert torch.isfinite(dh[others]).all() and torch.isfinite(loss[others]).all()
