"""Sums of float32 rows of more than 128 channels that are rescaled in place: maxima
that grow at every step of the table, at none, and at one step for some rows
only."""
import pytest
import torch

import candidates_oracle as co
from test_gpu_candidates import FP32, _check, _inputs, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [129, 172, 192, 193, 256])
@pytest.mark.parametrize("N,V", [(3, 1500), (130, 1500), (300, 5003)])
@pytest.mark.parametrize("how", ["grows", "falls", "once", "some rows"])
def test_growing_maxima(ops, gpu, N, V, D, how):  # noqa: F811
    g, h, w, b, go = _inputs(N + D, N, V, D, FP32, True)
    t = torch.randint(0, V, (N,), generator=g)
    if how == "grows":       # 9 or 10 powers of two a step of 32
        b += torch.arange(V) * 0.21
    elif how == "falls":
        b -= torch.arange(V) * 0.21
    elif how == "once":
        b[V // 2:] += 60.0
    else:                    # a channel that odd rows alone have, and late candidates alone
        h[:, 5] = torch.where(torch.arange(N) % 2 == 1, 8.0, 0.0)
        w[:, 5] = torch.where(torch.arange(V) >= V - 100, 3.0, 0.0)
    want, bound = co.loss(h, w, *co.labels(t), go, b)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu), bias=leaves[2])
    _check(loss, leaves, go, want, bound)
