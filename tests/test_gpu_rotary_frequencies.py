"""Frequencies that have no angle make their pairs NaN, in both passes and in
every form, and no others."""
import math

import pytest
import torch

from test_gpu_rotary import BF16, FP16, FP32, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,L,H,dh,P,dtype", [
    (1, 5, 2, 16, 8, FP32),
    (3, 1, 1, 43, 8, BF16),
    (1, 4, 1, 1040, 520, FP16),     # a lane forms its own
    (700, 41, 1, 43, 16, BF16),     # turned in LDS
])
@pytest.mark.parametrize("inter", [False, True], ids=["halves", "interleaved"])
def test_not_finite(ops, gpu, N, L, H, dh, P, dtype, inter):  # noqa: F811
    g = torch.Generator().manual_seed(dh)
    x = torch.randn(N, L, H, dh, generator=g).to(dtype).to(gpu).requires_grad_()
    pos = torch.randint(-1000, 1000, (N, L), generator=g).to(gpu)
    pos[0, 0] = 0   # (0 times an infinity is no angle either)
    freqs = 100.0 ** (-torch.arange(P, dtype=torch.float64) / P)
    bad = torch.zeros(P, dtype=torch.bool)
    for i, f in ((1, math.nan), (2, math.inf), (4, -math.inf), (6, 2.0 ** 128), (7, -1e300)):
        freqs[i], bad[i] = f, True
    y = ops.rotate(x, None, pos, None, freqs.to(gpu), interleaved=inter)[0]
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    lost = torch.zeros(dh, dtype=torch.bool)
    at = bad.nonzero()[:, 0]
    lost[torch.cat([2 * at, 2 * at + 1] if inter else [at, at + P])] = True
    for t in (y, dx):
        assert torch.equal(torch.isnan(t).cpu(), lost.expand(t.shape)) and torch.isfinite(t[..., ~lost.to(gpu)]).all()
