"""Rotary positions over the forms that sizes choose: lanes of whole and of
shared channels, rows of odd bytes, a channel or pair at a time, more pairs
than a workgroup forms the steps of, several workgroups a side."""
import pytest
import torch

import candidates_oracle as co
from test_gpu_rotary import BF16, FP16, FP32, _close, ops  # noqa: F401

pytestmark = pytest.mark.gpu

FORMS = [  # N, L, H, dh, pairs, dtype
    (9, 13, 3, 44, 22, BF16),     # a last lane that shares its neighbour's channels
    (9, 13, 3, 44, 21, FP32),
    (7, 11, 2, 43, 21, BF16),     # rows of odd bytes, one channel that is not turned
    (7, 11, 2, 43, 17, FP16),
    (7, 11, 2, 29, 4, FP16),      # ... and more of them than a load
    (5, 6, 2, 22, 3, BF16),       # fewer pairs than a lane takes
    (5, 6, 2, 23, 1, FP16),
    (5, 6, 2, 22, 1, FP32),
    (5, 6, 2, 22, 0, FP16),       # a copy
    (5, 6, 2, 5, 0, FP32),
    (2, 3, 1, 1030, 515, FP16),   # more pairs than a workgroup keeps
    (2, 3, 1, 1031, 513, FP32),
    (40, 31, 1, 100, 32, BF16),   # several workgroups
    # rows of an odd number of channels, many: turned in LDS, stretches that end anywhere
    (601, 35, 3, 43, 21, BF16),
    (700, 41, 1, 43, 16, FP16),
    (257, 33, 2, 127, 63, FP16),
    (600, 251, 1, 3, 1, BF16),
    (300, 43, 2, 43, 21, FP32),
    (150, 41, 1, 121, 5, FP32),
]


@pytest.mark.parametrize("inter", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("N,L,H,dh,P,dtype", FORMS)
def test_forms(ops, gpu, N, L, H, dh, P, dtype, inter):  # noqa: F811
    g = torch.Generator().manual_seed(dh + P)
    q, k = torch.randn(N, L, H, dh, generator=g).to(dtype), torch.randn(N, 1, 1, dh, generator=g).to(dtype)
    qp, kp = (torch.randint(-3_000_000, 3_000_000, (N, n), generator=g) for n in (L, 1))
    freqs = 500.0 ** (-torch.arange(P, dtype=torch.float64) / max(P, 1))
    args = [x.to(gpu) for x in (q, k, qp, kp, freqs)]
    got = ops.rotate(*args, interleaved=inter)
    for y, x, p, what in ((got[0], q, qp, "q"), (got[1], k, kp, "k")):
        _close(y, *co.rotate(x, p, freqs, inter), what)
    for y, z in zip(got, ops.rotate(*args, interleaved=inter)):
        assert torch.equal(y, z)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=["fp32", "bf16", "fp16"])
def test_nan_and_infinities_stay_in_their_pairs(ops, gpu, dtype):  # noqa: F811
    x = torch.ones(1, 2, 2, 44, dtype=dtype)
    x[0, 0, 0, 3], x[0, 1, 1, 43] = float("nan"), float("inf")
    pos = torch.tensor([[5, 7]])
    freqs = 100.0 ** (-torch.arange(21, dtype=torch.float64) / 21)
    y = ops.rotate(x.to(gpu), None, pos.to(gpu), None, freqs.to(gpu))[0].cpu()
    bad = ~torch.isfinite(y)
    assert bad[0, 0, 0, [3, 24]].all() and bad[0, 1, 1, 43] and int(bad.sum()) == 3
