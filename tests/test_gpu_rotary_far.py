"""Rotary positions far from zero: stamps in seconds to nanoseconds and the ends
of int64, each channel against the definition with exact angles.

An angle is within 2^-32 of a turn (0.03 x 2^-24); as a float within an eighth of a
turn it is off by 3 roundings of 0.79, 2.4 x 2^-24, and by as much its sine and cosine,
which add 1 x 2^-24 (0.03 of it their series'); the gain and its product 2, the
products and sum of a pair 1 and 1.4: 8 x 2^-24 = 2^-21 of gain (|a| + |b|)."""
import math
from fractions import Fraction

import pytest
import torch

import candidates_oracle as co
from test_gpu_rotary import BF16, FP16, FP32, _close, ops  # noqa: F401

pytestmark = pytest.mark.gpu
STAMPS = [0, 1, -1, 1_700_000_000, 1_700_000_000_123, 1_700_000_000_123_456, 1_700_000_000_123_456_789,
          -1_699_999_999_999_999_999, 1 << 62, -(1 << 62) - 12345, (1 << 63) - 1, -(1 << 63)]


def _rotate(x, pos, freqs, interleaved=False, gain=1.0, way=1.0):
    """(the rotated tensor, the bound of the module's docstring)."""
    P = len(freqs)
    turns = [Fraction(f) * co.INV_2PI for f in freqs.tolist()]
    angle = torch.tensor([[2 * math.pi * float(t * f % 1) for f in turns] for t in pos.flatten().tolist()],
                         dtype=torch.float64).view(*pos.shape, P)
    c, s = gain * torch.cos(angle)[:, :, None], way * gain * torch.sin(angle)[:, :, None]
    at = torch.arange(P)
    i, j = (2 * at, 2 * at + 1) if interleaved else (at, at + P)
    out, bound = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    a, b = out[..., i].clone(), out[..., j].clone()
    out[..., i], out[..., j] = a * c - b * s, a * s + b * c
    bound[..., i] = bound[..., j] = (a.abs() + b.abs()) * abs(gain) * 2.0 ** -21
    t = torch.finfo(x.dtype)
    rounded = bound + t.eps / 2 * (out.abs() + bound) + t.smallest_normal * t.eps
    rounded[..., 2 * P:] = 0.0
    return out, rounded


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("inter", [False, True], ids=["halves", "interleaved"])
def test_stamps(ops, gpu, dtype, inter):  # noqa: F811
    g = torch.Generator().manual_seed(0)
    pos = torch.tensor([STAMPS, [s ^ 0x5A5 for s in STAMPS]])
    freqs = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    q, k = (torch.randn(2, len(STAMPS), H, 67, generator=g).to(dtype) for H in (3, 1))
    gq, gk = torch.randn(q.shape, generator=g).to(dtype), torch.randn(k.shape, generator=g).to(dtype)
    leaves = [x.to(gpu).requires_grad_() for x in (q, k)]
    outs = ops.rotate(*leaves, pos.to(gpu), pos.flip(1).to(gpu), freqs.to(gpu), interleaved=inter, gain=1.25)
    grads = torch.autograd.grad(outs, leaves, (gq.to(gpu), gk.to(gpu)))
    for got, x, p, way, what in ((outs[0], q, pos, 1.0, "q"), (outs[1], k, pos.flip(1), 1.0, "k"),
                                 (grads[0], gq, pos, -1.0, "dq"), (grads[1], gk, pos.flip(1), -1.0, "dk")):
        _close(got, *_rotate(x, p, freqs, inter, 1.25, way), what)


def test_any_frequency(ops, gpu):  # noqa: F811
    """Frequencies from far under a turn over all of int64 to far over one a unit."""
    freqs = torch.tensor([1.0, -0.3, 2 * math.pi / 3600, 1e-9, -1e-18, 2.0 ** -64, 1e-30, 0.0, 7.5, 1e6, -2.0 ** 52,
                          1.5 * 2.0 ** 53, 1e20, 2.0 ** 116, 1.9 * 2.0 ** 127, 5e-324], dtype=torch.float64)
    x = torch.randn(1, len(STAMPS), 2, 32, generator=torch.Generator().manual_seed(1))
    pos = torch.tensor([STAMPS])
    got = ops.rotate(x.to(gpu), None, pos.to(gpu), None, freqs.to(gpu))[0]
    _close(got, *_rotate(x, pos, freqs), "x")


def test_many_pairs_and_odd_heads(ops, gpu):  # noqa: F811
    """The forms that each lane forms its steps in, and that turn in LDS."""
    g = torch.Generator().manual_seed(2)
    pos = torch.tensor([STAMPS])
    freqs = 500.0 ** (-torch.arange(515, dtype=torch.float64) / 515)
    x = torch.randn(1, len(STAMPS), 1, 1030, generator=g).to(FP16)
    _close(ops.rotate(x.to(gpu), None, pos.to(gpu), None, freqs.to(gpu))[0], *_rotate(x, pos, freqs), "many")
    freqs = 500.0 ** (-torch.arange(3, dtype=torch.float64) / 3)
    pos = torch.randint(-(1 << 63), (1 << 63) - 1, (350, len(STAMPS)), generator=g)
    x = torch.randn(350, len(STAMPS), 8, 127, generator=g).to(BF16)
    _close(ops.rotate(x.to(gpu), None, pos.to(gpu), None, freqs.to(gpu))[0], *_rotate(x, pos, freqs), "odd")


def test_scores_of_stamps_depend_on_distances(ops, gpu):  # noqa: F811
    """Nanosecond stamps with frequencies of a radian a second and slower."""
    g = torch.Generator().manual_seed(3)
    freqs = ops.frequencies(64, scaling="linear", factor=1e9, device=gpu)
    q, k = (torch.randn(1, 1, 2, 64, generator=g).to(gpu) for _ in range(2))
    scores = []
    for at in (0, 1_700_000_000_123_456_789, -(1 << 62)):
        pos = [torch.tensor([[t]], device=gpu) for t in (at + 40_000_000_000, at)]
        a, b = ops.rotate(q, k, *pos, freqs)
        scores.append((a.double() * b.double()).sum(-1))
    # each rotated value within 2^-21 of its pair's sizes, 64 products of two of them
    most = float((2.0 ** -20 * 2 * q.norm(dim=-1).double() * k.norm(dim=-1).double()).max())
    for s in scores[1:]:
        assert float((s - scores[0]).abs().max()) <= 2 * most
