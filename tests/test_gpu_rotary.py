"""Rotary positions on the GPU against their definition in float64 with angles
from exact integers (candidates_oracle): every type, both layouts, parts of a
head, far and negative positions, strided inputs; gradients; other calls."""
import math

import pytest
import torch

import candidates_oracle as co

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops(gpu):
    from starry_unigraph.native import rotary
    return rotary


def _close(got, want, bound, what):
    most = torch.finfo(got.dtype).max
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    # (a value past the type's largest is rounded to inf)
    bad = ~(((got - want).abs() <= bound) | ((got == want.sign() * math.inf) & (want.abs() + bound > most)))
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs()[bad].max()))


CASES = [  # N, Lq, Lk, Hq, Hkv, dh, pairs, dtype, interleaved
    (1, 1, 1, 1, 1, 2, 1, FP32, False),
    (1, 1, 1, 1, 1, 1, 0, FP32, True),
    (3, 1, 5, 2, 2, 50, 25, FP32, False),
    (3, 4, 1, 2, 1, 50, 25, FP32, True),
    (2, 7, 9, 4, 2, 43, 21, BF16, True),
    (2, 7, 9, 4, 1, 43, 21, BF16, False),
    (2, 33, 3, 3, 3, 64, 16, FP16, False),
    (2, 3, 33, 8, 2, 128, 64, BF16, False),
    (2, 3, 33, 8, 2, 128, 64, FP16, True),
    (5, 2, 2, 1, 1, 7, 2, FP16, True),
    (5, 2, 2, 1, 1, 300, 9, BF16, False),
]


@pytest.mark.parametrize("N,Lq,Lk,Hq,Hkv,dh,P,dtype,inter", CASES)
def test_rotate(ops, gpu, N, Lq, Lk, Hq, Hkv, dh, P, dtype, inter):
    g = torch.Generator().manual_seed(dh)
    q, k = (torch.randn(N, L, H, dh, generator=g).to(dtype) for L, H in ((Lq, Hq), (Lk, Hkv)))
    qp, kp = (torch.randint(-5000, 2_700_000, (N, L), generator=g) for L in (Lq, Lk))
    freqs = 10000.0 ** (-torch.arange(P, dtype=torch.float64) / max(P, 1))
    gq, gk = torch.randn(q.shape, generator=g).to(dtype), torch.randn(k.shape, generator=g).to(dtype)
    leaves = [x.to(gpu).requires_grad_() for x in (q, k)]
    outs = ops.rotate(*leaves, qp.to(gpu), kp.to(gpu), freqs.to(gpu), interleaved=inter, gain=1.25)
    grads = torch.autograd.grad(outs, leaves, (gq.to(gpu), gk.to(gpu)))
    for got, x, p, way, what in ((outs[0], q, qp, 1.0, "q"), (outs[1], k, kp, 1.0, "k"), (grads[0], gq, qp, -1.0, "dq"),
                                 (grads[1], gk, kp, -1.0, "dk")):
        _close(got, *co.rotate(x, p, freqs, inter, 1.25, way), what)
    alone = ops.rotate(q.to(gpu), None, qp.to(gpu), None, freqs.to(gpu), interleaved=inter, gain=1.25)
    assert alone[1] is None and torch.equal(alone[0], outs[0])


def test_far_positions_and_any_frequency(ops, gpu):
    big = (1 << 62) + 12345
    pos = torch.tensor([[0, 1, -1, 1_700_000_000, -1_700_000_000, 1 << 40, big, -big, -(1 << 63), (1 << 63) - 1]])
    freqs = torch.tensor([1.0, -0.3, 2.0 * math.pi / 3600, 1e-9, 0.0, 7.5], dtype=torch.float64)
    x = torch.randn(1, 10, 1, 12, generator=torch.Generator().manual_seed(1))
    near = torch.tensor([[0, 1, -1, 1_700_000_000, -1_700_000_000, 1 << 40, 5, 6, 7, 8]])
    got = ops.rotate(x.to(gpu), None, near.to(gpu), None, freqs.to(gpu))[0]
    _close(got, *co.rotate(x, near, freqs), "near")
    # beyond a double's digits of the frequency: still a rotation
    far = ops.rotate(x.to(gpu), None, pos.to(gpu), None, freqs.to(gpu))[0].cpu()
    assert torch.allclose(far.square().sum(-1), x.square().sum(-1), rtol=1e-5)
    # frequencies that are whole fractions of a turn: exact at any position
    freqs = 2.0 * math.pi * torch.tensor([0.25, 0.125, 0.5, 0.0625, 1.0, 0.75], dtype=torch.float64)
    _close(ops.rotate(x.to(gpu), None, pos.to(gpu), None, freqs.to(gpu))[0].cpu()[:, :6],
           *(t[:, :6] for t in co.rotate(x, pos, freqs)), "fractions")


def test_strides(ops, gpu):
    g = torch.Generator().manual_seed(2)
    for dtype in (FP32, BF16):
        packed = torch.randn(3, 6, 5, 3, 45, generator=g).to(dtype).to(gpu)   # q, k, v of a row side by side
        q, k, _ = packed[..., 1:45].unbind(3)
        pos = torch.randint(0, 1000, (6, 3), generator=g).to(gpu).t()
        freqs = ops.frequencies(32, device=gpu)
        got = ops.rotate(q, k, pos, pos, freqs, interleaved=True)
        want = ops.rotate(q.contiguous(), k.contiguous(), pos.contiguous(), pos.contiguous(), freqs, interleaved=True)
        turned = ops.rotate(q.transpose(2, 3).contiguous().transpose(2, 3), k, pos, pos, freqs, interleaved=True)
        one = ops.rotate(q[:, :1].expand(3, 6, 5, 44), None, pos, None, freqs, interleaved=True)[0]
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(turned[0], want[0])
        assert torch.equal(one[:, 0], want[0][:, 0])


def test_scores_depend_on_distances(ops, gpu):
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randn(1, 1, 2, 64, generator=g).to(gpu) for _ in range(2))
    freqs = ops.frequencies(64, device=gpu)
    scores = []
    for at in (0, 17, 1_000_000, -123_456_789):
        a, b = ops.rotate(q, k, torch.tensor([[at + 40]], device=gpu), torch.tensor([[at]], device=gpu), freqs)
        scores.append((a * b).sum(-1))
    for s in scores[1:]:   # (64 products of numbers of about 1 in float32)
        assert torch.allclose(s, scores[0], rtol=0, atol=2e-5)


def test_empty_and_captured(ops, gpu):
    freqs = ops.frequencies(8, device=gpu)
    z = torch.zeros(0, 4, 2, 8, device=gpu, requires_grad=True)
    p = torch.zeros(0, 4, dtype=torch.int64, device=gpu)
    out = ops.rotate(z, z, p, p, freqs)
    assert out[0].shape == z.shape and torch.autograd.grad(out[0].sum() + out[1].sum(), z)[0].shape == z.shape
    x = torch.randn(3, 5, 2, 8, device=gpu)
    pos = torch.arange(15, device=gpu).view(3, 5)
    none = torch.zeros(3, 0, 2, 8, device=gpu)
    a, b = ops.rotate(x, none, pos, pos[:, :0], freqs)
    assert b.shape == none.shape and torch.equal(a, ops.rotate(x, None, pos, None, freqs)[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.rotate(x, x, pos, pos, freqs)
    for i in range(3):
        x.copy_(torch.randn(3, 5, 2, 8, device=gpu))
        graph.replay()
        want = ops.rotate(x, x, pos, pos, freqs)
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])
