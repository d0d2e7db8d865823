"""The rows' gradients of the losses over all candidates where one candidate has
nearly all of a row's probability: they are of 1 - p there, and a weight that is
rounded to the type beside an exact 1 would leave none of its digits.

The kernels' coefficient of a candidate is a_v / sum a - q_v with a_v = p_v (1 + d_v),
|d_v| <= d = u + 2 es + 4 F: the rounding of a weight to the type (u = eps / 2; 0
in float32), a score's error es (its products, sums and factors in float32, F =
2^-24 a step) in the weight and its exponential's own. The error's share by d is p_v sum_w
p_w (d_v - d_w) / (1 + sum p d), at most 2 d / (1 - d) p_v (1 - p_v): it vanishes with
1 - p. What is left are the float32 sums: F (V / 16 + 64) p_v for those of weights and
products (a step of 16 or 32 candidates a rounding, the joins), F (K + 16) q_v for the targets'."""
import math

import pytest
import torch

import candidates_oracle as co
from test_gpu_candidates import BF16, FP16, FP32, _close, _rand, ops  # noqa: F401

pytestmark = pytest.mark.gpu
F = 2.0 ** -24


def _rows_grad(h, w, b, ids, q, go, T=1.0):
    """(dh, its bound) in float64."""
    u = co.unit(h.dtype) if h.dtype != FP32 else 0.0
    H, W, b = h.double(), w.double(), b.double()
    V, D = W.shape
    s = (H @ W.t() + b) / T
    size = (H.abs() @ W.abs().t() + b.abs()) / T
    es = F * (D + 8) * size.amax(1, keepdim=True) + 4 * F * s.abs().amax(1, keepdim=True)
    p = torch.softmax(s, 1)
    rest = torch.zeros_like(p)   # 1 - p without the cancellation
    for v in range(V):
        if bool((p[:, v] > 0.25).any()):
            rest[:, v] = p[:, :v].sum(1) + p[:, v + 1:].sum(1)
        else:
            rest[:, v] = 1 - p[:, v]
    Q = torch.zeros_like(p).scatter_add_(1, ids, q)
    d = u + 2 * es + 4 * F
    err = 2 * d / (1 - d) * p * rest + F * (V / 16 + 64) * p + F * (ids.shape[1] + 16) * Q
    if h.dtype == FP16:   # weights under 2^-24 of what is put at 2^7 and more: half a step
        err = err + 2.0 ** -31
    G = go.double()[:, None] * T
    coef = torch.where(Q == 1, -rest, p - Q)
    want, bound = G * (coef @ W), G.abs() * (err @ W.abs())
    t = torch.finfo(h.dtype)
    return want, bound + t.eps / 2 * (want.abs() + bound) + t.smallest_normal * t.eps


SHAPES = [  # N, V, D: few rows, half and whole tiles, rows in order, pieces of the table, the widest
    (40, 64, 64),
    (3, 200, 100),
    (100, 200, 172),
    (300, 300, 256),
    (1100, 100, 43),
    (300, 20_011, 100),
    (5, 5000, 256),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("gap", [2.0, 5.0, 5.5, 9.0])
@pytest.mark.parametrize("N,V,D", SHAPES)
def test_target_with_nearly_all(ops, gpu, N, V, D, gap, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(N + D)
    h, w = _rand(g, N, D, dtype=dtype), _rand(g, V, D, dtype=dtype, std=0.2 / math.sqrt(D))
    b = torch.full((V,), -40.0)
    b[0], b[40] = 0.0, gap        # in two steps of 32 candidates: the second one's weight is over the first's maximum
    go = torch.rand(N, generator=g) + 0.5
    t = torch.full((N,), 40)
    want, bound = _rows_grad(h, w, b, t[:, None], torch.ones(N, 1, dtype=torch.float64), go)
    x, y = h.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
    loss = ops.cross_entropy(x, y, t.to(gpu), bias=b.to(gpu))
    _close(torch.autograd.grad(loss, x, go.to(gpu))[0], want, bound, "dh")
    alone = h.to(gpu).requires_grad_()   # without the table's gradient
    loss = ops.cross_entropy(alone, y.detach(), t.to(gpu), bias=b.to(gpu))
    _close(torch.autograd.grad(loss, alone, go.to(gpu))[0], want, bound, "dh alone")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V,D,T", [(40, 64, 64, 1.0), (300, 700, 172, 2.0), (7, 200, 256, 0.5)])
def test_student_near_its_teacher(ops, gpu, N, V, D, T, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(V)
    h, w = _rand(g, N, D, dtype=dtype), _rand(g, V, D, dtype=dtype, std=0.2 / math.sqrt(D))
    b = torch.full((V,), -60.0 * T)
    b[0], b[40] = 0.0, 5.5 * T
    go = torch.rand(N, generator=g) + 0.5
    ids = torch.tensor([[0, 40, -1]]).expand(N, 3)
    z = torch.tensor([[0.0, 5.0 * T, 9.0]]).expand(N, 3).contiguous()
    i, q, _, _ = co.teacher(ids, z, T)
    want, bound = _rows_grad(h, w, b, i, q, go, T)
    x = h.to(gpu).requires_grad_()
    loss = ops.distillation(x, w.to(gpu).requires_grad_(), ids.to(gpu), z.to(gpu), bias=b.to(gpu), temperature=T)
    _close(torch.autograd.grad(loss, x, go.to(gpu))[0], want, bound, "dh")
