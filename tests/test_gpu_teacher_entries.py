"""A teacher's entries that are none, with anything beside the mark that makes
them so."""
import math

import pytest
import torch

import candidates_oracle as co
from test_gpu_candidates import BF16, FP32, _check, _inputs, _rand, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_entries_that_are_none(ops, gpu, dtype):  # noqa: F811
    """A logit of -inf is no entry whatever its id (past the table too), a negative id whatever its logit."""
    N, V, D, K = 40, 90, 32, 6
    g, h, w, b, go = _inputs(3, N, V, D, dtype, True)
    ids, z = torch.randint(0, V, (N, K), generator=g), _rand(g, N, K)
    clean, live = ids.clone(), z.clone()
    clean[::2, 1], live[1::3, 4], clean[2, :], clean[::5, 0] = -1, -math.inf, -1, -1
    want, bound = co.loss(h, w, *co.teacher(clean, live, 1.0), go, b)
    ids, z = clean.clone(), live.clone()
    for at, i in (((1, 4), V), ((4, 4), V + 5), ((7, 4), 1 << 40), ((10, 4), (1 << 63) - 1)):
        ids[at] = i                       # (their logits are -inf)
    ids[2, :3], z[2, :3] = V, -math.inf
    z[::5, 0] = torch.tensor([math.nan, math.inf, -math.inf, 3e38, 0.0, -3e38, math.nan, math.inf])
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    loss = ops.distillation(leaves[0], leaves[1], ids.to(gpu), z.to(gpu), bias=leaves[2])
    _check(loss, leaves, go, want, bound)
    ids[1, 0], z[1, 0] = V, 0.0           # an entry past the table
    loss = ops.distillation(leaves[0], leaves[1], ids.to(gpu), z.to(gpu), bias=leaves[2])
    assert torch.isnan(loss).nonzero().tolist() == [[1]]
    assert not torch.autograd.grad(loss.sum(), leaves[0])[0][1].any()


@pytest.mark.parametrize("T", [0.01, 0.5, 1.0])
def test_logits_at_the_ends_of_float32(ops, gpu, T):  # noqa: F811
    """Logits whose quotient by the temperature is beyond float32: their distribution is not."""
    N, V, D = 5, 70, 32
    g, h, w, b, go = _inputs(7, N, V, D, FP32, False)
    ids = torch.arange(4).repeat(N, 1) + 3
    z = torch.tensor([[3e38, 3e38, -3e38, 0.0], [3e38, 1.0, 2.0, -3e38], [-3e38, -3e38, -3.4e38, -math.inf],
                      [2e38, 2e38, 2e38, 2e38], [1e38, 1e38, 0.0, 0.0]])
    want, bound = co.loss(h, w, *co.teacher(ids, z, T), go, temperature=T)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w)]
    _check(ops.distillation(leaves[0], leaves[1], ids.to(gpu), z.to(gpu), temperature=T), leaves, go, want, bound)


@pytest.mark.parametrize("T", [1e-10, 1e-25, 1e-30])
def test_loss_at_temperatures_whose_square_is_lost(ops, gpu, T):  # noqa: F811
    """T^2 times a divergence of the order of 1 / T is of the order of T."""
    N, V, D = 5, 70, 32
    g, h, w, _, go = _inputs(8, N, V, D, FP32, False)
    ids, z = torch.arange(2).repeat(N, 1) + 3, torch.zeros(N, 2)
    want, bound = co.loss(h, w, *co.teacher(ids, z, T), go, temperature=T)
    with torch.no_grad():
        got = ops.distillation(h.to(gpu), w.to(gpu), ids.to(gpu), z.to(gpu), temperature=T).cpu().double()
    assert bool((want["loss"] > 100 * bound["loss"]).all())
    assert bool(((got - want["loss"]).abs() <= bound["loss"]).all())


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,V,K,T", [(3, 1, 2, 1.0), (40, 1, 20, 2.0), (300, 2, 7, 0.5), (40, 2, 33, 1.0),
                                     (5000, 3, 4, 1.0)])
def test_entries_of_one_candidate_where_it_has_nearly_all(ops, gpu, N, V, K, T, dtype):  # noqa: F811
    """Each entry counts by itself: sum q (log q - log p) is negative where p exceeds its parts of q."""
    g, h, w, b, go = _inputs(N + K, N, V, 32, dtype, True)
    b *= 6.0
    ids, z = torch.randint(0, V, (N, K), generator=g), _rand(g, N, K, std=2.0)
    ids[0] = 0
    want, bound = co.loss(h, w, *co.teacher(ids, z, T), go, b, temperature=T)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    loss = ops.distillation(leaves[0], leaves[1], ids.to(gpu), z.to(gpu), bias=leaves[2], temperature=T)
    assert bool((want["loss"] < -0.05).any())
    _check(loss, leaves, go, want, bound)


def test_a_matched_teacher_of_one_entry_each_is_not_under_zero(ops, gpu):  # noqa: F811
    """Without an entry given twice the divergence is 0 or more, rounding or not."""
    g, h, w, b, go = _inputs(1, 400, 6, 32, FP32, False)
    z = (h.double() @ w.double().t()).float()
    ids = torch.arange(6).expand(400, 6)
    with torch.no_grad():
        loss = ops.distillation(h.to(gpu), w.to(gpu), ids.to(gpu), z.to(gpu))
    assert bool((loss >= 0).all()) and float(loss.max()) < 1e-5
