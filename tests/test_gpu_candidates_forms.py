"""The losses over all candidates in the forms that larger sizes take (pieces
of the table shared by workgroups, rows put in order, steps of channels left
out, many blocks of candidates) and in other calls: streams, hooks, captured
graphs, far strides."""
import math

import pytest
import torch

import candidates_oracle as co
from test_gpu_candidates import BF16, FP16, FP32, _check, _close, _inputs, _rand, ops  # noqa: F401

pytestmark = pytest.mark.gpu

FORMS = [  # N, V, D, dtype, bias: the last channels' steps of 16 left out (0, 1, 2 of the last 64 channels)
    (40, 300, 48, BF16, False),
    (40, 300, 33, FP16, True),
    (300, 300, 90, BF16, True),
    (300, 300, 96, FP16, False),
    (300, 300, 97, BF16, True),
    (300, 300, 112, FP16, True),
    (300, 300, 160, BF16, False),
    (300, 300, 161, FP16, True),
    (300, 300, 176, BF16, True),
    (300, 300, 224, FP16, False),
    (300, 300, 239, BF16, True),
    (300, 300, 104, FP32, True),
    (300, 300, 185, FP32, False),
    # whole and half tiles of rows
    (250, 500, 90, BF16, True),
    (250, 500, 172, FP16, False),
    (1100, 200, 160, BF16, True),
    (100, 500, 172, BF16, True),
    # pieces of the table and of the rows shared by workgroups, ragged at both ends
    (600, 20011, 100, BF16, False),
    (270, 40003, 172, FP16, True),
    (600, 33333, 64, FP32, True),
    (1, 70001, 172, BF16, True),
    (32, 70001, 100, FP16, False),
    (16500, 333, 43, BF16, True),
    (9000, 2100, 20, FP32, False),
]


@pytest.mark.parametrize("N,V,D,dtype,biased", FORMS)
def test_forms(ops, gpu, N, V, D, dtype, biased):  # noqa: F811
    g, h, w, b, go = _inputs(N * 3 + V + D, N, V, D, dtype, biased)
    t = torch.randint(0, V, (N,), generator=g)
    if N > 3:
        t[torch.rand(N, generator=g) < 0.3] = -1
        h[t < 0] = math.nan
    if b is not None:
        out = torch.rand(V, generator=g) < 0.1
        out[t.clamp(min=0)] = False
        b[out] = -math.inf
        w[out] = math.nan
    want, bound = co.loss(h, w, *co.labels(t), go, b)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b) if x is not None]
    loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu), bias=leaves[2] if biased else None)
    grads = _check(loss, leaves, go, want, bound)
    again = torch.autograd.grad(ops.cross_entropy(leaves[0], leaves[1], t.to(gpu), bias=leaves[2] if biased else None),
                                leaves, go.to(gpu))
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.parametrize("N,V,D,K,dtype", [
    (3, 400_001, 16, 5, BF16),      # more blocks of candidates than are counted at once
    (1500, 3000, 72, 1, FP16),      # one entry a row, no order of the rows
    (70, 20_000, 172, 300, BF16),
    (2000, 500, 36, 9, FP32),
])
def test_teacher_forms(ops, gpu, N, V, D, K, dtype):  # noqa: F811
    g, h, w, b, go = _inputs(N + V, N, V, D, dtype, True)
    ids, z = torch.randint(0, V, (N, K), generator=g), _rand(g, N, K, std=2.0)
    ids[0, 0], ids[-1, -1] = V - 1, 0
    ids[torch.rand(N, K, generator=g) < 0.2] = -5
    want, bound = co.loss(h, w, *co.teacher(ids, z, 2.0), go, b, temperature=2.0)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    loss = ops.distillation(leaves[0], leaves[1], ids.to(gpu), z.to(gpu), bias=leaves[2], temperature=2.0)
    _check(loss, leaves, go, want, bound)


@pytest.mark.parametrize("N", [1023, 1024, 5000, (1 << 18) + 3])
def test_rows_in_order(ops, gpu, N):  # noqa: F811
    """Rows without a target between the others, in front, behind, everywhere."""
    V, D = 33, 8
    g, h, w, b, go = _inputs(N, N, V, D, FP32, False)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w)]
    for dead in (torch.rand(N, generator=g) < 0.5, torch.arange(N) < N - 3, torch.arange(N) > 2,
                 torch.ones(N, dtype=torch.bool), torch.zeros(N, dtype=torch.bool)):
        t = torch.where(dead, -1, torch.randint(0, V, (N,), generator=g))
        want, bound = co.loss(h, w, *co.labels(t), go)
        loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu))
        _check(loss, leaves, go, want, bound)
    t = torch.full((N,), V)   # past the table: no gradient, no loss
    loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu))
    assert torch.isnan(loss).all() and not any(x.any() for x in torch.autograd.grad(loss.sum(), leaves))


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_far_and_shared_rows(ops, gpu, dtype):  # noqa: F811
    """Rows of the table as far apart as the kernels take and further (copied),
    and one row that all share: its gradient is the sum."""
    N, V, D = 5, 67, 24
    g, h, w, _, go = _inputs(2, N, V, D, dtype, False)
    t = torch.randint(0, V, (N,), generator=g)
    want, bound = co.loss(h, w, *co.labels(t), go)
    x = h.to(gpu).requires_grad_()
    for far in (ops.MAX_STRIDE, ops.MAX_STRIDE + 1):
        room = torch.empty((V - 1) * far + D, dtype=dtype, device=gpu)
        table = room.as_strided((V, D), (far, 1))
        table.copy_(w)
        table = table.detach().requires_grad_()
        assert table.stride(0) == far
        _check(ops.cross_entropy(x, table, t.to(gpu)), [x, table], go, want, bound)
        del room, table
    row = w[:1].to(gpu).requires_grad_()
    one = h[:1].to(gpu).requires_grad_()
    loss = ops.cross_entropy(one.expand(N, D), row.expand(V, D), t.to(gpu))   # equal scores
    assert (loss - math.log(V)).abs().max() < 1e-5
    dh, dw = torch.autograd.grad(loss, [one, row], go.to(gpu))
    assert dh.shape == (1, D) and dw.shape == (1, D)
    # (p and the target's 1 cancel: what is left are roundings of p to the type)
    most = co.unit(dtype) + 2.0 ** -20
    assert dh.abs().max() <= 2 * most * go.sum() * float(w[0].abs().max()) + V * most * 1e-3
    assert dw.abs().max() <= 4 * V * most * float((go[:, None] * h.abs()).sum(0).max())


def test_streams_and_two_calls_at_once(ops, gpu):  # noqa: F811
    g, h, w, b, go = _inputs(31, 700, 9000, 100, BF16, True)
    t = torch.randint(-1, 9000, (700,), generator=g).to(gpu)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    go = go.to(gpu)

    def step():
        loss = ops.cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        return (loss.detach(), *torch.autograd.grad(loss, leaves, go))

    want = step()
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in sides:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(x, y) for x, y in zip(want, out))


def test_two_graphs_in_turn(ops, gpu):  # noqa: F811
    """Graphs of different sizes from one pool, replayed in turn."""
    pool, held = None, []
    for N, V, D, K in ((50, 4000, 64, 0), (900, 300, 100, 12), (1, 5000, 172, 0)):
        g, h, w, b, go = _inputs(N, N, V, D, FP16, True)
        leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
        t = torch.randint(0, V, (N, max(K, 1)), generator=g).to(gpu)
        z, go = _rand(g, N, max(K, 1)).to(gpu), go.to(gpu)

        def step(leaves=leaves, t=t, z=z, go=go, K=K):
            loss = (ops.distillation(leaves[0], leaves[1], t, z, bias=leaves[2]) if K else
                    ops.cross_entropy(leaves[0], leaves[1], t[:, 0], bias=leaves[2]))
            return (loss.detach(), *torch.autograd.grad(loss, leaves, go))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side, pool=pool):
                out = step()
            pool = pool or graph.pool()
        torch.cuda.current_stream().wait_stream(side)
        held.append((graph, [x.clone() for x in step()], out, (leaves, t, z, go)))   # (the inputs stay where they are)
    for _ in range(3):
        for graph, want, out, _ in held:
            graph.replay()
            assert all(torch.equal(x, y) for x, y in zip(want, out))   # (before the next graph reuses the pool)


def test_hooks_repeated_backward_and_second_order(ops, gpu):  # noqa: F811
    g, h, w, b, go = _inputs(37, 60, 500, 50, FP32, True)
    t = torch.randint(0, 500, (60,), generator=g).to(gpu)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    go = go.to(gpu)
    loss = ops.cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    want = torch.autograd.grad(loss, leaves, go, retain_graph=True)
    for x, y in zip(want, torch.autograd.grad(loss, leaves, go)):
        assert torch.equal(x, y)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x.cpu(), lambda x: x.to(gpu)):
        away = ops.cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    for x, y in zip(want, torch.autograd.grad(away, leaves, go)):
        assert torch.equal(x, y)
    loss = ops.cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    first = torch.autograd.grad(loss, leaves, go.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
        first[0].sum().backward()
    go = go.detach()
    loss = ops.cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    with torch.no_grad():
        leaves[1].mul_(2.0)   # a saved tensor written in between
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(loss, leaves, go)


@pytest.mark.parametrize("scale", [1.0, -1.0, 0.0, 40.0])
@pytest.mark.parametrize("N,V,D,dtype", [(5, 1000, 64, BF16), (300, 640, 100, FP16), (520, 1111, 172, BF16),
                                         (300, 999, 100, FP32), (2000, 129, 256, BF16)])
def test_loss_alone(ops, gpu, N, V, D, dtype, scale):  # noqa: F811
    """Without gradients and a bias, scores that grow along the table or fall."""
    g, h, w, _, go = _inputs(N + D, N, V, D, dtype, False)
    for growth in (torch.linspace(0.1, 3.0, V), torch.linspace(3.0, 0.1, V)):
        table = (w.float().abs() * growth[:, None]).to(dtype)
        rows = h.abs()
        t = torch.randint(0, V, (N,), generator=g)
        want, bound = co.loss(rows, table, *co.labels(t), go, scale=scale)
        with torch.no_grad():
            got = ops.cross_entropy(rows.to(gpu), table.to(gpu), t.to(gpu), scale=scale)
        _close(got, want["loss"], bound["loss"], "loss")
