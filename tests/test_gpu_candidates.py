"""The losses over all candidates on the GPU against their definitions in
float64 (candidates_oracle): every type, single rows and many, odd sizes,
strided inputs, candidates that are left out, rows that are; gradients against
the formula's and against differences; the same bits from run to run."""
import math

import pytest
import torch

import candidates_oracle as co

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops(gpu):
    from starry_unigraph.native import candidates
    return candidates


def _rand(g, *shape, dtype=FP32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype)


def _close(got, want, bound, what):
    most = torch.finfo(got.dtype).max
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    # (a value past the type's largest is rounded to inf)
    bad = ~(((got - want).abs() <= bound) | ((got == want.sign() * math.inf) & (want.abs() + bound > most)))
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs()[bad].max()),
                           float(bound.expand_as(got)[bad].max()))


def _inputs(seed, N, V, D, dtype, biased, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    h, w = _rand(g, N, D, dtype=dtype), _rand(g, V, D, dtype=dtype, std=spread / math.sqrt(D))
    b = _rand(g, V, std=0.7) if biased else None
    go = (torch.rand(N, generator=g) + 0.5) * (256.0 if dtype == FP16 else 1.0) / N
    return g, h, w, b, go


def _check(out, leaves, go, want, bound):
    names = ["dh", "dtable", "dbias"][:len(leaves)]
    grads = torch.autograd.grad(out, leaves, go.to(out.device).view(out.shape))
    _close(out.flatten(), want["loss"], bound["loss"], "loss")
    for n, x in zip(names, grads):
        _close(x, want[n], bound[n], n)
    return grads


SIZES = [  # N, V, D, dtype, bias
    (1, 1, 1, FP32, False),
    (1, 2, 3, BF16, True),
    (1, 1000, 172, BF16, False),
    (7, 65, 43, FP16, True),
    (32, 129, 64, FP32, True),
    (33, 1000, 100, FP32, False),
    (33, 1000, 100, BF16, True),
    (5, 3000, 256, FP32, False),
    (20, 700, 256, BF16, True),
    (20, 515, 193, FP16, False),
    (200, 1000, 100, FP32, True),
    (257, 1023, 172, BF16, False),
    (300, 777, 256, FP16, True),
    (300, 777, 255, BF16, False),
    (130, 515, 256, FP32, True),
    (129, 64, 65, FP32, False),
    (1200, 67, 8, BF16, True),
    (513, 300, 17, FP16, True),
    (2500, 9, 129, BF16, False),
]


@pytest.mark.parametrize("N,V,D,dtype,biased", SIZES)
def test_cross_entropy(ops, gpu, N, V, D, dtype, biased):
    g, h, w, b, go = _inputs(N * 7 + V, N, V, D, dtype, biased)
    t = torch.randint(0, V, (N,), generator=g)
    if N > 3:
        t[torch.rand(N, generator=g) < 0.3] = -1
        h[t < 0] = math.nan   # padding may hold anything
    if b is not None and V > 3:
        out = torch.rand(V, generator=g) < 0.2
        out[t.clamp(min=0)] = False
        b[out] = -math.inf
        w[out] = math.inf
    want, bound = co.loss(h, w, *co.labels(t), go, b)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b) if x is not None]
    loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu), bias=leaves[2] if biased else None)
    _check(loss, leaves, go, want, bound)
    with torch.no_grad():   # without gradients: the same numbers to their bounds
        plain = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu), bias=leaves[2] if biased else None)
    _close(plain, want["loss"], bound["loss"], "loss alone")


DISTILL = [  # N, V, D, K, dtype, bias, temperature
    (1, 50, 100, 1, FP32, False, 1.0),
    (3, 50, 172, 50, BF16, True, 2.0),
    (33, 1000, 100, 20, FP32, True, 1.0),
    (70, 515, 43, 64, BF16, False, 4.0),
    (300, 777, 256, 100, FP16, True, 2.0),
    (257, 200, 65, 7, FP16, False, 0.5),
    (40, 3000, 64, 1024, FP32, False, 3.0),
    (600, 130, 129, 33, BF16, True, 1.5),
]


@pytest.mark.parametrize("N,V,D,K,dtype,biased,T", DISTILL)
def test_distillation(ops, gpu, N, V, D, K, dtype, biased, T):
    g, h, w, b, go = _inputs(N * 5 + V, N, V, D, dtype, biased)
    ids = torch.randint(0, V, (N, K), generator=g)   # (some twice)
    z = _rand(g, N, K, std=1.5, mean=3.0)
    if N > 2:
        ids[torch.rand(N, K, generator=g) < 0.1] = -1
        z[torch.rand(N, K, generator=g) < 0.05] = -math.inf
        ids[1] = -1                                  # nothing
        if K > 2:
            ids[2, 1:] = ids[2, 0] = 3               # one candidate in every entry
            z[2] = 1.0
    want, bound = co.loss(h, w, *co.teacher(ids, z, T), go, b, temperature=T)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b) if x is not None]
    loss = ops.distillation(leaves[0], leaves[1], ids.to(gpu), z.to(gpu), bias=leaves[2] if biased else None,
                            temperature=T)
    _check(loss, leaves, go, want, bound)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_scale_strides_and_leading_dimensions(ops, gpu, dtype):
    g, h, w, b, go = _inputs(3, 60, 130, 50, dtype, True)
    t = torch.randint(0, 130, (60,), generator=g)
    want, bound = co.loss(h, w, *co.labels(t), go, b, scale=-0.7)
    big = torch.zeros(6, 10, 77, dtype=dtype, device=gpu)
    big[..., 5:55] = h.to(gpu).view(6, 10, 50)
    table = torch.zeros(50, 131, dtype=dtype, device=gpu)
    table[:, 1:] = w.to(gpu).t()
    table = table.t()[1:]                            # columns apart by rows: copied
    wide = torch.zeros(130, 53, dtype=dtype, device=gpu)
    wide[:, 3:] = w.to(gpu)
    for tb in (table, wide[:, 3:]):
        leaves = [big[..., 5:55].requires_grad_(), tb.requires_grad_(), b.to(gpu).requires_grad_()]
        loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu).view(6, 10), bias=leaves[2], scale=-0.7)
        assert loss.shape == (6, 10)
        dh, dw, db = torch.autograd.grad(loss, leaves, go.to(gpu).view(6, 10))
        _close(loss.flatten(), want["loss"], bound["loss"], "loss")
        _close(dh.reshape(60, 50), want["dh"], bound["dh"], "dh")
        _close(dw, want["dtable"], bound["dtable"], "dtable")
        _close(db, want["dbias"], bound["dbias"], "dbias")


def test_rows_without_an_answer(ops, gpu):
    g, h, w, b, go = _inputs(5, 6, 40, 32, BF16, True)
    b[7] = -math.inf
    t = torch.tensor([3, -1, 40, 7, -(1 << 62), 1 << 40])
    leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu), bias=leaves[2])
    dh, dw, db = torch.autograd.grad(loss.sum(), leaves)
    got = loss.tolist()
    assert got[1] == got[4] == 0 and math.isnan(got[2]) and math.isnan(got[5]) and got[3] == math.inf
    assert not dh[1:].any() and dh[0].any() and torch.isfinite(dw).all() and not dw[7].any() and db[7] == 0
    one = torch.where(torch.arange(6) == 0, t, torch.tensor(-1))
    alone = ops.cross_entropy(leaves[0], leaves[1], one.to(gpu), bias=leaves[2])
    for x, y in zip((dh, dw, db), torch.autograd.grad(alone.sum(), leaves)):
        assert torch.equal(x, y)
    # every candidate left out
    none = torch.full((40,), -math.inf, device=gpu, requires_grad=True)
    loss = ops.cross_entropy(leaves[0], leaves[1], t.clamp(0, 39).to(gpu), bias=none)
    assert not loss.any()
    assert not any(x.any() for x in torch.autograd.grad(loss.sum(), [*leaves[:2], none]))
    # a teacher's rows: an id past the table, one left out, none
    ids = torch.tensor([[3, 5], [3, 40], [7, 5], [-1, -1], [3, -1], [5, 5]])
    loss = ops.distillation(leaves[0], leaves[1], ids.to(gpu), torch.zeros(6, 2, device=gpu), bias=leaves[2])
    dh = torch.autograd.grad(loss.sum(), leaves)[0]
    got = loss.tolist()
    assert math.isnan(got[1]) and got[2] == math.inf and got[3] == 0
    assert not dh[1:4].any() and all(dh[i].any() for i in (0, 4, 5))


def test_not_finite_rows_spoil_themselves(ops, gpu):
    g, h, w, b, go = _inputs(9, 40, 200, 64, BF16, False)
    h[4, 7], h[6, 3] = math.nan, math.inf
    t = torch.randint(0, 200, (40,), generator=g)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w)]
    loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu))
    dh, dw = torch.autograd.grad(loss.sum(), leaves)
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[4, 6]] = True
    assert (torch.isnan(loss.cpu()) == bad).all() and (torch.isnan(dh).all(1).cpu() == bad).all()
    assert torch.isfinite(dh[~bad.to(gpu)]).all() and torch.isnan(dw).any()
    # the same rows left out: nothing of them is seen
    t[bad] = -1
    loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu))
    assert all(torch.isfinite(x).all() for x in (loss, *torch.autograd.grad(loss.sum(), leaves)))


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("N,V", [(3, 700), (300, 700)])
def test_scores_far_from_zero_and_growing(ops, gpu, N, V, dtype):
    """Maxima that grow along the table by far more than the softmax's slack, and
    a bias far below zero for all."""
    g, h, w, b, go = _inputs(11, N, V, 100, dtype, True)
    t = torch.randint(0, V, (N,), generator=g)
    for shift in (torch.linspace(-80.0, 80.0, V), torch.full((V,), -3000.0), torch.linspace(300.0, -300.0, V)):
        bias = b + shift
        want, bound = co.loss(h, w, *co.labels(t), go, bias)
        leaves = [x.to(gpu).requires_grad_() for x in (h, w, bias)]
        loss = ops.cross_entropy(leaves[0], leaves[1], t.to(gpu), bias=leaves[2])
        _check(loss, leaves, go, want, bound)
    lowest = torch.full((V,), torch.finfo(FP32).min, device=gpu)
    with torch.no_grad():   # equal scores: log V
        loss = ops.cross_entropy(h.to(gpu), w.to(gpu), t.to(gpu), bias=lowest)
    assert (loss.cpu() - math.log(V)).abs().max() < 1e-5


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("size", [1e-6, 1.0, 3e4])
def test_gradients_over_the_range_of_magnitudes(ops, gpu, dtype, size):
    g, h, w, b, go = _inputs(13, 70, 300, 64, dtype, False)
    go = go * size
    t = torch.randint(0, 300, (70,), generator=g)
    want, bound = co.loss(h, w, *co.labels(t), go)
    leaves = [x.to(gpu).requires_grad_() for x in (h, w)]
    _check(ops.cross_entropy(leaves[0], leaves[1], t.to(gpu)), leaves, go, want, bound)


def test_gradients_against_differences(ops, gpu):
    g, h, w, b, go = _inputs(17, 9, 40, 12, FP32, True)
    t = torch.randint(0, 40, (9,), generator=g)
    ids, z = torch.randint(0, 40, (9, 5), generator=g), _rand(g, 9, 5)
    for call in (lambda *x: ops.cross_entropy(x[0], x[1], t.to(gpu), bias=x[2], scale=0.5),
                 lambda *x: ops.distillation(x[0], x[1], ids.to(gpu), z.to(gpu), bias=x[2], temperature=2.0)):
        leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
        grads = torch.autograd.grad(call(*leaves), leaves, go.to(gpu))
        for i, x in enumerate(leaves):
            way = _rand(g, *x.shape).to(gpu)
            ends = []
            for sign in (1, -1):
                moved = [y.detach() + (sign * 2.0 ** -7 * way if j == i else 0) for j, y in enumerate(leaves)]
                ends.append(float((call(*moved).double() * go.to(gpu)).sum()))
            slope = (ends[0] - ends[1]) * 64
            got = float((grads[i].double() * way).sum())
            # a difference in float32: 2^-24 of a loss of about 4, times 64; a step's third order
            assert abs(slope - got) < 2e-3 * max(1.0, abs(slope)), (i, slope, got)


def test_parts_that_need_no_gradient(ops, gpu):
    g, h, w, b, go = _inputs(19, 50, 300, 100, BF16, True)
    t = torch.randint(0, 300, (50,), generator=g).to(gpu)
    full = [x.to(gpu).requires_grad_() for x in (h, w, b)]
    want = torch.autograd.grad(ops.cross_entropy(full[0], full[1], t, bias=full[2]).sum(), full)
    for on in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
        part = [x.detach().clone().requires_grad_(o) for x, o in zip(full, on)]
        got = torch.autograd.grad(ops.cross_entropy(part[0], part[1], t, bias=part[2]).sum(),
                                  [x for x, o in zip(part, on) if o])
        for x, y in zip(got, [y for y, o in zip(want, on) if o]):
            # (without h's gradient the forward takes another form: another order of sums at most)
            assert torch.allclose(x.float(), y.float(), rtol=2e-2, atol=1e-6)


def test_results_repeat_and_replay(ops, gpu):
    for N, V, K in ((40, 5000, 9), (3000, 500, 30)):
        g, h, w, b, go = _inputs(23, N, V, 72, BF16, True)
        leaves = [x.to(gpu).requires_grad_() for x in (h, w, b)]
        ids, z = torch.randint(0, V, (N, K), generator=g).to(gpu), _rand(g, N, K).to(gpu)
        go = go.to(gpu)

        def step():
            loss = ops.distillation(leaves[0], leaves[1], ids, z, bias=leaves[2], temperature=2.0)
            return (loss.detach(), *torch.autograd.grad(loss, leaves, go))

        first = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                held = step()
        torch.cuda.current_stream().wait_stream(side)
        for _ in range(3):
            graph.replay()
            eager = step()
            for x, y, e in zip(first, held, eager):
                assert torch.equal(x, y) and torch.equal(x, e)


def test_empty_batch(ops, gpu):
    h = torch.zeros(0, 50, device=gpu, requires_grad=True)
    w = torch.ones(10, 50, device=gpu, requires_grad=True)
    loss = ops.cross_entropy(h, w, torch.zeros(0, dtype=torch.int64, device=gpu))
    assert loss.shape == (0,)
    dh, dw = torch.autograd.grad(loss.sum(), [h, w])
    assert dh.shape == (0, 50) and not dw.any()
