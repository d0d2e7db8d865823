"""Calls of the history operators that their documentation allows and that are
easily wrong: the widest groups of heads with the largest tables, operands that
are one tensor or share memory, some of the leaves, expanded gradients, the
smallest heads, channels and rows, and captured training steps of every form."""
import math

import pytest
import torch

import history_oracle as ho
from test_gpu_history import _attend_inputs, _close, _norm_inputs, _oracle_scan, _rand, _run_attend, _run_norm, _run_scan
from test_gpu_history import _scan_bound, _scan_inputs

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops(gpu):
    from starry_unigraph.native import history
    return history


def _want(t, cols):
    t = {k: t.get(k) for k in ("q", "k", "v", "go", "q_lens", "k_lens", "key_mask", "bias")}
    return ho.attend(**t, cols=cols)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("case", [  # N, Lq, Lk, Hq, Hkv, dh
    (2, 1, 40, 64, 2, 128),     # 32 heads to a key head, one wave a sequence
    (2, 1, 200, 32, 1, 128),
    (2, 1, 70, 64, 1, 128),     # 64 heads: rows in tiles
    (2, 3, 150, 128, 2, 128),
    (70, 6, 66, 64, 1, 64),     # eight waves a workgroup
    (60, 9, 66, 63, 1, 33),     # an odd number of them
    (3, 2, 66, 30, 2, 17),
], ids=str)
def test_attention_of_many_heads_and_columns(ops, gpu, case, dtype):
    t, kw, cols = _attend_inputs(*case, dtype, 32, 1, True, True, True)
    o, grads = _run_attend(ops, t, kw, gpu)
    want, bound = _want(t, cols)
    _close(o, want["o"], bound["o"], "o")
    for k, got in grads.items():
        _close(got, want[k], bound[k], k)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("dh", [1, 2, 3, 5, 7, 9])
def test_attention_of_the_smallest_heads(ops, gpu, dh, dtype):
    for Lq, Lk in ((3, 9), (40, 70)):
        t, kw, cols = _attend_inputs(3, Lq, Lk, 4, 2, dh, dtype, 5, 0, True, True, True)
        o, grads = _run_attend(ops, t, kw, gpu)
        want, bound = _want(t, cols)
        _close(o, want["o"], bound["o"], "o")
        for k, got in grads.items():
            _close(got, want[k], bound[k], k)


@pytest.mark.parametrize("Lq, Lk", [(5, 20), (33, 80), (130, 130)])
def test_attention_of_shared_and_transposed_operands(ops, gpu, Lq, Lk):
    """Keys that are the values; heads before rows in memory; some of the
    leaves; a gradient that is one expanded number: each as with tensors of
    their own, contiguous ones, all leaves and a full gradient."""
    t, kw, _ = _attend_inputs(40, Lq, Lk, 4, 2, 24, BF16, 6, 0, True, True, True)
    d = {k: x.to(gpu) for k, x in t.items()}
    extra = {k: d[k] for k in ("q_lens", "k_lens", "key_mask", "q_pos", "k_pos")}
    call = lambda q, k, v, bias: ops.cross_attention(q, k, v, bias=bias, **extra, **kw)
    leaf = lambda x: x.detach().clone().requires_grad_()
    q, k, v, b = (leaf(d[n]) for n in ("q", "k", "k", "bias"))
    o = call(q, k, v, b)
    want = torch.autograd.grad(o, (q, k, v, b), torch.ones_like(o))
    # one tensor as keys and values
    both = leaf(d["k"])
    o2 = call(q, both, both, b)
    assert torch.equal(o, o2)
    g = torch.autograd.grad(o2.sum(), (q, both, b))
    assert torch.equal(g[0], want[0]) and torch.equal(g[2], want[3])
    assert torch.equal(g[1], want[1] + want[2])
    # heads first in memory
    qt, kt, vt = (leaf(x.detach().transpose(1, 2).contiguous()) for x in (q, k, v))
    o3 = call(*(x.transpose(1, 2) for x in (qt, kt, vt)), b)
    assert torch.equal(o, o3)
    for got, w in zip(torch.autograd.grad(o3.sum(), (qt, kt, vt)), want):
        assert torch.equal(got.transpose(1, 2), w)
    # one leaf at a time
    for i in range(4):
        args = [x if j == i else x.detach() for j, x in enumerate((q, k, v, b))]
        assert torch.equal(torch.autograd.grad(call(*args).sum(), args[i])[0], want[i])
    # keys and values of one sequence for all (a broadcast input's gradient is summed)
    k1, v1 = leaf(d["k"][:1]), leaf(d["v"][:1])
    ke, ve = (leaf(x.detach().expand(40, -1, -1, -1)) for x in (k1, v1))
    a = torch.autograd.grad(call(q, k1.expand(40, -1, -1, -1), v1.expand(40, -1, -1, -1), b).sum(), (k1, v1))
    e = torch.autograd.grad(call(q, ke, ve, b).sum(), (ke, ve))
    for got, w in zip(a, e):
        assert torch.equal(got, w.sum(0, keepdim=True))


def test_scan_of_one_channel_and_broadcast_inputs(ops, gpu):
    for dtype in (FP32, BF16):
        for case in ((70, 9, 1, dtype, True, True, True), (1, 2000, 1, dtype, True, False, True)):
            t, gh, gl = _scan_inputs(*case)
            h, last, grads = _run_scan(ops, t, gh, gl, gpu)
            wh, wl, wg = _oracle_scan(t, gh, gl)
            M, G, e = _scan_bound(t, gh, gl, wh)
            _close(h, wh, ho.unit(dtype) * wh.abs() + 2 * e * M, "h")
            _close(last, wl, 2 * e * M, "last")
            _close(grads["state"], wg["state"], 2 * e * G, "state")
    g = torch.Generator().manual_seed(1)
    row = _rand(g, 1, 1, 24).to(gpu).requires_grad_()
    value = _rand(g, 6, 30, 24).to(gpu)
    full = row.detach().expand(6, 30, 24).contiguous().requires_grad_()
    a, b = ops.gated_scan(row.expand(6, 30, 24), value), ops.gated_scan(full, value)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga = torch.autograd.grad(a[0].sum() + a[1].sum(), row)[0]
    gb = torch.autograd.grad(b[0].sum() + b[1].sum(), full)[0]
    assert torch.equal(ga, gb.sum((0, 1), keepdim=True))
    # the last state alone, and the outputs alone
    v = value.clone().requires_grad_()
    h, last = ops.gated_scan(full, v)
    only = torch.autograd.grad(last.sum(), v, retain_graph=True)[0]
    both = torch.autograd.grad((h, last), v, (torch.zeros_like(h), torch.ones_like(last)))[0]
    assert torch.equal(only, both)


@pytest.mark.parametrize("dtype", [FP32, FP16])
def test_norm_of_one_row_broadcast_over_a_batch(ops, gpu, dtype):
    t, gs = _norm_inputs(40, 36, dtype, False, seed=9)
    t["gate"] = t["gate"][:1].expand(40, 36).contiguous()
    y, n, grads = _run_norm(ops, t, gs, gpu, False)
    d = {k: v.to(gpu).requires_grad_() for k, v in t.items()}
    one = t["gate"][:1].to(gpu).requires_grad_()
    kw = {k: d[k] for k in d if k.endswith(("weight", "bias"))}
    y2, n2 = ops.gated_norm(d["x"], d["z"], one.expand(40, 36), d["scale"], **kw)
    assert torch.equal(y, y2) and torch.equal(n, n2)
    g = torch.autograd.grad((y2, n2), (one, d["z"]), [x.to(gpu) for x in gs])
    assert torch.equal(g[0], grads["gate"].sum(0, keepdim=True)) and torch.equal(g[1], grads["z"])
    # the same tensor in every place
    x = t["x"].to(gpu).requires_grad_()
    a, b, c = (t["x"].to(gpu).requires_grad_() for _ in range(3))
    s = torch.autograd.grad(ops.gated_norm(x, x, x, d["scale"], **kw)[1].sum(), x)[0]
    p = torch.autograd.grad(ops.gated_norm(a, b, c, d["scale"], **kw)[1].sum(), (a, b, c))
    assert torch.allclose(s.float(), sum(i.float() for i in p), rtol=4 * ho.unit(dtype), atol=8 * ho.unit(dtype))


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("case", [(6, 4, 20, 4, 2, 24), (3, 50, 60, 4, 2, 24), (2, 1, 900, 4, 2, 24),
                                  (70, 130, 70, 4, 1, 24)], ids=str)
def test_captured_steps_of_every_form(ops, gpu, case, dtype):
    """A training step captured and replayed on new values, three times, with
    eager work between: the eager bits every time."""
    t, kw, _ = _attend_inputs(*case, dtype, 16, 0, True, True, True)
    d = {k: x.to(gpu) for k, x in t.items()}
    leaves = [d[k].requires_grad_() for k in ("q", "k", "v", "bias")]
    extra = {k: d[k] for k in ("q_lens", "k_lens", "key_mask", "q_pos", "k_pos")}

    def step():
        o = ops.cross_attention(d["q"], d["k"], d["v"], bias=d["bias"], **extra, **kw)
        return [o.detach(), *torch.autograd.grad(o, leaves, d["go"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        static = step()
    for scale in (0.5, 30.0, 0.001):   # (the bias gradient's and fp16's powers of two change with the values)
        with torch.no_grad():
            d["v"].mul_(scale)
            d["go"].mul_(1 / scale)
            d["k_lens"].copy_(d["k_lens"].roll(1))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in static]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
