"""The forms of the history operators that only larger problems take: row blocks
shared by waves, two heads of the same queries together, key tiles in several
waves, parts of a long history joined, pieces of a sequence composed; against
the definitions in float64 (history_oracle), with its bounds."""
import math

import pytest
import torch

import history_oracle as ho
from test_gpu_history import (_attend_inputs, _close, _oracle_scan, _rand, _run_attend, _run_scan, _scan_bound,
                              _scan_inputs)

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops(gpu):
    from starry_unigraph.native import history
    return history


def _columns(ops, q_pos, k_pos, buckets, m, two):
    """The bias columns by the framework's own bucket function (checked
    against the definition elsewhere)."""
    d = q_pos[:, :, None] - k_pos[:, None, :]
    at = ops.distance_bucket(d if two else d.clamp_min(0), buckets, m)
    return torch.where(d < 0, at + buckets, at) if two else at


def _inputs(ops, N, Lq, Lk, Hq, Hkv, dh, dtype, buckets, m, two, mask, far):
    t, _, _ = _attend_inputs(N, Lq, Lk, Hq, Hkv, dh, dtype, 0, 0, False, True, mask, seed=N + Lq)
    kw, cols = {}, None
    if buckets:
        g = torch.Generator().manual_seed(Lk)
        t["bias"] = _rand(g, Hq, buckets * (2 if two else 1))
        span = 2 ** 61 if far else 2 ** 20
        t["q_pos"], t["k_pos"] = (torch.randint(-span, span, (N, L), generator=g) for L in (Lq, Lk))
        kw = dict(resolution=m, two_sided=two)
        cols = _columns(ops, t["q_pos"], t["k_pos"], buckets, m, two)
    return t, kw, cols


def _want(t, cols):
    return ho.attend(**{k: t.get(k) for k in ("q", "k", "v", "go", "q_lens", "k_lens", "key_mask", "bias")}, cols=cols)


FORMS = [  # N, Lq, Lk, Hq, Hkv, dh, dtype, buckets, m, two, mask, far
    (24, 129, 130, 8, 2, 64, BF16, 32, 0, True, False, False),    # four heads a key head
    (24, 130, 131, 6, 2, 50, FP16, 12, 1, True, True, False),     # three
    (48, 127, 65, 4, 4, 32, BF16, 64, 2, False, True, True),      # one; positions past 32 bits
    (34, 129, 70, 4, 2, 100, FP32, 24, 1, True, True, False),     # wide heads in float32
    (34, 129, 70, 4, 2, 30, FP32, 24, 1, False, False, True),
    (24, 131, 66, 8, 2, 128, BF16, 16, 0, True, True, False),
    (24, 131, 66, 4, 1, 72, FP16, 0, 0, False, False, False),     # no bias; few tiles of keys
    (2, 1, 5000, 8, 2, 64, BF16, 40, 1, False, False, False),     # a long history in parts, joined
    (3, 1, 4099, 4, 4, 43, FP32, 20, 0, True, True, True),
    (20, 7, 300, 8, 2, 64, FP16, 32, 0, True, True, False),       # two row blocks a wave
]


@pytest.mark.parametrize("case", FORMS, ids=str)
def test_attention_forms(ops, gpu, case):
    t, kw, cols = _inputs(ops, *case)
    o, grads = _run_attend(ops, t, kw, gpu)
    want, bound = _want(t, cols)
    _close(o, want["o"], bound["o"], "o")
    for k, got in grads.items():
        _close(got, want[k], bound[k], k)


@pytest.mark.parametrize("case", [FORMS[0], FORMS[7], (3, 40, 200, 4, 2, 64, BF16, 16, 0, True, True, False)], ids=str)
def test_bias_gradient_of_bf16_heads_is_as_exact_as_float32s(ops, gpu, case):
    """The sums of a column nearly cancel: the outputs' rounding to bf16 must
    not reach them. The bounds are those of the same values in float32 tensors
    (operands exact, no rounding of p, o or ds)."""
    t, kw, cols = _inputs(ops, *case)
    _, grads = _run_attend(ops, t, kw, gpu)
    wide = {k: v.float() if k in ("q", "k", "v", "go") else v for k, v in t.items()}
    want, bound = _want(wide, cols)
    _close(grads["dbias"], want["dbias"], bound["dbias"], "dbias")


def test_serving_forms_equal_training_forms_within_rounding(ops, gpu):
    """Without gradients p is multiplied in one part: o within the bounds too."""
    for case in (FORMS[0], FORMS[1], FORMS[9]):
        t, kw, cols = _inputs(ops, *case)
        d = {k: v.to(gpu) if v is not None else None for k, v in t.items()}
        with torch.no_grad():
            o = ops.cross_attention(d["q"], d["k"], d["v"],
                                    **{k: v for k, v in d.items() if k not in ("q", "k", "v", "go")}, **kw)
        want, bound = _want(t, cols)
        _close(o, want["o"], bound["o"], "o")


def test_bias_gradient_cells_that_overflow_are_nan(ops, gpu):
    """The table's gradient is summed in 64-bit cells of fixed point; sums that
    do not fit are NaN, never wrapped. (One row's gradient of an infinity.)"""
    t, kw, _ = _inputs(ops, *FORMS[0])
    t["go"][0, 0, 0, 0] = math.inf
    _, grads = _run_attend(ops, t, kw, gpu)
    db = grads["dbias"].cpu()
    # (the four heads of a key head share their cells' power of two)
    assert torch.isnan(db[0]).any() and torch.isfinite(db[4:]).all()


SCAN = [  # N, L, D, dtype, decay, lens, state
    (2, 3001, 70, FP32, True, True, True),
    (1, 8191, 128, BF16, True, False, True),
    (3, 4097, 33, FP16, False, True, False),
    (300, 40, 100, BF16, True, True, True),
]


@pytest.mark.parametrize("case", SCAN, ids=str)
def test_scan_pieces(ops, gpu, case):
    t, gh, gl = _scan_inputs(*case)
    h, last, grads = _run_scan(ops, t, gh, gl, gpu)
    wh, wl, wg = _oracle_scan(t, gh, gl)
    M, G, e = _scan_bound(t, gh, gl, wh)
    u = ho.unit(case[3])
    _close(h, wh, u * wh.abs() + 2 * e * M, "h")
    _close(last, wl, 2 * e * M, "last")
    for k in ("gate", "value"):
        _close(grads[k], wg[k], u * wg[k].abs() + 4 * e * G * max(M, 1) + torch.finfo(case[3]).smallest_normal, k)
    if "state" in wg:
        _close(grads["state"], wg["state"], 2 * e * G, "state")


def test_calls_on_two_streams_do_not_meet(ops, gpu):
    """Two problems with workspaces, issued on two streams at once, give the
    bits that each gives alone."""
    cases = [FORMS[0], FORMS[1]]
    runs = [_inputs(ops, *c)[:2] for c in cases]
    alone = [_run_attend(ops, t, kw, gpu) for t, kw in runs]
    data = [{k: v.to(gpu) if v is not None else None for k, v in t.items()} for t, _ in runs]
    streams = [torch.cuda.Stream(gpu) for _ in runs]
    torch.cuda.synchronize()
    out = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i] = _run_attend(ops, data[i], runs[i][1], gpu)
    torch.cuda.synchronize()
    for (o, g), (wo, wg) in zip(out, alone):
        assert torch.equal(o, wo) and all(torch.equal(g[k], wg[k]) for k in wg)


def test_saved_tensors_may_come_back_elsewhere(ops, gpu):
    """Hooks that move what a backward reads (host offloading, recomputation)
    give the same gradients."""
    for case in (FORMS[9], (5, 1, 10, 2, 2, 50, FP32, 32, 0, False, True, False)):
        t, kw, _ = _inputs(ops, *case)
        _, want = _run_attend(ops, t, kw, gpu)
        with torch.autograd.graph.save_on_cpu():
            _, got = _run_attend(ops, t, kw, gpu)
        assert all(torch.equal(got[k], want[k]) for k in want)
    t, gh, gl = _scan_inputs(4, 40, 50, FP32, True, True, True)
    want = _run_scan(ops, t, gh, gl, gpu)[2]
    with torch.autograd.graph.save_on_cpu():
        got = _run_scan(ops, t, gh, gl, gpu)[2]
    assert all(torch.equal(got[k], want[k]) for k in want)


@pytest.mark.parametrize("case", [(3, 100, 1, 3, 3, 100, BF16), (27, 400, 1, 4, 1, 64, FP16), (5, 20, 1, 12, 3, 64, FP32),
                                  (300, 80, 1, 2, 1, 32, BF16), (4, 3, 1, 4, 2, 40, FP16)], ids=str)
def test_a_single_key_has_no_gradient(ops, gpu, case):
    """p is 1 whatever q, k and the bias are: their gradients are 0, not small."""
    t, kw, _ = _inputs(ops, *case, 17, 1, True, False, False)
    _, grads = _run_attend(ops, t, kw, gpu)
    for k in ("dq", "dk", "dbias"):
        assert not grads[k].any(), (k, float(grads[k].abs().max()))
