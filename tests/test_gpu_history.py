"""The history operators on the GPU against their definitions in float64
(history_oracle): every type, ragged lengths, strided inputs, masks that leave
rows empty, single events and long sequences; gradients against the formula's
and against differences; the same bits from run to run; captured graphs."""
import math

import pytest
import torch

import history_oracle as ho

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops(gpu):
    from starry_unigraph.native import history
    return history


def _rand(g, *shape, dtype=FP32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype)


def _lens(g, n, most, empty=True):
    """Full, empty, single and any: every kind is there when n >= 4."""
    x = torch.randint(0, most + 1, (n,), generator=g)
    x[0] = most
    if n > 1 and empty:
        x[1] = 0
    if n > 2:
        x[2] = min(1, most)
    return x.to(torch.int32)


def _close(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs()[bad].max()),
                           float(bound.expand_as(got)[bad].max()))


# ------------------------------------------------------------------ gated scan
SCAN = [  # N, L, D, dtype, decay, lens, state
    (1, 1, 1, FP32, False, False, False),
    (3, 1, 100, FP32, True, False, True),
    (5, 20, 100, FP32, True, True, True),
    (7, 16, 43, FP32, False, True, False),
    (4, 33, 50, BF16, True, True, True),
    (4, 17, 43, BF16, True, True, False),
    (3, 40, 6, FP16, False, True, True),
    (2, 130, 3, FP16, True, True, True),
    (4, 1000, 64, FP32, True, True, True),     # cut into chunks
    (4, 997, 33, BF16, False, True, True),
    (5, 2049, 10, FP32, False, True, False),
]


def _scan_inputs(N, L, D, dtype, decay, lens, state, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = dict(gate=_rand(g, N, L, D, dtype=dtype, std=2.0, mean=1.0), value=_rand(g, N, L, D, dtype=dtype),
             lens=_lens(g, N, L) if lens else None, state=_rand(g, N, D) if state else None, gaps=None, decay=None)
    if decay:
        t["gaps"] = torch.empty(N, L).exponential_(1.0, generator=g)
        t["decay"] = torch.rand(D, generator=g) * 0.5
    gh, gl = _rand(g, N, L, D, dtype=dtype), _rand(g, N, D)
    return t, gh, gl


def _run_scan(ops, t, gh, gl, dev):
    d = {k: v.detach().to(dev) if v is not None else None for k, v in t.items()}
    names = [k for k in ("gate", "value", "state", "decay") if d[k] is not None]
    for k in names:
        d[k].requires_grad_()
    h, last = ops.gated_scan(d["gate"], d["value"], **{k: d[k] for k in ("lens", "state", "gaps", "decay")})
    grads = torch.autograd.grad((h, last), [d[k] for k in names], (gh.to(dev), gl.to(dev)))
    return h, last, dict(zip(names, grads))


def _oracle_scan(t, gh, gl):
    w = {k: v.detach().double().requires_grad_() if k in ("gate", "value", "state", "decay") and v is not None else v
         for k, v in t.items()}
    names = [k for k in ("gate", "value", "state", "decay") if w[k] is not None]
    h, last = ho.scan(**w)
    live = ho.live_rows(t["lens"], *h.shape[:2])[..., None]
    grads = torch.autograd.grad((h, last), [w[k] for k in names], (torch.where(live, gh.double(), 0.0), gl.double()))
    return h.detach(), last.detach(), dict(zip(names, grads))


def _scan_bound(t, gh, gl, want_h):
    """A step forms a (1 + 8 F) and (1 - a) (1 + 16 F) (exponentials, a
    reciprocal, products) and adds; a <= 1 and the states stay below M, so an
    error of e a step becomes at most e / (1 - a) or e a step for the length:
    the smaller of L and that, here L (the longest) as the cover."""
    L = t["gate"].shape[1]
    M = max(float(want_h.abs().max()), float(t["value"].abs().max()),
            float(t["state"].abs().max()) if t["state"] is not None else 0.0)
    G = float(gh.double().abs().max()) * min(L, 200) + float(gl.abs().max())   # (sigmoid(7) ^ 200 < 0.85)
    gap = float(t["gaps"].max() * t["decay"].max()) if t["gaps"] is not None else 0.0
    return M, G, (24 + 4 * gap) * ho.F * min(L, 64)


@pytest.mark.parametrize("case", SCAN, ids=str)
def test_scan(ops, gpu, case):
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
    if "decay" in wg:   # a sum over every event
        terms = case[0] * case[1]
        _close(grads["decay"], wg["decay"], 8 * e * G * M * float(t["gaps"].max()) * math.sqrt(terms)
               + terms * ho.F * wg["decay"].abs().max(), "decay")


def test_scan_strides_and_garbage_past_the_lengths(ops, gpu):
    """Channels of a wider tensor, sequences interleaved, NaN and infinities
    past every length: the same bits as contiguous clean inputs."""
    t, gh, gl = _scan_inputs(6, 21, 20, FP32, True, True, True, seed=3)
    live = ho.live_rows(t["lens"], 6, 21)[..., None]
    h, last, grads = _run_scan(ops, t, gh, gl, gpu)
    bad = torch.full((21, 6, 64), math.nan)
    dirty = dict(t)
    for name, col, x in (("gate", 1, math.inf), ("value", 37, math.nan)):
        wide = bad.clone()
        wide[..., col:col + 20] = torch.where(live, t[name], x).transpose(0, 1)
        dirty[name] = wide.to(gpu).transpose(0, 1)[..., col:col + 20]
        assert not dirty[name].is_contiguous()
    dirty["gaps"] = torch.where(live[..., 0], t["gaps"], math.nan)
    ghd = torch.where(live, gh, math.nan)
    h2, last2, grads2 = _run_scan(ops, dirty, ghd, gl, gpu)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    assert all(torch.equal(grads[k], grads2[k]) for k in grads)
    assert not h[~live[..., 0].to(gpu)].any()


def test_scan_one_event_at_a_time_is_the_whole(ops, gpu):
    """Serving: each event with the state before it gives the states of the
    whole sequence, and an empty sequence keeps its state."""
    t, _, _ = _scan_inputs(5, 9, 12, FP32, True, False, True, seed=4)
    d = {k: v.to(gpu) if v is not None else None for k, v in t.items()}
    h, last = ops.gated_scan(d["gate"], d["value"], state=d["state"], gaps=d["gaps"], decay=d["decay"])
    s = d["state"]
    for i in range(9):
        hi, s = ops.gated_scan(d["gate"][:, i:i + 1], d["value"][:, i:i + 1], state=s, gaps=d["gaps"][:, i:i + 1],
                               decay=d["decay"])
        assert torch.equal(hi[:, 0], h[:, i])
    assert torch.equal(s, last)
    none = torch.zeros(5, dtype=torch.int32, device=gpu)
    h0, s0 = ops.gated_scan(d["gate"], d["value"], lens=none, state=d["state"])
    assert not h0.any() and torch.equal(s0, d["state"])
    h0, s0 = ops.gated_scan(d["gate"][:, :0], d["value"][:, :0], state=d["state"])
    assert h0.shape == (5, 0, 12) and torch.equal(s0, d["state"])


def test_scan_gates_at_their_ends(ops, gpu):
    """Gates of +-100 and +-30: nothing overflows, 1 - a keeps its digits."""
    gate = torch.tensor([100.0, 30.0, 12.0, -12.0, -30.0, -100.0]).reshape(1, 1, 6).expand(2, 5, 6).contiguous()
    t = dict(gate=gate, value=torch.ones(2, 5, 6), lens=None, state=torch.zeros(2, 6), gaps=None, decay=None)
    gh, gl = torch.ones(2, 5, 6), torch.zeros(2, 6)
    h, _, grads = _run_scan(ops, t, gh, gl, gpu)
    wh, _, wg = _oracle_scan(t, gh, gl)
    # each factor is good to its own digits; the gate's gradient lam (h - value) a (1 - a) has the difference of
    # two float32 values of at most one, off by a rounding for each of the five steps, and lam is at most five
    diff = 5 * 5 * 2 * ho.F * torch.sigmoid(gate.double()) * torch.sigmoid(-gate.double())
    _close(h, wh, 64 * ho.F * wh.abs() + 1e-37, "h")
    _close(grads["value"], wg["value"], 64 * ho.F * wg["value"].abs() + 1e-37, "value")
    _close(grads["gate"], wg["gate"], 64 * ho.F * wg["gate"].abs() + diff + 1e-37, "gate")


# ------------------------------------------------------------------ cross attention
#        N  Lq  Lk  Hq Hkv dh  dtype  buckets m two lens mask
ATTEND = [
    (1, 1, 1, 1, 1, 1, FP32, 0, 0, False, False, False),
    (5, 1, 10, 2, 2, 50, FP32, 32, 0, False, True, False),
    (4, 20, 32, 4, 4, 43, BF16, 32, 0, True, True, True),
    (3, 5, 7, 4, 2, 16, FP16, 8, 1, False, True, True),
    (2, 65, 64, 2, 1, 64, BF16, 16, 2, True, True, False),
    (2, 33, 130, 6, 2, 32, FP32, 32, 4, True, True, True),
    (2, 64, 129, 3, 3, 100, FP32, 12, 0, True, True, False),
    (1, 130, 70, 4, 1, 128, BF16, 64, 1, False, False, True),
    (2, 17, 65, 8, 1, 72, FP16, 0, 0, False, True, True),
    (3, 1, 300, 8, 2, 64, BF16, 40, 1, False, True, False),
    (2, 3, 257, 2, 2, 33, FP16, 20, 3, True, True, True),
    (6, 16, 16, 1, 1, 8, BF16, 4, 0, True, True, True),
]


def _attend_inputs(N, Lq, Lk, Hq, Hkv, dh, dtype, buckets, m, two, lens, mask, seed=0, grad_std=1.0):
    g = torch.Generator().manual_seed(seed)
    t = dict(q=_rand(g, N, Lq, Hq, dh, dtype=dtype), k=_rand(g, N, Lk, Hkv, dh, dtype=dtype),
             v=_rand(g, N, Lk, Hkv, dh, dtype=dtype), go=_rand(g, N, Lq, Hq, dh, dtype=dtype, std=grad_std))
    t["q_lens"], t["k_lens"] = (_lens(g, N, Lq), _lens(g, N, Lk).flip(0)) if lens else (None, None)
    t["key_mask"] = torch.rand(N, Lk, generator=g) < 0.7 if mask else None
    if mask:
        t["key_mask"][0] = False   # rows without a live key
    kw, cols = {}, None
    if buckets:
        t["bias"] = _rand(g, Hq, buckets * (2 if two else 1))
        far = 2 ** 34 if N > 2 else 1 << 12
        t["q_pos"] = torch.randint(-far, far, (N, Lq), generator=g)
        t["k_pos"] = torch.randint(-far, far, (N, Lk), generator=g) if N % 2 else \
            t["q_pos"][:, :1] - torch.randint(-70, 70, (N, Lk), generator=g)
        kw = dict(resolution=m, two_sided=two)
        cols = ho.columns(t["q_pos"], t["k_pos"], buckets, m, two)
    return t, kw, cols


def _run_attend(ops, t, kw, dev):
    d = {k: v.detach().to(dev) if v is not None else None for k, v in t.items()}
    leaves = [k for k in ("q", "k", "v", "bias") if d.get(k) is not None]
    for k in leaves:
        d[k].requires_grad_()
    o = ops.cross_attention(d["q"], d["k"], d["v"], **{k: v for k, v in d.items() if k not in ("q", "k", "v", "go")},
                            **kw)
    return o, dict(zip(["d" + k for k in leaves], torch.autograd.grad(o, [d[k] for k in leaves], d["go"])))


@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attention(ops, gpu, case):
    t, kw, cols = _attend_inputs(*case)
    o, grads = _run_attend(ops, t, kw, gpu)
    want, bound = ho.attend(**{k: t.get(k) for k in ("q", "k", "v", "go", "q_lens", "k_lens", "key_mask", "bias")},
                            cols=cols)
    _close(o, want["o"], bound["o"], "o")
    for k, got in grads.items():
        _close(got, want[k], bound[k], k)


@pytest.mark.parametrize("std", [1e-5, 3e3])
def test_attention_half_gradients_keep_their_digits(ops, gpu, std):
    """fp16 gradients far from one: ds neither vanishes nor overflows."""
    t, kw, cols = _attend_inputs(2, 24, 40, 2, 2, 32, FP16, 8, 0, True, True, False, grad_std=std)
    o, grads = _run_attend(ops, t, kw, gpu)
    want, bound = ho.attend(**{k: t.get(k) for k in ("q", "k", "v", "go", "q_lens", "k_lens", "key_mask", "bias")},
                            cols=cols)
    for k, got in grads.items():
        _close(got, want[k], bound[k], k)


def test_attention_strides_and_garbage_in_masked_places(ops, gpu):
    """Heads out of a fused projection, sequences interleaved, NaN and
    infinities in keys past the length or masked and in rows past the query
    length: the same bits as clean contiguous inputs."""
    for dtype in (FP32, BF16):
        t, kw, _ = _attend_inputs(4, 19, 37, 4, 2, 24, dtype, 16, 1, True, True, True, seed=5)
        o, grads = _run_attend(ops, t, kw, gpu)
        keys = (ho.live_rows(t["k_lens"], 4, 37) & t["key_mask"])[..., None, None]
        rows = ho.live_rows(t["q_lens"], 4, 19)[..., None, None]
        d = dict(t)
        d["q"] = torch.where(rows, t["q"], math.nan).to(dtype)
        d["go"] = torch.where(rows, t["go"], math.nan).to(dtype)
        kv = torch.full((37, 4, 5, 24), math.nan, dtype=dtype)
        kv[:, :, 0:2] = torch.where(keys, t["k"], math.inf).to(dtype).transpose(0, 1)
        kv[:, :, 3:5] = torch.where(keys, t["v"], -math.inf).to(dtype).transpose(0, 1)
        kv = kv.to(gpu).transpose(0, 1)
        d["k"], d["v"] = kv[:, :, 0:2], kv[:, :, 3:5]
        d["k_pos"] = t["k_pos"].t().contiguous().to(gpu).t()
        d["key_mask"] = t["key_mask"].t().contiguous().to(gpu).t()
        o2, grads2 = _run_attend(ops, d, kw, gpu)
        assert torch.equal(o, o2)
        for k in grads:
            assert torch.equal(grads[k], grads2[k]), k
        assert not o[~rows[..., 0, 0].to(gpu)].any()
        assert not grads["dk"][~keys[..., 0, 0].to(gpu)].any()


def test_attention_broadcast_positions_and_index_bias(ops, gpu):
    """Positions as indexes, one row expanded over the sequences; a bias whose
    one bucket holds everything adds nothing to the softmax."""
    t, _, _ = _attend_inputs(3, 6, 11, 2, 2, 8, FP32, 0, 0, False, True, False, seed=6)
    qp, kp = torch.arange(6, device=gpu).expand(3, 6), torch.arange(11, device=gpu).expand(3, 11)
    d = {k: v.to(gpu) if v is not None else None for k, v in t.items()}
    plain = ops.cross_attention(d["q"], d["k"], d["v"], q_lens=d["q_lens"], k_lens=d["k_lens"])
    one = ops.cross_attention(d["q"], d["k"], d["v"], q_lens=d["q_lens"], k_lens=d["k_lens"],
                              bias=torch.full((2, 1), 0.5, device=gpu), q_pos=qp, k_pos=kp)
    assert torch.allclose(plain, one, rtol=1e-5, atol=1e-6)
    table = torch.randn(2, 8, generator=torch.Generator().manual_seed(1))
    got = ops.cross_attention(d["q"], d["k"], d["v"], q_lens=d["q_lens"], k_lens=d["k_lens"], bias=table.to(gpu),
                              q_pos=qp, k_pos=kp, two_sided=True)
    cols = ho.columns(qp.cpu(), kp.cpu(), 4, 0, True)
    want, bound = ho.attend(t["q"], t["k"], t["v"], t["go"], q_lens=t["q_lens"], k_lens=t["k_lens"], bias=table,
                            cols=cols)
    _close(got, want["o"], bound["o"], "o")


def test_attention_shapes_without_work(ops, gpu):
    e = lambda *s: torch.randn(*s, device=gpu, requires_grad=True)
    for N, Lq, Lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v, b = e(N, Lq, 2, 8), e(N, Lk, 2, 8), e(N, Lk, 2, 8), e(2, 4)
        z = lambda n: torch.zeros(N, n, dtype=torch.int64, device=gpu)
        o = ops.cross_attention(q, k, v, bias=b, q_pos=z(Lq), k_pos=z(Lk))
        assert o.shape == (N, Lq, 2, 8) and not o.any()
        for g in torch.autograd.grad(o, (q, k, v, b), torch.ones_like(o)):
            assert not g.any()


def test_distance_bucket_matches_the_definition(ops, gpu):
    d = sorted({s * (x + y) for x in [0] + [1 << e for e in range(40)] for y in (-1, 0, 1) for s in (1, -1)})
    t = torch.tensor(d)
    for m in range(5):
        for nb in (1, 5, 32, 64):
            got = ops.distance_bucket(t, nb, m)
            assert got.tolist() == [ho.bucket(x, nb, m, True) - (nb if x < 0 else 0) for x in d]


# ------------------------------------------------------------------ gated norm
NORM = [(1, 1, FP32, False), (3, 5, FP32, False), (400, 100, FP32, False), (77, 100, FP32, True), (33, 172, BF16, False),
        (50, 43, BF16, True), (9, 512, FP16, True), (130, 64, FP16, False), (6, 1000, BF16, False), (5, 1025, FP32, True),
        (4, 2048, BF16, True), (3, 3001, FP32, False), (2, 8192, FP16, False), (2, 8191, FP32, True)]


def _norm_inputs(rows, D, dtype, rms, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = dict(x=_rand(g, rows, D, dtype=dtype), z=_rand(g, rows, D, dtype=dtype, std=2.0, mean=0.5),
             gate=_rand(g, rows, D, dtype=dtype, std=2.0), scale=_rand(g, D, std=0.2, mean=0.5),
             post_weight=_rand(g, D, std=0.2, mean=1.0), pre_weight=_rand(g, D, std=0.2, mean=1.0))
    if not rms:
        t.update(post_bias=_rand(g, D, std=0.2), pre_bias=_rand(g, D, std=0.2))
    return t, (_rand(g, rows, D, dtype=dtype), _rand(g, rows, D, dtype=dtype))


def _run_norm(ops, t, gs, dev, rms):
    d = {k: v.detach().to(dev).requires_grad_() for k, v in t.items()}
    y, n = ops.gated_norm(d["x"], d["z"], d["gate"], d["scale"], rms=rms,
                          **{k: d[k] for k in d if k.endswith(("weight", "bias"))})
    return y, n, dict(zip(d, torch.autograd.grad((y, n), list(d.values()), [g.to(dev) for g in gs])))


@pytest.mark.parametrize("case", NORM, ids=str)
def test_norm(ops, gpu, case):
    rows, D, dtype, rms = case
    t, gs = _norm_inputs(*case)
    y, n, grads = _run_norm(ops, t, gs, gpu, rms)
    w = {k: v.double().requires_grad_() for k, v in t.items()}
    wy, wn = ho.norm(w["x"], w["z"], w["gate"], w["scale"], w["post_weight"], w["pre_weight"], w.get("post_bias"),
                     w.get("pre_bias"), rms=rms)
    wg = dict(zip(w, torch.autograd.grad((wy, wn), list(w.values()), [g.double() for g in gs])))
    # a row's sums of D terms (in a tree of lanes: under 2 sqrt(D) + 16 roundings) and some twenty
    # products; a row's own 1 / sqrt(var + eps) multiplies what its values are off by
    u, e = ho.unit(dtype), (2 * math.sqrt(D) + 40) * ho.F
    def spread(t):
        c = t if rms else t - t.mean(-1, keepdim=True)
        return torch.rsqrt(c.square().mean(-1, keepdim=True) + 1e-5)
    top = lambda t: t.abs().amax(-1, keepdim=True)
    ry, rz = spread(wy.detach()), spread(w["z"].detach())
    by = e * (top(wy) + 4 * rz * top(t["z"].double())).detach()
    bn = (4 * by * ry * (1 + top(wn)) + e * top(wn)).detach()
    _close(y, wy.detach(), u * wy.detach().abs() + by, "y")
    _close(n, wn.detach(), u * wn.detach().abs() + bn, "n")
    big = (top(gs[0].double()) + 8 * top(gs[1].double()) * (ry + 1)) * 8
    amp = (1 + ry * by / e) * (1 + top(wn)).detach()
    for k in ("x", "z", "gate"):
        extra = (1 + rz) * (1 + top(t["z"].double()) * rz) if k == "z" else 1 + top(t["z"].double()) * rz
        _close(grads[k], wg[k], u * wg[k].abs() + e * big * amp * extra + torch.finfo(dtype).smallest_normal, k)
    row = (e * big * amp * (1 + top(t["z"].double()) * rz) ** 2).sum(0)
    for k in grads:
        if k not in ("x", "z", "gate"):
            _close(grads[k], wg[k], 4 * row + rows * ho.F * wg[k].abs().max(), k)


def test_norm_strides_parts_and_single_outputs(ops, gpu):
    """Rows of a wider tensor and a 3-d view give the contiguous rows' bits;
    one output's gradient alone is that of the other being zero."""
    t, gs = _norm_inputs(24, 20, FP32, False, seed=2)
    y, n, grads = _run_norm(ops, t, gs, gpu, False)
    wide = torch.full((24, 90), math.nan, device=gpu)
    d = {k: v.to(gpu) for k, v in t.items()}
    for i, k in enumerate(("x", "z", "gate")):
        wide[:, 30 * i + 1:30 * i + 21] = d[k]
        d[k] = wide[:, 30 * i + 1:30 * i + 21].unflatten(0, (4, 6)).detach().requires_grad_()
    kw = {k: d[k] for k in d if k.endswith(("weight", "bias"))}
    y2, n2 = ops.gated_norm(d["x"], d["z"], d["gate"], d["scale"], **kw)
    assert torch.equal(y2.reshape(24, 20), y) and torch.equal(n2.reshape(24, 20), n)
    g2 = torch.autograd.grad((y2, n2), (d["x"], d["z"], d["gate"]), [g.to(gpu).reshape(4, 6, 20) for g in gs])
    for k, got in zip(("x", "z", "gate"), g2):
        assert torch.equal(got.reshape(24, 20), grads[k])
    y3, n3 = ops.gated_norm(d["x"], d["z"], d["gate"], d["scale"], **kw)
    only = torch.autograd.grad(y3, d["z"], torch.ones_like(y3), retain_graph=True)[0]
    both = torch.autograd.grad((y3, n3), d["z"], (torch.ones_like(y3), torch.zeros_like(n3)))[0]
    assert torch.equal(only, both)
    none = ops.gated_norm(*[torch.randn(0, 8, device=gpu)] * 3, torch.ones(8, device=gpu),
                          post_weight=torch.ones(8, device=gpu), pre_weight=torch.ones(8, device=gpu))
    assert none[0].shape == (0, 8)


def test_norm_constant_rows(ops, gpu):
    """A row without spread: eps alone divides; nothing is infinite."""
    t, gs = _norm_inputs(4, 32, FP32, False, seed=7)
    t["z"] = torch.full((4, 32), 3.0)
    t["x"], t["post_bias"] = torch.zeros(4, 32), torch.zeros(32)
    y, n, grads = _run_norm(ops, t, gs, gpu, False)
    assert not y.any() and torch.equal(n.cpu(), t["pre_bias"].expand(4, 32))
    assert all(torch.isfinite(g).all() for g in grads.values())


# ------------------------------------------------------------------ the three together
def _block(ops, p, x, cnt, q, gaps, pos, qpos):
    """A window encoder: norm, scan, gated residual, attention of one root row."""
    n0 = torch.nn.functional.layer_norm(x, x.shape[-1:])
    f, v, g = (n0 @ p["in"]).chunk(3, -1)
    h, _ = ops.gated_scan(f, v, lens=cnt, gaps=gaps, decay=p["decay"])
    y, n = ops.gated_norm(x, h, g, p["scale"], post_weight=p["post"], pre_weight=p["pre"], rms=True)
    k, val = (n @ p["kv"]).unflatten(-1, (2, 2, -1)).unbind(2)
    return ops.cross_attention((q @ p["q"]).unflatten(-1, (4, -1)), k, val, k_lens=cnt, bias=p["bias"], q_pos=qpos,
                               k_pos=pos)


class _Oracle:
    """The same calls in float64 (differentiable)."""

    @staticmethod
    def gated_scan(f, v, lens, gaps, decay):
        return ho.scan(f, v, lens, None, gaps, decay)

    @staticmethod
    def gated_norm(x, z, g, scale, post_weight, pre_weight, rms):
        return ho.norm(x, z, g, scale, post_weight, pre_weight, rms=rms)

    @staticmethod
    def cross_attention(q, k, v, k_lens, bias, q_pos, k_pos):
        G = q.shape[2] // k.shape[2]
        k, v = (t.repeat_interleave(G, 2).permute(0, 2, 1, 3) for t in (k, v))
        s = q.permute(0, 2, 1, 3) @ k.transpose(-1, -2) * q.shape[-1] ** -0.5
        s = s + bias[:, ho.columns(q_pos, k_pos, bias.shape[1], 0, False)].permute(1, 0, 2, 3)
        on = ho.live_rows(k_lens, *k.shape[::2][:2])[:, None, None]
        w = torch.softmax(s.masked_fill(~on, -1e300), -1) * on
        return (w @ v).permute(0, 2, 1, 3)


def test_encoder_block_and_differences(ops, gpu):
    """The operators in a row, forward and backward, against the oracle's, and
    the loss's change along random directions against the gradients."""
    g = torch.Generator().manual_seed(11)
    N, L, D = 6, 12, 16
    p = {"in": _rand(g, D, 3 * D, std=0.3), "kv": _rand(g, D, 2 * D, std=0.3), "q": _rand(g, D, 2 * D, std=0.3),
         "decay": torch.rand(D, generator=g) * 0.3, "scale": _rand(g, D, std=0.1, mean=0.5),
         "post": _rand(g, D, std=0.1, mean=1.0), "pre": _rand(g, D, std=0.1, mean=1.0), "bias": _rand(g, 4, 12)}
    x, q, cnt = _rand(g, N, L, D), _rand(g, N, 1, D), _lens(g, N, L)
    gaps = torch.rand(N, L, generator=g)
    pos = torch.sort(torch.randint(0, 1000, (N, L), generator=g)).values
    qpos, go = torch.full((N, 1), 1001), _rand(g, N, 1, 4, D // 2)
    d = {k: v.to(gpu).requires_grad_() for k, v in p.items()}
    dev = lambda t: t.to(gpu)
    o = _block(ops, d, dev(x), dev(cnt), dev(q), dev(gaps), dev(pos), dev(qpos))
    grads = torch.autograd.grad(o, list(d.values()), dev(go))
    w = {k: v.double().requires_grad_() for k, v in p.items()}
    want = _block(_Oracle, w, x.double(), cnt, q.double(), gaps.double(), pos, qpos)
    wg = torch.autograd.grad(want, list(w.values()), go.double())
    assert torch.allclose(o.cpu().double(), want, rtol=1e-4, atol=1e-5)
    for k, a, b in zip(p, grads, wg):
        assert torch.allclose(a.cpu().double(), b, rtol=1e-3, atol=1e-4 * float(b.abs().max())), k
    # central differences of the oracle's loss (float64) along a direction, against the kernels' gradients
    for k, a in zip(p, grads):
        step = _rand(g, *p[k].shape).double()
        eps = 1e-5
        loss = []
        for s in (eps, -eps):
            moved = {n: (t.double() + s * step if n == k else t.double()) for n, t in p.items()}
            loss.append((_block(_Oracle, moved, x.double(), cnt, q.double(), gaps.double(), pos, qpos) * go).sum())
        diff = float(loss[0] - loss[1]) / (2 * eps)
        along = float((a.cpu().double() * step).sum())
        size = float((a.cpu().double().abs() * step.abs()).sum())
        assert abs(diff - along) <= 1e-4 * size + 1e-6, k


def test_results_repeat_and_replay(ops, gpu):
    """Bit-identical run to run, on another stream, and from a captured graph
    (forward and backward) replayed on new inputs."""
    ts, gh, gl = _scan_inputs(4, 700, 32, BF16, True, True, True, seed=8)
    ta, kw, _ = _attend_inputs(3, 40, 90, 4, 2, 32, BF16, 16, 0, True, True, True, seed=8)
    tn, gs = _norm_inputs(300, 172, BF16, False, seed=8)

    def everything():
        h, last, sg = _run_scan(ops, ts, gh, gl, gpu)
        o, ag = _run_attend(ops, ta, kw, gpu)
        y, n, ng = _run_norm(ops, tn, gs, gpu, False)
        return [h, last, *sg.values(), o, *ag.values(), y, n, *ng.values()]

    first = everything()
    again = everything()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = everything()
    side.synchronize()
    for a, b, c in zip(first, again, other):
        assert torch.equal(a, b) and torch.equal(a, c)

    # a captured step: static inputs, new values between the replays
    sx = {k: v.to(gpu) for k, v in ta.items() if v is not None}
    leaves = [sx[k].requires_grad_() for k in ("q", "k", "v", "bias")]
    extra = {k: v for k, v in sx.items() if k not in ("q", "k", "v", "go")}

    def step():
        o = ops.cross_attention(sx["q"], sx["k"], sx["v"], **extra, **kw)
        hs, _ = ops.gated_scan(o.flatten(2), o.flatten(2) * 0.5, lens=sx["q_lens"])
        y, n = ops.gated_norm(hs, o.flatten(2), hs, w, post_weight=w, pre_weight=w)
        return [y, n, *torch.autograd.grad((y, n), leaves, (one, one))]

    w = torch.ones(128, device=gpu)
    one = torch.ones(3, 40, 128, dtype=BF16, device=gpu)
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        static = step()
    for i in range(3):
        with torch.no_grad():
            sx["q"].mul_(0.9)
            sx["k"].add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i
