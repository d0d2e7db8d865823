"""Operators of a model that answers with the next node, in cases that can be
timed and compared: softmax cross entropy of rows over every candidate node,
distillation from a teacher's top candidates, and rotary positions of queries
and keys by event time.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges,
``prepare`` makes what a program has in hand before the call, ``run`` is one
pass (the plain form in 32 bits, or with ``own`` the framework's operators),
``work`` the bytes and operations it cannot do without and ``exact`` the same
results in 64 bits.

Sizes are the benchmark's streams: 9,227 nodes (1,000 of them items) with 100
channels, 1,140,149 nodes with 100 or 172; batches of 200, 600 and 4,000
events. Logits have a spread of about 2, targets favour some candidates.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DEV = "cuda:0"
_TYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_NODES = 1_140_149
_SPAN = 2_700_000   # seconds of the stream
_PADDED = 0.3       # share of the rows without a target where a case is padded


# ------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # serving: how likely one event's destination was among all nodes
        dict(name="loss_event", op="loss", train=False, N=1, V=_NODES, D=172, dtype="bf16", bias=False, padded=False),
        # the smallest step: a batch of 200 events over the items of the small stream
        dict(name="loss_items", op="loss", train=True, N=200, V=1000, D=100, dtype="fp32", bias=False, padded=False),
        # a batch of 600 over the small stream's nodes, with a learned popularity
        dict(name="loss_batch", op="loss", train=True, N=600, V=9227, D=100, dtype="fp32", bias=True, padded=False),
        # the next node at every place of a batch's windows, padded places among them
        dict(name="loss_windows", op="loss", train=True, N=24000, V=9227, D=172, dtype="bf16", bias=False,
             padded=True),
        # a batch of 600 over all nodes of the large stream
        dict(name="loss_nodes", op="loss", train=True, N=600, V=_NODES, D=100, dtype="bf16", bias=False,
             padded=False),
        # the widest configuration: 4,000 events, 172 channels
        dict(name="loss_large", op="loss", train=True, N=4000, V=_NODES, D=172, dtype="bf16", bias=True,
             padded=False),
        # a small student of the small stream, a teacher's 20 best
        dict(name="distill_batch", op="distill", train=True, N=600, V=9227, D=100, K=20, dtype="fp32", bias=False,
             temperature=1.0),
        # both endpoints of a batch of 600 over all nodes, 64 best
        dict(name="distill_nodes", op="distill", train=True, N=1200, V=_NODES, D=172, K=64, dtype="bf16", bias=False,
             temperature=2.0),
        # many rows, wide, an odd number of candidates, scaled half precision
        dict(name="distill_wide", op="distill", train=True, N=4000, V=50001, D=256, K=100, dtype="fp16", bias=True,
             temperature=2.0),
        # serving: the query and the key of a new event of 400 roots, heads of 50
        dict(name="rotate_event", op="rotate", train=False, N=400, Lq=1, Lk=1, Hq=2, Hkv=2, dh=50, rot=50,
             dtype="fp32", interleaved=False, scaling="none"),
        # a batch's windows, odd heads, most of a head rotated
        dict(name="rotate_windows", op="rotate", train=True, N=4000, Lq=20, Lk=32, Hq=4, Hkv=4, dh=43, rot=42,
             dtype="bf16", interleaved=True, scaling="linear"),
        # few nodes' whole histories, four query heads to a key head
        dict(name="rotate_long", op="rotate", train=True, N=16, Lq=8191, Lk=8191, Hq=8, Hkv=2, dh=128, rot=128,
             dtype="fp16", interleaved=False, scaling="wavelength"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(["loss", "loss", "loss", "distill", "distill", "rotate"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "rotate":
        Hkv = rng.choice([1, 2, 3, 4])
        dh = rng.choice([8, 43, 50, 64, 100, 128, rng.randint(2, 128)])
        c = dict(op=op, train=rng.random() < 0.6, Lq=_log(rng, 1, 8191), Lk=_log(rng, 1, 8191),
                 Hq=Hkv * rng.choice([1, 2, 4]), Hkv=Hkv, dh=dh, rot=2 * rng.randint(1, dh // 2), dtype=dtype,
                 interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "base", "wavelength"]))
        c["N"] = _log(rng, 1, max(1, min(4000, 160_000_000 // ((c["Lq"] * c["Hq"] + c["Lk"] * Hkv) * dh))))
        return c
    train = op == "distill" or rng.random() < 0.75
    D = rng.choice([100, 172, rng.randint(1, 256)])
    c = dict(op=op, train=train, V=_log(rng, 3 if op == "loss" else 200, 1_150_000), D=D, dtype=dtype,
             bias=rng.random() < 0.4)
    most = 7.8e11 if dtype != "fp32" else 4e10
    c["N"] = _log(rng, 1, max(1, min(30000, int(most / (c["V"] * D)))))
    if op == "loss":
        c["padded"] = rng.random() < 0.3
    else:
        c.update(K=_log(rng, 1, 128), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]))
    return c


# ------------------------------------------------------------------ inputs from the seed
def _gen(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(_DEV).manual_seed((int(seed) * 1_000_003 + salt * 7919) % (1 << 62))


def _normal(g, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device=_DEV) * std + mean).to(dtype)


def prepare(case: dict, seed: int) -> dict:
    return _PREPARE[case["op"]](case, seed)


def _prepare_rows(c, g) -> dict:
    """Rows, table and bias, and the gradient that reaches each row's loss (a
    weighted mean; half precision trains with scaled losses)."""
    dt = _TYPE[c["dtype"]]
    s = dict(op=c["op"], train=c["train"], bias=None)
    s["h"] = _normal(g, c["N"], c["D"], dtype=dt)
    s["table"] = _normal(g, c["V"], c["D"], dtype=dt, std=2.0 / math.sqrt(c["D"]))
    leaves = ["h", "table"]
    if c["bias"]:
        s["bias"] = _normal(g, c["V"], std=0.7)
        leaves.append("bias")
    if c["train"]:
        top = 65536.0 if c["dtype"] == "fp16" else 1.0
        s["grads"] = ((torch.rand(c["N"], generator=g, device=_DEV) + 0.5) * (top / c["N"]),)
        s["leaves"] = [s[k].requires_grad_() for k in leaves]
    return s


def _prepare_loss(c, seed):
    g = _gen(seed, 1)
    s = _prepare_rows(c, g)
    u = torch.rand(c["N"], generator=g, device=_DEV)
    s["target"] = (u * u * c["V"]).long().clamp(max=c["V"] - 1)
    if c["padded"]:
        s["target"][torch.rand(c["N"], generator=g, device=_DEV) < _PADDED] = -1
    return s


def _prepare_distill(c, seed):
    g = _gen(seed, 2)
    s = _prepare_rows(c, g)
    N, V, K = c["N"], c["V"], c["K"]
    # K different candidates a row, best first; a few rows have fewer
    step = torch.randint(1, V // K + 1, (N, K), generator=g, device=_DEV)
    at = step.cumsum(1) + torch.randint(0, V, (N, 1), generator=g, device=_DEV)
    order = torch.rand(N, K, generator=g, device=_DEV).argsort(1)
    s["ids"] = torch.gather(at % V, 1, order)
    fewer = (torch.rand(N, 1, generator=g, device=_DEV) < 0.1) & (torch.arange(K, device=_DEV) >= (K + 1) // 2)
    s["ids"][fewer] = -1
    s["logits"] = torch.sort(_normal(g, N, K, std=1.5, mean=4.0), dim=1, descending=True).values
    s["temperature"] = c["temperature"]
    return s


def _prepare_rotate(c, seed):
    g, dt = _gen(seed, 3), _TYPE[c["dtype"]]
    N, Lq, Lk, dh = c["N"], c["Lq"], c["Lk"], c["dh"]
    s = dict(op="rotate", train=c["train"], rot=c["rot"], interleaved=c["interleaved"],
             gain=1.1 if c["scaling"] == "wavelength" else 1.0)
    s["q"] = _normal(g, N, Lq, c["Hq"], dh, dtype=dt)
    s["k"] = _normal(g, N, Lk, c["Hkv"], dh, dtype=dt)
    s["k_pos"] = torch.sort(torch.randint(0, _SPAN, (N, Lk), generator=g, device=_DEV), dim=1).values
    s["q_pos"] = _SPAN + torch.sort(torch.randint(0, 5000, (N, Lq), generator=g, device=_DEV), dim=1).values
    # angles a second, one for each pair of channels
    i = torch.arange(c["rot"] // 2, device=_DEV, dtype=torch.float64)
    base = 10000.0 * (30.0 if c["scaling"] == "base" else 1.0)
    f = base ** (-2.0 * i / c["rot"])
    if c["scaling"] == "linear":
        f = f / 60.0
    if c["scaling"] == "wavelength":   # long waves stretched, short ones kept
        keep = ((f * 8192.0 / (2.0 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * keep + f / 16.0 * (1.0 - keep)
    s["freqs"] = f
    if c["train"]:
        s["grads"] = (_normal(g, N, Lq, c["Hq"], dh, dtype=dt), _normal(g, N, Lk, c["Hkv"], dh, dtype=dt))
        s["leaves"] = [s[k].requires_grad_() for k in ("q", "k")]
    return s


_PREPARE = {"loss": _prepare_loss, "distill": _prepare_distill, "rotate": _prepare_rotate}


# ------------------------------------------------------------------ one pass
def run(state: dict):
    """The operator's outputs and, in training, the gradients of every leaf."""
    s = state
    if not own:
        with torch.no_grad():
            return _PLAIN[s["op"]](s)
    if not s["train"]:
        with torch.no_grad():
            return _OWN[s["op"]](s)
    outs = _OWN[s["op"]](s)
    return (*outs, *torch.autograd.grad(outs, s["leaves"], s["grads"]))


def _native():
    if "starry_unigraph" not in sys.modules:
        path = str(Path(__file__).resolve().parents[1] / "starrygl-unidyngraph_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
    from starry_unigraph.native import candidates, rotary
    return candidates, rotary


def _own_loss(s):
    return (_native()[0].cross_entropy(s["h"], s["table"], s["target"], bias=s["bias"]),)


def _own_distill(s):
    return (_native()[0].distillation(s["h"], s["table"], s["ids"], s["logits"], bias=s["bias"],
                                      temperature=s["temperature"]),)


def _own_rotate(s):
    return _native()[1].rotate(s["q"], s["k"], s["q_pos"], s["k_pos"], s["freqs"], interleaved=s["interleaved"],
                               gain=s["gain"])


_OWN = {"loss": _own_loss, "distill": _own_distill, "rotate": _own_rotate}


def _plain_rows(s, ids, weight, const, temperature):
    """The loss of rows whose wanted distribution is ``weight`` [N, K] on the
    candidates ``ids`` (``const``: its sum of w log w), over pieces of the
    table, and the gradients."""
    h, table, bias = s["h"].float(), s["table"], s["bias"]
    (N, D), V = h.shape, table.shape[0]
    scale = 1.0 / temperature
    piece = max(1, 120_000_000 // N)
    live = weight.sum(1) > 0

    def scores(lo, hi):
        z = torch.matmul(h, table[lo:hi].float().t())
        return (z if bias is None else z + bias[lo:hi]) * scale

    top = torch.full((N, 1), -torch.inf, device=h.device)
    total = torch.zeros(N, 1, device=h.device)
    for lo in range(0, V, piece):
        z = scores(lo, min(V, lo + piece))
        m = torch.maximum(top, z.amax(1, keepdim=True))
        total = total * torch.exp(top - m) + torch.exp(z - m).sum(1, keepdim=True)
        top = m
    lse = top + torch.log(total)
    rows = table[ids].float()                       # [N, K, D]
    mine = (h.unsqueeze(1) * rows).sum(-1)
    mine = (mine if bias is None else mine + bias[ids]) * scale
    loss = const + (weight * (lse - mine)).sum(1)
    loss = torch.where(live, loss * temperature * temperature, 0.0)
    if not s["train"]:
        return (loss,)
    g = torch.where(live, s["grads"][0] * temperature, 0.0).unsqueeze(1)
    dh = -(weight.unsqueeze(-1) * rows).sum(1) * g
    dtable = torch.empty(V, D, device=h.device)
    dbias = torch.empty(V, device=h.device)
    for lo in range(0, V, piece):
        hi = min(V, lo + piece)
        p = torch.exp(scores(lo, hi) - lse) * g
        dh = dh + torch.matmul(p, table[lo:hi].float())
        dtable[lo:hi] = torch.matmul(p.t(), h)
        dbias[lo:hi] = p.sum(0)
    wanted = weight * g
    dtable.index_add_(0, ids.flatten(), -(wanted.unsqueeze(-1) * h.unsqueeze(1)).flatten(0, 1))
    dbias.index_add_(0, ids.flatten(), -wanted.flatten())
    grads = (dh.to(s["h"].dtype), dtable.to(table.dtype))
    return (loss, *grads) if bias is None else (loss, *grads, dbias)


def _plain_loss(s):
    t = s["target"].unsqueeze(1)
    return _plain_rows(s, t.clamp(min=0), (t >= 0).float(), 0.0, 1.0)


def _plain_distill(s):
    live = s["ids"] >= 0
    z = torch.where(live, s["logits"] / s["temperature"], -torch.inf)
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    weight = e / total
    const = torch.where(live, weight * (z - torch.log(total)), 0.0).sum(1)
    return _plain_rows(s, s["ids"].clamp(min=0), weight, const, s["temperature"])


def _plain_rotate(s):
    rot, inter = s["rot"], s["interleaved"]

    def turn(x, pos, sign):
        t = pos.double().unsqueeze(-1) * s["freqs"]
        c, n = (torch.cos(t) * s["gain"]).float().unsqueeze(2), (torch.sin(t) * (sign * s["gain"])).float().unsqueeze(2)
        y = x.float()
        a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if inter else (y[..., :rot // 2], y[..., rot // 2:rot])
        u, v = a * c - b * n, a * n + b * c
        turned = torch.stack((u, v), -1).flatten(-2) if inter else torch.cat((u, v), -1)
        return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)

    outs = (turn(s["q"], s["q_pos"], 1.0), turn(s["k"], s["k_pos"], 1.0))
    if not s["train"]:
        return outs
    gq, gk = s["grads"]
    return (*outs, turn(gq, s["q_pos"], -1.0), turn(gk, s["k_pos"], -1.0))


_PLAIN = {"loss": _plain_loss, "distill": _plain_distill, "rotate": _plain_rotate}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    c, size = case, 4 if case["dtype"] == "fp32" else 2
    if c["op"] == "rotate":
        n = c["N"] * (c["Lq"] * c["Hq"] + c["Lk"] * c["Hkv"])
        passes = 2 if c["train"] else 1
        pos = 8 * c["N"] * (c["Lq"] + c["Lk"])
        return {"bytes": 2 * passes * n * c["dh"] * size + pos, "flops": 3 * passes * n * c["rot"]}
    N, V, D = c["N"], c["V"], c["D"]
    live = N * (1 - _PADDED) if c.get("padded") else N
    read = (live * D + V * D) * size + (4 * V if c["bias"] else 0)
    read += 12 * N * c["K"] if c["op"] == "distill" else 8 * N
    written, flops = 4 * N, 2 * live * V * D
    if c["train"]:   # the scores twice (they are not kept), and a product for each gradient
        read += 4 * N
        written += (N + V) * D * size + (4 * V if c["bias"] else 0)
        flops *= 4
    return {"bytes": read + written, "flops": flops}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](s)


def _exact_wanted(s, wanted_of, temperature):
    """Rows in blocks, each with its whole distribution: ``wanted_of(lo, hi)``
    is (ids, probabilities, sum of their w log w, live rows)."""
    h, table = s["h"].double(), s["table"].double()
    (N, D), V = h.shape, table.shape[0]
    bias = None if s["bias"] is None else s["bias"].double()
    loss = torch.zeros(N, dtype=torch.float64, device=h.device)
    dh, dtable = torch.zeros_like(h), torch.zeros_like(table)
    dbias = torch.zeros(V, dtype=torch.float64, device=h.device)
    block = max(1, 400_000_000 // V)
    for lo in range(0, N, block):
        hi = min(N, lo + block)
        ids, w, plogp, live = wanted_of(lo, hi)
        z = torch.mm(h[lo:hi], table.t())
        if bias is not None:
            z += bias
        logp = torch.log_softmax(z / temperature, 1)
        del z
        loss[lo:hi] = temperature ** 2 * (plogp - (w * logp.gather(1, ids)).sum(1)) * live
        if not s["train"]:
            continue
        d = logp.exp_() * live.unsqueeze(1)
        d.scatter_add_(1, ids, -w)
        d *= temperature * s["grads"][0][lo:hi].double().unsqueeze(1)
        dh[lo:hi] = torch.mm(d, table)
        dtable += torch.mm(d.t(), h[lo:hi])
        dbias += d.sum(0)
    if not s["train"]:
        return (loss,)
    return (loss, dh, dtable) if bias is None else (loss, dh, dtable, dbias)


def _exact_loss(s):
    def wanted(lo, hi):
        t = s["target"][lo:hi]
        live = (t >= 0).double()
        return t.clamp(min=0).unsqueeze(1), live.unsqueeze(1), torch.zeros_like(live), live

    return _exact_wanted(s, wanted, 1.0)


def _exact_distill(s):
    def wanted(lo, hi):
        ids = s["ids"][lo:hi]
        logq = torch.log_softmax((s["logits"][lo:hi].double() / s["temperature"]).masked_fill(ids < 0, -torch.inf), 1)
        w = logq.exp()
        return ids.clamp(min=0), w, (w * logq.masked_fill(ids < 0, 0.0)).sum(1), torch.ones_like(w[:, 0])

    return _exact_wanted(s, wanted, s["temperature"])


def _exact_rotate(s):
    rot = s["rot"]
    at = torch.arange(rot, device=_DEV)
    # each channel's pair, its partner, and the sign of the partner's sine
    pair = at // 2 if s["interleaved"] else at % (rot // 2)
    partner = at ^ 1 if s["interleaved"] else (at + rot // 2) % rot
    second = at % 2 == 1 if s["interleaved"] else at >= rot // 2
    sign = torch.where(second, 1.0, -1.0).double()

    def turn(x, pos, way):
        angle = (pos.double()[..., None] * s["freqs"])[..., None, pair]
        y = x.double().clone()
        z = y[..., :rot]
        y[..., :rot] = s["gain"] * (z * torch.cos(angle) + way * sign * z[..., partner] * torch.sin(angle))
        return y

    outs = (turn(s["q"], s["q_pos"], 1.0), turn(s["k"], s["k_pos"], 1.0))
    if not s["train"]:
        return outs
    return (*outs, turn(s["grads"][0], s["q_pos"], -1.0), turn(s["grads"][1], s["k_pos"], -1.0))


_EXACT = {"loss": _exact_loss, "distill": _exact_distill, "rotate": _exact_rotate}
