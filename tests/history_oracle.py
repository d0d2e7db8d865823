"""The history operators from their definitions in float64 on the CPU, with
bounds on how far a correct kernel may be from them (tests only).

Rounding an operand to a type is off by at most u = eps / 2 of its value;
sums and functions in float32 by F = 2^-24 a step. The bounds add what the
kernels round: the outputs, and for 16-bit tensors the attention's weights
and their gradients before a product."""
import math

import torch

F = 2.0 ** -24


def unit(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def live_rows(lens, n, most):
    at = torch.arange(most)[None]
    return at < lens.clamp(0, most).long()[:, None] if lens is not None else torch.ones(n, most, dtype=torch.bool)


def sigmoid(x):
    """Written out: its derivative then keeps its digits far from zero too."""
    return 1.0 / (1.0 + torch.exp(-x))


def scan(gate, value, lens=None, state=None, gaps=None, decay=None):
    """(h, last) in float64 (differentiable)."""
    f, v = gate.double(), value.double()
    N, L, D = f.shape
    live = live_rows(lens, N, L)
    f, v = (torch.where(live[..., None], t, torch.zeros((), dtype=t.dtype)) for t in (f, v))
    s = state.double() if state is not None else torch.zeros(N, D, dtype=torch.float64)
    out = []
    for t in range(L):
        a, b = sigmoid(f[:, t]), sigmoid(-f[:, t])
        if decay is not None:
            u = torch.where(live[:, t], gaps[:, t].double(), 0.0)[:, None] * decay.double()
            a, b = a * torch.exp(-u), b - a * torch.expm1(-u)
        new = a * s + b * v[:, t]   # (1 - a without taking a from one)
        on = live[:, t, None]
        s = torch.where(on, new, s)
        out.append(torch.where(on, new, torch.zeros_like(new)))
    return torch.stack(out, 1), s


def bucket(d, buckets, resolution, two_sided):
    """A distance at a time, in Python integers."""
    neg = d < 0
    n = min(abs(d) if two_sided else max(d, 0), 2 ** 32 - 1)
    if n < 2 ** resolution:
        b = n
    else:
        e = n.bit_length() - 1
        b = (e - resolution) * 2 ** resolution + (n >> (e - resolution))
    b = min(b, buckets - 1)
    return b + buckets if two_sided and neg else b


def columns(q_pos, k_pos, buckets, resolution, two_sided):
    d = (q_pos[:, :, None] - k_pos[:, None, :])
    flat = [bucket(int(x), buckets, resolution, two_sided) for x in d.flatten().tolist()]
    return torch.tensor(flat, dtype=torch.long).reshape(d.shape)


def attend(q, k, v, go, q_lens=None, k_lens=None, key_mask=None, bias=None, cols=None, scale=None):
    """dict of o, dq, dk, dv, dbias in float64 and ``bound``, the same of what
    the kernels may be off by. ``cols``: the bias columns [N, Lq, Lk]."""
    N, Lq, Hq, dh = q.shape
    Lk, Hkv = k.shape[1:3]
    G = Hq // Hkv
    c = dh ** -0.5 if scale is None else scale
    u = unit(q.dtype) if q.dtype != torch.float32 else 0.0
    live = live_rows(k_lens, N, Lk)
    if key_mask is not None:
        live = live & key_mask
    rows = live_rows(q_lens, N, Lq)
    z = torch.zeros((), dtype=torch.float64)
    Q, GO = (torch.where(rows[:, :, None, None], t.double(), z) for t in (q, go))
    K, V = (torch.where(live[:, :, None, None], t.double(), z) for t in (k, v))
    at = torch.arange(Hq) // G
    Q, GO, K, V = (t.permute(0, 2, 1, 3) for t in (Q, GO, K[:, :, at], V[:, :, at]))
    s = c * Q @ K.transpose(-1, -2)
    # a score: a product of dh terms, the scale, the bias and the maximum taken off
    es = F * (dh + 4) * abs(c) * (Q.abs() @ K.abs().transpose(-1, -2))
    if bias is not None:
        s = s + bias.double()[:, cols].permute(1, 0, 2, 3)
        es = es + 4 * F * bias.double().abs().max()
    on = (live[:, None, None, :] & rows[:, None, :, None]).expand_as(s)
    es = es + 4 * F * torch.where(on, s.abs(), z).amax(-1, keepdim=True)
    s = s.masked_fill(~on, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    ep = p * (2 * es.amax(-1, keepdim=True) + (8 + Lk) * F)      # p in float32
    o = p @ V
    eo = (ep + u * p) @ V.abs() + Lk * F * (p @ V.abs())
    out = {"o": o}
    bound = {"o": eo + unit(q.dtype) * (o.abs() + eo)}
    dp = GO @ V.transpose(-1, -2)
    edp = F * (dh + 2) * (GO.abs() @ V.abs().transpose(-1, -2))
    D = (GO * o).sum(-1, keepdim=True)
    eD = (GO.abs() * (bound["o"] + F * (dh + 2) * o.abs())).sum(-1, keepdim=True)
    ds = p * (dp - D)
    eds = ep * (dp - D).abs() + (p + ep) * (edp + eD) + 4 * F * ds.abs()
    eds = torch.where(on, eds, z)
    r = eds + u * (ds.abs() + eds)                              # rounded before the products
    steps = (Lq * G + Lk) * F
    out["dq"], bq = c * ds @ K, c * (r @ K.abs() + steps * (ds.abs() @ K.abs()))
    dk, bk = c * ds.transpose(-1, -2) @ Q, c * (r + steps * ds.abs()).transpose(-1, -2) @ Q.abs()
    rp = ep + u * (p + ep)
    dv, bv = p.transpose(-1, -2) @ GO, (rp + steps * p).transpose(-1, -2) @ GO.abs()
    share = lambda t: t.reshape(N, Hkv, G, Lk, dh).sum(2).permute(0, 2, 1, 3)
    out["dk"], out["dv"] = share(dk), share(dv)
    bk, bv = share(bk), share(bv)
    back = lambda t: t.permute(0, 2, 1, 3)
    out["o"], bound["o"], out["dq"], bq = back(o), back(bound["o"]), back(out["dq"]), back(bq)
    for n, b in (("dq", bq), ("dk", bk), ("dv", bv)):
        bound[n] = b + unit(q.dtype) * (out[n].abs() + b)
    if bias is not None:
        C = bias.shape[1]
        col = cols[:, None].expand_as(ds)
        db, bb = torch.zeros(Hq, C, dtype=torch.float64), torch.zeros(Hq, C, dtype=torch.float64)
        for h in range(Hq):
            db[h].index_add_(0, col[:, h].flatten(), ds[:, h].flatten())
            bb[h].index_add_(0, col[:, h].flatten(), (eds + (Lq * Lk + 64) * F * ds.abs())[:, h].flatten())
        out["dbias"], bound["dbias"] = db, bb + F * db.abs()
    # values below a type's normal range are off by half its smallest step
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    for n in ("o", "dq", "dk", "dv"):
        bound[n] = bound[n] + tiny
    return out, bound


def norm(x, z, gate, scale, post_w, pre_w, post_b=None, pre_b=None, eps=1e-5, rms=False):
    def std(t):
        t = t if rms else t - t.mean(-1, keepdim=True)
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)

    post = std(z.double()) * post_w.double()
    post = post if post_b is None else post + post_b.double()
    y = x.double() + scale.double() * torch.sigmoid(gate.double()) * post
    n = std(y) * pre_w.double()
    return y, n if pre_b is None else n + pre_b.double()
