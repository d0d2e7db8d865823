"""The losses over all candidates and the rotary positions from their
definitions in float64 on the CPU, with bounds on how far a correct kernel may
be from them (tests only).

Rounding an operand to a type is off by at most u = eps / 2 of its value; sums
and functions in float32 by F = 2^-24 a step. The bounds add what the kernels
round: the outputs, and for 16-bit tensors the softmax weights before a product."""
import math
from fractions import Fraction

import torch

INV_2PI = Fraction("0.15915494309189533576888376337251436203445964574045644874766734405889679763422653509")
F = 2.0 ** -24


def unit(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def loss(h, table, ids, weight, konst, dead, g, bias=None, scale=1.0, temperature=1.0):
    """(dict of loss, dh, dtable, dbias, the bounds) of rows that want ``weight``
    [N, K] of the candidates ``ids`` (weights of a row sum to 1; ``konst``: the
    sum of weight log weight); ``dead``: rows without loss or gradient."""
    t = h.dtype
    u = unit(t) if t != torch.float32 else 0.0
    T = float(temperature)
    (N, D), V = h.shape, table.shape[0]
    live = torch.ones(V, dtype=torch.bool) if bias is None else bias > -math.inf
    H = torch.where(dead[:, None], 0.0, h.double())
    W = torch.where(live[:, None], table.double(), 0.0)
    b = torch.zeros(V, dtype=torch.float64) if bias is None else bias.double()
    s = (scale * H @ W.t() + b) / T
    # a score: a product of D terms, the scales, the bias, the maximum taken off
    size = torch.where(live, (abs(scale) * H.abs() @ W.abs().t() + torch.where(live, b, 0.0).abs()) / T, 0.0)
    es = (F * (D + 8) * size).amax(1, keepdim=True) + 4 * F * torch.where(live, s.abs(), 0.0).amax(1, keepdim=True)
    logp = torch.log_softmax(s, 1)
    p = logp.exp()
    steps = F * (V / 8 + 32)
    rel = 2 * es + steps                                  # of p, in float32
    out, bound = {}, {}
    value = T * T * (konst - (weight * logp.gather(1, ids)).sum(1))
    err = T * T * (rel[:, 0] + F * (ids.shape[1] + 8) * (konst.abs() + (weight * logp.gather(1, ids).abs()).sum(1)))
    out["loss"], bound["loss"] = torch.where(dead, 0.0, value), torch.where(dead, 0.0, err + 2 * F * value.abs())
    G = torch.where(dead, 0.0, g.double())[:, None] * T
    q = torch.zeros_like(p).scatter_add_(1, ids, torch.where(dead[:, None], 0.0, weight))
    p = torch.where(dead[:, None], 0.0, p)
    ep = p * (rel + u)
    k = F * (ids.shape[1] + 16)
    out["dh"] = scale * G * ((p - q) @ W)
    bound["dh"] = abs(scale) * G.abs() * ((ep + k * q + 8 * F * p) @ W.abs())
    c, ec = G * (p - q), G.abs() * (p * rel + k * q + u * (p - q).abs())
    more = F * (N / 4 + 16)
    out["dtable"] = scale * c.t() @ H
    bound["dtable"] = abs(scale) * (ec + more * c.abs()).t() @ H.abs()
    out["dbias"] = c.sum(0)
    bound["dbias"] = (G.abs() * (p * rel + k * q) + more * c.abs()).sum(0)
    for n in ("dh", "dtable"):
        bound[n] = bound[n] + unit(t) * (out[n].abs() + bound[n]) + \
            torch.finfo(t).smallest_normal * torch.finfo(t).eps
    # a weight under 2^-126 of its row's largest is 0 (in bf16 one under 2^-126
    # after the factors too)
    flush = 2.0 ** -124
    bound["dh"] = bound["dh"] + flush * abs(scale) * G.abs() * W.abs().sum(0)
    bound["dtable"] = bound["dtable"] + flush * abs(scale) * ((G.abs() + 1).t() @ H.abs())
    bound["dbias"] = bound["dbias"] + flush * G.abs().sum()
    # a 16-bit weight far below its row's or column's largest is off by a step of
    # the type's least (fp16: 2^-24 of what is put at 2^7 or 2^10 and more)
    if t == torch.float16:
        bound["dh"] = bound["dh"] + abs(scale) * G.abs() * 2.0 ** -31 * W.abs().sum(0)
        bound["dtable"] = bound["dtable"] + abs(scale) * 2.0 ** -34 * c.abs().amax(0)[:, None] * H.abs().sum(0)
    return out, bound


def labels(target):
    """(ids, weight, konst, dead) of one target a row."""
    dead = target < 0
    return target.clamp(min=0)[:, None], torch.ones(len(target), 1, dtype=torch.float64), \
        torch.zeros(len(target), dtype=torch.float64), dead


def teacher(ids, logits, temperature):
    """(ids, weight, konst, dead) of a teacher's entries."""
    on = (ids >= 0) & (logits > -math.inf)
    z = torch.where(on, logits.double() / temperature, -math.inf)
    dead = ~on.any(1)
    logq = torch.log_softmax(z, 1)
    q = torch.where(on, logq.exp(), 0.0)
    return ids.clamp(min=0), q, torch.where(on, q * logq, 0.0).sum(1), dead


def rotate(x, pos, freqs, interleaved=False, gain=1.0, way=1.0):
    """(the rotated tensor, the bound) with angles from Python integers."""
    P = len(freqs)
    angle = torch.zeros(*pos.shape, P, dtype=torch.float64)
    flat = angle.view(pos.numel(), P)
    for i, f in enumerate(freqs.tolist()):
        turns = Fraction(f) * INV_2PI
        for j, t in enumerate(pos.flatten().tolist()):
            flat[j, i] = 2 * math.pi * float(t * turns % 1)
    c, s = gain * torch.cos(angle)[:, :, None], way * gain * torch.sin(angle)[:, :, None]
    y = x.double().clone()
    a, b = (y[..., 0:2 * P:2], y[..., 1:2 * P:2]) if interleaved else (y[..., :P], y[..., P:2 * P])
    new = a * c - b * s, a * s + b * c
    size = (a.abs() + b.abs()) * abs(gain)
    # the angle: the frequency in turns to 2^-63, a position times (its double
    # parts hold 2^-104 of it); the sine and cosine, products and a sum: 2^-22
    err = size * (2.0 ** -22 + pos.double().abs()[:, :, None, None] * 2.0 ** -60)
    out, bound = y.clone(), torch.zeros_like(y)
    if interleaved:
        out[..., 0:2 * P:2], out[..., 1:2 * P:2] = new
        bound[..., 0:2 * P:2], bound[..., 1:2 * P:2] = err, err
    else:
        out[..., :P], out[..., P:2 * P] = new
        bound[..., :P], bound[..., P:2 * P] = err, err
    rounded = bound + unit(x.dtype) * (out.abs() + bound) + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    rounded[..., 2 * P:] = 0.0
    return out, rounded
