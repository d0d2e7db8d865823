"""A root's embedding from its window of past events as a sequence: one block of
a gated recurrence over the window and one attention of the root over the
block's outputs (native.history's operators). The reference has no such
embedding (its own attends over the window's rows as a set,
backends/ctdg/runtime/models.py:77-137)."""
from __future__ import annotations

import torch
import torch.nn as nn

from starry_unigraph.native import history, rotary


class HistoryEncoder(nn.Module):
    """Embeddings [N, dim] of N roots, each with a window of up to K events
    (oldest first, as the sampler returns them):

        x          = W_x event                                    [N, K, dim]
        f, v, c    = W_f x, W_v x, W_c x
        h          = gated_scan(f, v)       gate decays with the time between events
        y, n       = gated_norm(x, h, c)                 residual, then the next norm
        o          = cross_attention(W_q root, W_k n, W_v' n)   event ages by ``positions``
        _, out     = gated_norm(root, W_o o, W_g o)

    ``mean_gap``: the time that the decay rates start around (they are learned,
    one a channel, from 1/64 to 4 per mean gap). ``positions``: how the
    attention sees an event's age, "bias" (a learned bias by ``buckets`` of it)
    or "rotary" (queries and keys turned by it, the fastest pair one radian a
    mean gap)."""

    def __init__(self, dim: int, event_dim: int, heads: int = 2, buckets: int = 32, mean_gap: float = 1.0,
                 positions: str = "bias") -> None:
        super().__init__()
        if dim % heads:
            raise ValueError(f"history embedding: {dim} channels over {heads} heads")
        if positions not in ("bias", "rotary"):
            raise ValueError(f"history embedding: positions {positions!r}, expected 'bias' or 'rotary'")
        if positions == "rotary" and dim // heads < 2:
            raise ValueError("history embedding: rotary positions need heads of 2 channels or more")
        self.dim, self.event_dim, self.heads, self.positions = dim, event_dim, heads, positions
        self.per_gap = 1.0 / mean_gap if mean_gap > 0 else 1.0
        self.inp = nn.Linear(event_dim, dim)
        self.gates = nn.Linear(dim, 3 * dim)
        self.log_rate = nn.Parameter(torch.linspace(-6.0, 2.0, dim) * 0.6931471805599453)
        self.q = nn.Linear(dim, dim)
        self.kv = nn.Linear(dim, 2 * dim)
        if positions == "bias":
            self.age_bias = nn.Parameter(torch.zeros(heads, buckets))
        else:
            freqs = rotary.frequencies(dim // heads // 2 * 2, scaling="linear", factor=1.0 / self.per_gap, device="cpu")
            # (as integers: a module's casts leave their 64 bits alone)
            self.register_buffer("freq_bits", freqs.view(torch.int64), persistent=False)
        self.out = nn.Linear(dim, 2 * dim)
        self.norms = nn.ParameterDict({
            **{f"{at}_{w}_{k}": nn.Parameter((torch.ones if k == "w" else torch.zeros)(dim))
               for at in ("event", "root") for w in ("post", "pre") for k in ("w", "b")},
            **{f"{at}_scale": nn.Parameter(torch.ones(dim)) for at in ("event", "root")}})

    @property
    def freqs(self) -> torch.Tensor:
        """The rotary frequencies, float64 [pairs]."""
        return self.freq_bits.view(torch.float64)

    @freqs.setter
    def freqs(self, value: torch.Tensor) -> None:
        self.freq_bits = value.to(torch.float64).view(torch.int64)

    def _norm(self, at: str, x, z, gate):
        n = self.norms
        return history.gated_norm(x.contiguous(), z, gate, n[f"{at}_scale"], post_weight=n[f"{at}_post_w"],
                                  post_bias=n[f"{at}_post_b"], pre_weight=n[f"{at}_pre_w"],
                                  pre_bias=n[f"{at}_pre_b"])

    def forward(self, root: torch.Tensor, events: torch.Tensor, cnt: torch.Tensor, age: torch.Tensor) -> torch.Tensor:
        """``root`` [N, dim]; ``events`` [N, K, event_dim]; ``cnt`` int32 [N];
        ``age`` float32 [N, K]: the time from each event to the root's query
        (places past a count may hold anything finite)."""
        N, K, _ = events.shape
        D, H = self.dim, self.heads
        # times between a window's events: 0 before its first (nothing to decay)
        gaps = torch.zeros_like(age)
        if K > 1:
            gaps[:, 1:] = (age[:, :-1] - age[:, 1:]).clamp_min(0.0) * self.per_gap
        x = self.inp(events)
        f, v, c = self.gates(x).split(D, -1)
        h, _ = history.gated_scan(f, v, lens=cnt, gaps=gaps, decay=self.log_rate.exp())
        _, n = self._norm("event", x, h, c)
        k, w = self.kv(n).view(N, K, 2, H, D // H).unbind(2)
        q = self.q(root).view(N, 1, H, D // H)
        q_pos, k_pos = torch.zeros(N, 1, dtype=torch.int64, device=age.device), age.to(torch.int64).neg()
        if self.positions == "rotary":
            q, k = rotary.rotate(q, k, q_pos, k_pos, self.freqs)
            o = history.cross_attention(q, k, w, k_lens=cnt)
        else:
            o = history.cross_attention(q, k, w, k_lens=cnt, bias=self.age_bias, q_pos=q_pos, k_pos=k_pos)
        z, gate = self.out(o.reshape(N, D)).split(D, -1)
        return self._norm("root", root, z, gate)[1]
