"""Which node comes next, out of all candidates: a learned row and bias a
candidate, and the losses of rows over all of them (native.candidates'
operators). The reference has no such head: it scores an event against one
drawn negative (backends/ctdg/runtime/models.py:313-324, runtime.py:124-136)."""
from __future__ import annotations

import torch
import torch.nn as nn

from starry_unigraph.native import candidates


class CandidateHead(nn.Module):
    """Scores ``<h, table_v> + bias_v`` of rows ``h`` [N, dim] over ``nodes``,
    the node ids (distinct, each in [0, num_nodes)) that may come next. Row i of
    the table is of ``nodes[i]``: the ids are kept in the state, and a state of
    other ids is refused (one of before they were kept is taken as of these)."""

    def __init__(self, nodes: torch.Tensor, num_nodes: int, dim: int) -> None:
        super().__init__()
        nodes = nodes.to(torch.int64).reshape(-1)
        if not 1 <= dim <= candidates.MAX_DIM:
            raise ValueError(f"candidate head: rows of {dim}, expected 1 to {candidates.MAX_DIM}")
        if nodes.numel() == 0 or int(nodes.min()) < 0 or int(nodes.max()) >= num_nodes:
            raise ValueError(f"candidate head: expected node ids in [0, {num_nodes}), at least one")
        rows = torch.full((num_nodes,), -1, dtype=torch.int64)
        rows[nodes.cpu()] = torch.arange(nodes.numel())
        if int((rows >= 0).sum()) != nodes.numel():
            raise ValueError("candidate head: a node id given twice")
        self.table = nn.Parameter(torch.randn(nodes.numel(), dim) * dim ** -0.5)
        self.bias = nn.Parameter(torch.zeros(nodes.numel()))
        self.register_buffer("nodes", nodes.clone())
        self.register_buffer("row_of", rows, persistent=False)

    def match_nodes(self, state: dict, prefix: str) -> str | None:
        """What is wrong with the node ids in a state that is to be loaded
        (None: nothing; ids that it lacks are added to it)."""
        ids = state.setdefault(prefix + "nodes", self.nodes)
        if ids.shape == self.nodes.shape and not torch.equal(ids.to(self.nodes.device), self.nodes):
            return f"{prefix}nodes: the table's rows are of other nodes."
        return None

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        wrong = self.match_nodes(state_dict, prefix)
        if wrong is not None:
            error_msgs.append(wrong)
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                                      error_msgs)

    def rows(self, ids: torch.Tensor) -> torch.Tensor:
        """The table's rows of node ids; -1 for those that are no candidate."""
        last = self.row_of.shape[0] - 1
        return torch.where((ids >= 0) & (ids <= last), self.row_of[ids.clamp(0, last)], -1)

    def forward(self, h: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
        """The scores [N] of one node a row; -inf where it is no candidate."""
        r = self.rows(ids)
        at = r.clamp_min(0)
        return torch.where(r >= 0, (h * self.table[at]).sum(-1) + self.bias[at], -torch.inf)

    def loss(self, h: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
        """The cross entropy [N] of the nodes that came (0 where one is no candidate)."""
        return candidates.cross_entropy(h, self.table, self.rows(ids), bias=self.bias)

    def distill(self, h: torch.Tensor, ids: torch.Tensor, logits: torch.Tensor,
                temperature: float = 1.0) -> torch.Tensor:
        """The divergence [N] from a teacher's top nodes ``ids`` [N, K] and their
        ``logits`` (those that are no candidates are left out)."""
        return candidates.distillation(h, self.table, self.rows(ids), logits, bias=self.bias, temperature=temperature)
