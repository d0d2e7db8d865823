"""A candidate head's state names the nodes that its rows are of."""
import pytest
import torch

from starry_unigraph.runtime.modules import CandidateHead


def _head(ids, seed=0):
    torch.manual_seed(seed)
    return torch.nn.ModuleDict({"head": CandidateHead(torch.tensor(ids), 9, 4)})


def test_other_nodes_are_refused():
    a, b, c = _head([1, 5, 7]), _head([1, 5, 8], 1), _head([5, 1, 7], 2)
    state = a.state_dict()
    assert state["head.nodes"].tolist() == [1, 5, 7]
    for other in (b, c):   # as many candidates; the same ones in another order
        before = [p.clone() for p in other.parameters()]
        with pytest.raises(RuntimeError, match="of other nodes"):
            other.load_state_dict(state)
        assert all(torch.equal(x, y) for x, y in zip(before, other.parameters()))
        assert other["head"].rows(torch.tensor([5])).tolist() == [1 if other is b else 0]
    with pytest.raises(RuntimeError, match="size mismatch"):
        _head([1, 5]).load_state_dict(state)
    same = _head([1, 5, 7], 3)
    same.load_state_dict(state)
    assert torch.equal(same["head"].table, a["head"].table)
    # one of before the ids were kept
    del state["head.nodes"]
    same = _head([1, 5, 7], 4)
    assert same.load_state_dict(state).missing_keys == []
    assert torch.equal(same["head"].table, a["head"].table) and "head.nodes" not in state
    with pytest.raises(RuntimeError, match="Missing key"):
        same.load_state_dict({})


@pytest.mark.gpu
def test_checkpoints(gpu, tmp_path):
    from starry_unigraph import SchedulerSession, synth
    from starry_unigraph.data import from_stream

    def session(shift, seed):
        cfg = {"model": {"family": "tgn", "hidden_dim": 36}, "data": {"name": "h", "format": "synthetic"},
               "train": {"batch_size": 50, "lr": 1e-3}, "runtime": {"device": "cuda"},
               "ctdg": {"mailbox_slots": 1, "num_head": 2, "embedding": "history", "objective": "next_node"},
               "sampling": {"neighbor_limit": [7], "history": 1, "strategy": "recent"}}
        torch.manual_seed(seed)
        stream = synth.bipartite_stream(seed=0)
        if shift:   # as many destinations: the last one is another node
            stream.dst[stream.dst == stream.dst.max()] = int(stream.src.min())
        s = SchedulerSession.from_config(cfg).with_events(from_stream(stream))
        s.build_runtime()
        return s.ctdg_session

    a, b, c = session(False, 0), session(False, 1), session(True, 2)
    path = tmp_path / "a.pt"
    a.save_checkpoint(path)
    b.load_checkpoint(path)
    for x, y in zip(a.online_runtime.model.parameters(), b.online_runtime.model.parameters()):
        assert torch.equal(x, y)
    assert c.online_runtime.model.head.table.shape == a.online_runtime.model.head.table.shape
    before = c.online_runtime.optimizer.inner.flat.clone()
    with pytest.raises(RuntimeError, match="of other nodes"):
        c.load_checkpoint(path)
    assert torch.equal(before, c.online_runtime.optimizer.inner.flat)
    old = torch.load(path, weights_only=True)   # one of before the ids were kept
    del old["model"]["head.nodes"]
    torch.save(old, path)
    b = session(False, 3)
    b.load_checkpoint(path)
    for x, y in zip(a.online_runtime.model.parameters(), b.online_runtime.model.parameters()):
        assert torch.equal(x, y)
    b.online_runtime.train_step(next(iter(b.online_runtime.iter_batches("train", 50))))
