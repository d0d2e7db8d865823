"""Rotary positions, attention over a window and losses over all candidates run
together: as ctdg.positions = rotary and ctdg.objective = next_node run them in
the runtime's step (loss and the gradients of every parameter against the same
modules in float64 on the CPU with the operators' definitions), and as one
captured step in 16 bits."""
import copy

import pytest
import torch
import torch.nn.functional as F

import history_oracle as ho
from test_gpu_history_embedding import _Oracle as _History


class _Rotary:
    @staticmethod
    def rotate(q, k, q_pos, k_pos, freqs):
        out = []
        for x, pos in ((q, q_pos), (k, k_pos)):
            P = freqs.shape[0]
            t = (pos.double()[..., None] * freqs)[:, :, None]
            a, b = x[..., :P], x[..., P:2 * P]
            out.append(torch.cat([a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos(), x[..., 2 * P:]], -1))
        return out


class _Attention(_History):
    @staticmethod
    def cross_attention(q, k, v, *, k_lens):
        q, k, v = (t.permute(0, 2, 1, 3) for t in (q, k, v))
        on = ho.live_rows(k_lens, k.shape[0], k.shape[2])[:, None, None]
        w = torch.softmax((q @ k.transpose(-1, -2) * q.shape[-1] ** -0.5).masked_fill(~on, -1e300), -1) * on
        return (w @ v).permute(0, 2, 1, 3)


class _Candidates:
    @staticmethod
    def cross_entropy(h, table, target, *, bias):
        s = torch.log_softmax(h @ table.t() + bias, -1)
        return torch.where(target >= 0, -s.gather(1, target.clamp_min(0)[:, None])[:, 0], 0.0)

    @staticmethod
    def distillation(h, table, ids, logits, *, bias, temperature):
        on = (ids >= 0) & (logits > -torch.inf)
        logq = torch.log_softmax(logits.double().div(temperature).masked_fill(~on, -1e300), -1)
        logp = torch.log_softmax((h @ table.t() + bias) / temperature, -1).gather(1, ids.clamp_min(0))
        return temperature ** 2 * torch.where(on, logq.exp() * (logq - logp), 0.0).sum(1)


def _runtime(seed=0, batch=50, **ctdg):
    from starry_unigraph import SchedulerSession, synth
    from starry_unigraph.data import from_stream
    cfg = {"model": {"family": "tgn", "hidden_dim": 36}, "data": {"name": "h", "format": "synthetic"},
           "train": {"batch_size": batch, "lr": 1e-3}, "runtime": {"device": "cuda"},
           "ctdg": {"mailbox_slots": 1, "num_head": 2, "embedding": "history", "positions": "rotary",
                    "objective": "next_node", **ctdg},
           "sampling": {"neighbor_limit": [7], "history": 1, "strategy": "recent"}}
    torch.manual_seed(seed)
    sess = SchedulerSession.from_config(cfg).with_events(from_stream(synth.bipartite_stream(seed=0)))
    sess.build_runtime()
    return sess.ctdg_session.online_runtime


def _teacher(rt, K=5):
    """Some nodes and logits an event, among them places without an entry, a
    node twice and nodes that are no candidate."""
    pool, nodes = rt.dataset.dst.unique(), rt.dataset.num_nodes

    def answer(batch):
        g = torch.Generator().manual_seed(batch.start)
        ids = pool[torch.randint(0, pool.numel(), (batch.size, K), generator=g)]
        ids[::3, 1] = ids[::3, 0]
        ids[1::4, 2] = -1
        ids[2::5, 3] = torch.randint(0, nodes, (len(ids[2::5]),), generator=g)
        return ids.to(rt.device), torch.randn(batch.size, K, generator=g).mul(2.0).to(rt.device)
    return answer


def test_options_are_checked():
    from starry_unigraph.backends.ctdg.runtime.models import build_ctdg_model
    from starry_unigraph.runtime.modules import CandidateHead, HistoryEncoder
    kw = dict(num_nodes=5, hidden_dim=8, edge_feat_dim=3)
    for bad in (dict(positions="rotary"), dict(objective="next_node"),
                dict(objective="next_node", embedding="time_projection")):
        with pytest.raises(ValueError, match="embedding = history"):
            build_ctdg_model("tgn", **bad, **kw)
    with pytest.raises(KeyError, match="next_node"):
        build_ctdg_model("tgn", embedding="history", objective="nodes", **kw)
    with pytest.raises(ValueError, match="rotary"):
        build_ctdg_model("tgn", embedding="history", positions="sine", **kw)
    with pytest.raises(ValueError, match="2 channels"):
        HistoryEncoder(2, 3, heads=2, positions="rotary")
    model = build_ctdg_model("tgn", embedding="history", positions="rotary", objective="next_node", **kw)
    assert model.head.table.shape == (5, 8) and not hasattr(model.history, "age_bias")
    assert "history.age_bias" in dict(build_ctdg_model("tgn", embedding="history", **kw).named_parameters())
    for nodes, match in (([], "at least one"), ([0, 5], "in \\[0, 5\\)"), ([-1], "in \\[0, 5\\)"), ([1, 1], "twice")):
        with pytest.raises(ValueError, match=match):
            CandidateHead(torch.tensor(nodes, dtype=torch.int64), 5, 8)
    with pytest.raises(ValueError, match="rows of 257"):
        CandidateHead(torch.arange(5), 5, 257)
    head = CandidateHead(torch.tensor([3, 1]), 5, 8)
    assert head.rows(torch.tensor([[0, 1, 2], [3, 4, 5], [-1, -7, 9]])).tolist() == [[-1, 1, -1], [0, -1, -1],
                                                                                    [-1, -1, -1]]


@pytest.mark.gpu
@pytest.mark.parametrize("taught", [False, True], ids=["labels", "teacher"])
@pytest.mark.parametrize("positions", ["rotary", "bias"])
def test_step_and_gradients_match_the_definitions(gpu, monkeypatch, taught, positions):
    from starry_unigraph.runtime.modules import candidates, history
    rt = _runtime(positions=positions)
    if taught:
        rt.set_teacher(_teacher(rt), weight=0.25, temperature=2.0)
    batches = list(rt.iter_batches("train", 50))
    for b in batches[300:303]:
        rt.train_step(b)
    with torch.no_grad():   # a table that is not zero, gates and norms that are not their first values
        g = torch.Generator().manual_seed(4)
        for p in rt.model.parameters():
            p.add_((torch.randn(p.shape, generator=g) * 0.1).to(p.device))
    model = copy.deepcopy(rt.model).cpu().double()
    out = rt.train_step(batches[303])
    grads = {n: p.grad.detach().cpu().clone() for n, p in rt.model.named_parameters()}
    b, d, n = rt.step.buf, rt.dims, batches[303].size
    U, K = int(b.num_roots), d.fanout
    cnt = b.hop.cnt[:U].cpu()
    events = b.X.view(-1, d.C)[:U * K].view(U, K, d.C)[..., :d.D + d.F].cpu().double()
    age = b.hop.dt[:U * K].view(U, K).cpu().double()
    live = ho.live_rows(cnt, U, K)
    events, age = torch.where(live[..., None], events, 0.0), torch.where(live, age, 0.0)
    monkeypatch.setattr(history, "history", _Attention if positions == "rotary" else _History)
    monkeypatch.setattr(history, "rotary", _Rotary)
    monkeypatch.setattr(candidates, "candidates", _Candidates)
    y = model.history(b.new_mem[:U].cpu().double(), events, cnt, age)
    lo = batches[303].start
    dst = rt.dataset.dst[lo:lo + n]
    src = y[b.ridx_src[:n].cpu().long()]
    h = model.src_fc(src)
    loss = model.head.loss(h, dst).mean()
    if taught:
        ids, logits = (t.cpu() for t in _teacher(rt)(batches[303]))
        loss = 0.75 * loss + 0.25 * model.head.distill(h, ids, logits, 2.0).mean()
    loss.backward()
    assert abs(out["loss"] - float(loss.detach())) < 1e-5
    want = model.head(h, dst)
    assert torch.allclose(b.pos[:n].cpu().double(), want, rtol=1e-4, atol=1e-5)
    for name, p in model.named_parameters():
        # float32 products of a few hundred terms each: 1e-4 of the largest entry
        err = (grads[name].double() - p.grad).abs().max()
        assert err <= 1e-4 * p.grad.abs().max() + 1e-9, (name, float(err), float(p.grad.abs().max()))


@pytest.mark.gpu
def test_steps_repeat_and_eval_leaves_the_parameters(gpu):
    runs = []
    for _ in range(2):
        rt = _runtime()
        rt.set_teacher(_teacher(rt))
        losses = [rt.train_step(b)["loss"] for b in list(rt.iter_batches("train", 50))[200:206]]
        assert all(torch.isfinite(torch.tensor(losses)))
        before = rt.optimizer.inner.flat.clone()
        val = next(iter(rt.iter_batches("val", 50)))
        out = rt.eval_step(val, "val")
        assert len(out["predictions"]) == val.size and 0.0 <= out["meta"]["metrics"]["ap"] <= 1.0
        assert torch.equal(before, rt.optimizer.inner.flat)
        runs.append((losses, before))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1])


@pytest.mark.gpu
def test_teacher_is_refused_without_the_objective(gpu):
    rt = _runtime(objective="link")
    with pytest.raises(ValueError, match="next_node"):
        rt.set_teacher(lambda batch: None)
    rt = _runtime()
    for kw in (dict(weight=1.5), dict(weight=float("nan")), dict(temperature=0.0), dict(temperature=float("inf"))):
        with pytest.raises(ValueError, match="set_teacher"):
            rt.set_teacher(lambda batch: None, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_captured_step_of_the_operators_together(gpu, dtype):
    """Rotated queries and keys, the attention of one new event over its window,
    both losses and every gradient, captured once and replayed on other inputs
    between eager steps: the eager step's bits each time."""
    from starry_unigraph.native import candidates, history, rotary
    N, L, H, dh, V, K = 70, 11, 2, 20, 700, 6
    dev, g = gpu, torch.Generator().manual_seed(0)
    freqs = rotary.frequencies(16, base=500.0, device=dev)

    def draw():
        x = dict(q=torch.randn(N, 1, H, dh, generator=g), k=torch.randn(N, L, H, dh, generator=g),
                 v=torch.randn(N, L, H, dh, generator=g), w=torch.randn(V, H * dh, generator=g) * 0.3)
        pos = torch.randint(0, 2000, (N, L), generator=g).sort(1)[0]
        rest = dict(b=torch.randn(V, generator=g), pos=pos, at=pos[:, -1:] + 5,
                    lens=torch.randint(0, L + 1, (N,), generator=g, dtype=torch.int32),
                    target=torch.randint(-1, V, (N,), generator=g), ids=torch.randint(-1, V, (N, K), generator=g),
                    z=torch.randn(N, K, generator=g))
        return {n: t.to(dev, dtype) for n, t in x.items()}, {n: t.to(dev) for n, t in rest.items()}

    def step(x, r):
        x = {n: t.detach().requires_grad_() for n, t in x.items()}
        b = r["b"].detach().requires_grad_()
        q, k = rotary.rotate(x["q"], x["k"], r["at"], r["pos"], freqs)
        h = history.cross_attention(q, k, x["v"], k_lens=r["lens"]).reshape(N, H * dh)
        ce = candidates.cross_entropy(h, x["w"], r["target"], bias=b)
        kl = candidates.distillation(h, x["w"], r["ids"], r["z"], bias=b, temperature=1.5)
        return (ce, kl, *torch.autograd.grad((ce, kl), (*x.values(), b), (torch.ones_like(ce), torch.ones_like(kl))))

    x, r = draw()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x, r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, r)
    for _ in range(4):
        nx, nr = draw()
        for into, new in ((x, nx), (r, nr)):
            for n in into:
                into[n].copy_(new[n])
        want = step(nx, nr)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, want):
            assert torch.equal(a, e)
            assert bool(torch.isfinite(a).all())
