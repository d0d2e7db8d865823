"""ctdg.embedding = history: the runtime's step with the windows read as
sequences. The step's loss and the gradients of every parameter against the
same modules in float64 on the CPU with the operators' definitions; eval,
repeatability and a short epoch."""
import copy

import pytest
import torch
import torch.nn.functional as F

import history_oracle as ho

FP32 = torch.float32


class _Oracle:
    """native.history's operators by their definitions (float64, differentiable)."""

    @staticmethod
    def gated_scan(f, v, *, lens, gaps, decay):
        return ho.scan(f, v, lens, None, gaps, decay)

    @staticmethod
    def gated_norm(x, z, g, scale, *, post_weight, post_bias, pre_weight, pre_bias):
        return ho.norm(x, z, g, scale, post_weight, pre_weight, post_bias, pre_bias)

    @staticmethod
    def cross_attention(q, k, v, *, k_lens, bias, q_pos, k_pos):
        q, k, v = (t.permute(0, 2, 1, 3) for t in (q, k, v))
        s = q @ k.transpose(-1, -2) * q.shape[-1] ** -0.5
        s = s + bias[:, ho.columns(q_pos, k_pos, bias.shape[1], 0, False)].permute(1, 0, 2, 3)
        on = ho.live_rows(k_lens, k.shape[0], k.shape[2])[:, None, None]
        w = torch.softmax(s.masked_fill(~on, -1e300), -1) * on
        return (w @ v).permute(0, 2, 1, 3)


def _runtime(seed=0, batch=50):
    from starry_unigraph import SchedulerSession, synth
    from starry_unigraph.data import from_stream
    cfg = {"model": {"family": "tgn", "hidden_dim": 36}, "data": {"name": "h", "format": "synthetic"},
           "train": {"batch_size": batch, "lr": 1e-3}, "runtime": {"device": "cuda"},
           "ctdg": {"mailbox_slots": 1, "num_head": 2, "embedding": "history"},
           "sampling": {"neighbor_limit": [7], "history": 1, "strategy": "recent"}}
    torch.manual_seed(seed)
    sess = SchedulerSession.from_config(cfg).with_events(from_stream(synth.bipartite_stream(seed=0)))
    sess.build_runtime()
    return sess.ctdg_session.online_runtime


def test_unknown_and_unsupported_embeddings_are_refused():
    from starry_unigraph.backends.ctdg.runtime.models import build_ctdg_model
    kw = dict(num_nodes=5, hidden_dim=8, edge_feat_dim=3)
    with pytest.raises(KeyError, match="history"):
        build_ctdg_model("tgn", embedding="sequence", **kw)
    with pytest.raises(ValueError, match="fp32"):
        build_ctdg_model("tgn", embedding="history", attention_gemm_dtype="bf16", **kw)
    with pytest.raises(ValueError, match="heads"):
        build_ctdg_model("tgn", embedding="history", num_head=3, **kw)
    assert build_ctdg_model("tgn", embedding="history", **kw).conv is None


@pytest.mark.gpu
def test_step_and_gradients_match_the_definitions(gpu, monkeypatch):
    from starry_unigraph.runtime.modules import history as module
    rt = _runtime()
    batches = list(rt.iter_batches("train", 50))
    for b in batches[300:303]:
        rt.train_step(b)
    with torch.no_grad():   # a table that is not zero, gates and norms that are not their first values
        g = torch.Generator().manual_seed(4)
        for p in rt.model.history.parameters():
            p.add_((torch.randn(p.shape, generator=g) * 0.1).to(p.device))
    model = copy.deepcopy(rt.model).cpu().double()
    out = rt.train_step(batches[303])
    grads = {n: p.grad.detach().cpu().clone() for n, p in rt.model.named_parameters()}
    b, d, n = rt.step.buf, rt.dims, batches[303].size
    U, K = int(b.num_roots), d.fanout
    cnt = b.hop.cnt[:U].cpu()
    assert int(cnt.max()) == K and int(cnt.min()) < K   # ragged windows
    events = b.X.view(-1, d.C)[:U * K].view(U, K, d.C)[..., :d.D + d.F].cpu().double()
    age = b.hop.dt[:U * K].view(U, K).cpu().double()
    live = ho.live_rows(cnt, U, K)
    events, age = torch.where(live[..., None], events, 0.0), torch.where(live, age, 0.0)
    monkeypatch.setattr(module, "history", _Oracle)
    y = model.history(b.new_mem[:U].cpu().double(), events, cnt, age)
    y = F.pad(y, (0, 0, 0, 1))
    rows = [r[:n].cpu().long() for r in (b.ridx_src, b.ridx_dst, b.ridx_neg)]
    want = model(*[y[r] for r in rows])
    loss = (F.binary_cross_entropy_with_logits(want.pos_logits, torch.ones_like(want.pos_logits))
            + F.binary_cross_entropy_with_logits(want.neg_logits, torch.zeros_like(want.neg_logits)))
    loss.backward()
    assert abs(out["loss"] - float(loss)) < 1e-5
    assert torch.allclose(b.pos[:n].cpu().double(), want.pos_logits, rtol=1e-4, atol=1e-5)
    for name, p in model.named_parameters():
        # float32 products of a few hundred terms each: 1e-4 of the largest entry
        err = (grads[name].double() - p.grad).abs().max()
        assert err <= 1e-4 * p.grad.abs().max() + 1e-9, (name, float(err), float(p.grad.abs().max()))


@pytest.mark.gpu
def test_steps_repeat_and_eval_leaves_the_parameters(gpu):
    runs = []
    for _ in range(2):
        rt = _runtime()
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
def test_first_events_have_empty_windows(gpu):
    rt = _runtime()
    for b in list(rt.iter_batches("train", 50))[:2]:   # no history yet
        assert torch.isfinite(torch.tensor(rt.train_step(b)["loss"]))
    assert bool(torch.isfinite(rt.optimizer.inner.flat).all())
