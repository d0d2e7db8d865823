"""The next-node objective's answers for the drawn negatives: the head's scores
of the ids that were drawn, whether or not they are roots of the batch, and the
metrics over them."""
import pytest
import torch

from test_gpu_next_node import _runtime

pytestmark = pytest.mark.gpu


def _ap(pos, neg):
    """Average precision of scores from its definition: over the thresholds in
    falling order, precision times the recall gained."""
    s = torch.cat([pos, neg])
    y = torch.cat([torch.ones_like(pos), torch.zeros_like(neg)])
    ap = hits = seen = 0.0
    for t in s.unique().flip(0):
        on = s == t
        gained = float(y[on].sum())
        hits, seen = hits + gained, seen + float(on.sum())
        ap += gained / len(pos) * hits / seen
    return ap


@pytest.mark.parametrize("mode", ["train", "eval", "predict"])
@pytest.mark.parametrize("ahead", [True, False], ids=["whole stream", "batch"])
def test_scores_of_the_drawn_nodes(gpu, mode, ahead):
    rt = _runtime()
    if not ahead:
        rt.neg_chunk = 1
    split = {"train": "train", "eval": "val", "predict": "test"}[mode]
    for b in list(rt.iter_batches("train", 50))[100:140]:
        rt.train_step(b)
    batch = next(iter(rt.iter_batches(split, 50)))
    drawn, serve = {}, rt._negatives_at

    def keep(b):
        buf, off = serve(b)
        drawn["ids"] = (buf[off:off + b.size] if off >= 0 else buf).clone()
        return buf, off
    rt._negatives_at = keep
    src_of, weights = {}, [p.detach().clone() for p in rt.model.parameters()]
    roots = rt._core().roots

    def encode(step, dims):
        y = roots(step, dims)
        src_of["h"] = y[step.buf.ridx_src[:batch.size]].detach().clone()
        return y
    rt._core().roots = encode
    out = {"train": rt.train_step, "eval": lambda b: rt.eval_step(b, split), "predict": rt.predict_step}[mode](batch)
    b, n = rt.step.buf, batch.size
    neg = drawn["ids"]
    assert int(((b.ridx_neg[:n] < 0) & (neg >= 0)).sum()) > n // 2   # (most of them are no root of the batch)
    with torch.no_grad():
        for p, w in zip(rt.model.parameters(), weights):
            p.copy_(w)   # (those the step began with)
        h = rt.model.src_fc(src_of["h"])
        head = rt.model.head
        r = head.rows(neg)
        assert bool((r >= 0).all())
        want = (h.double() * head.table.double()[r]).sum(-1) + head.bias.double()[r]
        size = (h.double() * head.table.double()[r]).abs().sum(-1) + head.bias.double()[r].abs()
    got = b.neg[:n].double()
    # a product of 36 terms and a sum in float32, half a step of 2^-24 each
    assert bool(((got - want).abs() <= (36 + 4) * 2.0 ** -24 * size).all())
    ap = _ap(b.pos[:n].sigmoid().double().cpu(), b.neg[:n].sigmoid().double().cpu())
    assert abs(out["meta"]["metrics"]["ap"] - ap) < 1e-6
