"""A teacher that fails, or answers in another form, leaves the runtime as it
was: the steps behind it have the bits of a run without the failed one."""
import pytest
import torch

from test_gpu_next_node import _runtime, _teacher

pytestmark = pytest.mark.gpu


class _Lost(Exception):
    pass


def _raise(ids, logits):
    raise _Lost


BAD = {
    "raises": (_raise, _Lost),
    "one tensor": (lambda ids, logits: ids, Exception),
    "rows": (lambda ids, logits: (ids[:-1], logits[:-1]), ValueError),
    "shapes": (lambda ids, logits: (ids, logits[:, :-1]), ValueError),
    "no entries": (lambda ids, logits: (ids[:, :0], logits[:, :0]), ValueError),
    "one dimension": (lambda ids, logits: (ids[:, 0], logits[:, 0]), ValueError),
    "ids": (lambda ids, logits: (ids.float(), logits), ValueError),
    "logits": (lambda ids, logits: (ids, logits.half()), ValueError),
    "host": (lambda ids, logits: (ids.cpu(), logits.cpu()), ValueError),
    "gradient": (lambda ids, logits: (ids, logits.requires_grad_()), ValueError),
}


def _run(bad=None, at=2):
    rt = _runtime()
    good = _teacher(rt)
    batches = list(rt.iter_batches("train", 50))[200:206]
    rt.set_teacher(good)
    out = []
    for i, b in enumerate(batches):
        if bad is not None and i == at:
            make, error = bad
            rt.set_teacher(lambda batch: make(*good(batch)))
            with pytest.raises(error):
                rt.train_step(b)
            rt.set_teacher(good)
        out.append(rt.train_step(b)["loss"])
    val = next(iter(rt.iter_batches("val", 50)))
    return out, rt.eval_step(val, "val"), rt.optimizer.inner.flat.clone()


@pytest.fixture(scope="module")
def plain(gpu):
    return _run()


@pytest.mark.parametrize("what", BAD)
def test_a_failed_step_leaves_nothing(gpu, plain, what):
    got = _run(BAD[what])
    assert got[0] == plain[0]
    assert got[1]["loss"] == plain[1]["loss"] and got[1]["predictions"] == plain[1]["predictions"]
    assert torch.equal(got[2], plain[2])


def test_temperatures_that_the_step_refuses(gpu):
    rt = _runtime()
    for kw in (dict(temperature=1e-39), dict(temperature=1e20), dict(temperature=-1.0), dict(temperature=float("nan")),
               dict(temperature=torch.ones(()).requires_grad_()), dict(weight=torch.ones(()).requires_grad_())):
        with pytest.raises(ValueError, match="set_teacher"):
            rt.set_teacher(_teacher(rt), **kw)
    batch = list(rt.iter_batches("train", 50))[200]
    for T in (1e-30, 1e18):   # the ends of what is taken: the step takes them too
        rt.set_teacher(_teacher(rt), weight=0.0, temperature=T)
        rt.train_step(batch)
