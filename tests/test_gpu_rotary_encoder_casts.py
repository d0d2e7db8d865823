"""The history embedding with rotary positions keeps its frequencies' 64 bits
when the module is cast, moved or copied."""
import copy

import pytest
import torch

from starry_unigraph.native import rotary
from starry_unigraph.runtime.modules import HistoryEncoder

CASTS = {"float": lambda m: m.float(), "half": lambda m: m.half(), "bfloat16": lambda m: m.bfloat16(),
         "double": lambda m: m.double(), "to": lambda m: m.to("cpu", torch.float32), "copy": copy.deepcopy}


@pytest.mark.parametrize("cast", CASTS)
def test_frequencies_keep_their_type(cast):
    m = HistoryEncoder(8, 5, heads=2, mean_gap=30.0, positions="rotary")
    want = rotary.frequencies(4, scaling="linear", factor=30.0, device="cpu")
    m = CASTS[cast](m)
    assert m.freqs.dtype == torch.float64 and torch.equal(m.freqs, want)
    assert not any("freq" in k for k in m.state_dict())
    m.freqs = want * 0.1 + 0.3
    assert torch.equal(CASTS[cast](m).freqs, want * 0.1 + 0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("positions", ["rotary", "bias"])
def test_a_cast_module_runs(gpu, positions):
    torch.manual_seed(0)
    m = HistoryEncoder(8, 5, heads=2, mean_gap=30.0, positions=positions).to(gpu)
    g = torch.Generator().manual_seed(0)
    args = [torch.randn(6, 8, generator=g).to(gpu), torch.randn(6, 7, 5, generator=g).to(gpu),
            torch.tensor([0, 1, 7, 3, 2, 7], dtype=torch.int32, device=gpu),
            torch.rand(6, 7, generator=g).mul(90.0).sort(1, descending=True)[0].to(gpu)]
    want = m(*args)
    for moved in (m.float(), copy.deepcopy(m).cpu().float().to(gpu), m.to(torch.float32)):
        got = moved(*args)
        assert torch.equal(got, want)
        got.sum().backward()
