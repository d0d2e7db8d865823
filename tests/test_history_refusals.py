"""What the history operators refuse, without a GPU: their checks come before
any launch (tensors here live on the meta device or the CPU)."""
import ctypes

import pytest
import torch

from starry_unigraph.lib import _capi
from starry_unigraph.native import history


@pytest.fixture
def anywhere(monkeypatch):
    """The operators' argument checks on CPU tensors."""
    monkeypatch.setattr(_capi, "require_gpu", lambda device=None: torch.device("cpu"))


def _f(*s, dtype=torch.float32):
    return torch.zeros(*s, dtype=dtype)


def test_cpu_tensors_are_refused():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        history.gated_scan(_f(1, 2, 3), _f(1, 2, 3))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        history.cross_attention(_f(1, 2, 3, 4), _f(1, 2, 3, 4), _f(1, 2, 3, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        history.gated_norm(_f(2, 3), _f(2, 3), _f(2, 3), _f(3), post_weight=_f(3), pre_weight=_f(3))


@pytest.mark.parametrize("kw, match", [
    (dict(gate=_f(2, 3)), "gate: 2 dimensions"),
    (dict(gate=_f(2, 3, 4, dtype=torch.float64)), "gate: torch.float64"),
    (dict(value=_f(2, 3, 5)), "value: shape"),
    (dict(value=_f(2, 3, 4, dtype=torch.bfloat16)), "value: torch.bfloat16"),
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "lens: torch.int64"),
    (dict(lens=torch.zeros(3, dtype=torch.int32)), "lens: shape"),
    (dict(state=_f(2, 4, dtype=torch.bfloat16)), "state: torch.bfloat16"),
    (dict(gaps=_f(2, 3)), "both or neither"),
    (dict(decay=_f(4)), "both or neither"),
    (dict(gaps=_f(2, 4), decay=_f(4)), "gaps: shape"),
    (dict(gaps=_f(2, 3).requires_grad_(), decay=_f(4)), "gaps: has no gradient"),
    (dict(gate=_f(2, 3, 0), value=_f(2, 3, 0)), "no channels"),
])
def test_scan_refusals(anywhere, kw, match):
    args = dict(gate=_f(2, 3, 4), value=_f(2, 3, 4))
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        history.gated_scan(args.pop("gate"), args.pop("value"), **args)


@pytest.mark.parametrize("kw, match", [
    (dict(q=_f(2, 3, 4)), "q: 3 dimensions"),
    (dict(k=_f(2, 5, 8)), "k: 3 dimensions"),
    (dict(k=_f(2, 5, 3, 8), v=_f(2, 5, 3, 8)), "4 heads over 3"),
    (dict(k=_f(3, 5, 2, 8)), "k: shape"),
    (dict(v=_f(2, 6, 2, 8)), "v: shape"),
    (dict(v=_f(2, 5, 2, 8, dtype=torch.float16)), "v: torch.float16"),
    (dict(q=_f(2, 3, 4, 129), k=_f(2, 5, 2, 129), v=_f(2, 5, 2, 129)), "heads of 129"),
    (dict(q_lens=torch.zeros(2)), "q_lens: torch.float32"),
    (dict(key_mask=_f(2, 5)), "key_mask: torch.float32"),
    (dict(bias=_f(4, 8)), "needs q_pos"),
    (dict(bias=_f(4, 65), pos=True), "at most 64"),
    (dict(bias=_f(4, 7), pos=True, two_sided=True), "even number"),
    (dict(bias=_f(3, 8), pos=True), "bias: shape"),
    (dict(bias=_f(4, 8), pos=True, resolution=5), "resolution: 5"),
    (dict(bias=_f(4, 8), q_pos=_f(2, 3), k_pos=_f(2, 5)), "q_pos: torch.float32"),
    (dict(scale=float("nan")), "scale"),
])
def test_attention_refusals(anywhere, kw, match):
    args = dict(q=_f(2, 3, 4, 8), k=_f(2, 5, 2, 8), v=_f(2, 5, 2, 8))
    args.update(kw)
    if args.pop("pos", False):
        args.update(q_pos=torch.zeros(2, 3, dtype=torch.int64), k_pos=torch.zeros(2, 5, dtype=torch.int64))
    with pytest.raises(ValueError, match=match):
        history.cross_attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)


@pytest.mark.parametrize("kw, match", [
    (dict(x=_f(2, 8193), z=_f(2, 8193), gate=_f(2, 8193)), "rows of 8193"),
    (dict(z=_f(3, 4)), "z: shape"),
    (dict(gate=_f(2, 4, dtype=torch.float16)), "gate: torch.float16"),
    (dict(scale=_f(4, dtype=torch.bfloat16)), "scale: torch.bfloat16"),
    (dict(pre_weight=_f(5)), "pre_weight: shape"),
    (dict(post_bias=_f(4)), "both or neither"),
])
def test_norm_refusals(anywhere, kw, match):
    args = dict(x=_f(2, 4), z=_f(2, 4), gate=_f(2, 4), scale=_f(4), post_weight=_f(4), pre_weight=_f(4))
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        history.gated_norm(*[args.pop(k) for k in ("x", "z", "gate", "scale")], **args)


def test_c_entries_refuse_bad_arguments():
    L = _capi.load_library()
    err = lambda: L.sgl_last_error().decode()
    one = ctypes.c_void_p(256)   # (never read: the checks come first)
    scan = lambda dt, n, l, d, gaps=None, decay=None, ws=0: L.sgl_gated_scan_forward(
        dt, n, l, d, one, 1, 1, one, 1, 1, None, None, gaps, 0, 0, decay, one, None, None, None, ws, None)
    assert scan(3, 1, 1, 1) == 1 and "element type" in err()
    assert scan(0, 1, 1, 0) == 1 and "sizes" in err()
    assert scan(0, 1, 1, 4, gaps=one) == 1 and "both" in err()
    assert scan(0, 1, 100000, 4) == 3 and "workspace" in err()
    p = _capi.Attention(dtype=0, heads_q=4, heads_kv=3, head_dim=8, n=1, lq=1, lk=1)
    fwd = lambda: L.sgl_cross_attention_forward(ctypes.byref(p), one, None, None, None, 0, None)
    assert fwd() == 1 and "heads" in err()
    p.heads_kv, p.head_dim = 2, 200
    assert fwd() == 1 and "head size" in err()
    p.head_dim, p.q, p.k, p.v = 8, 256, 256, 256
    p.bias, p.buckets = 256, 65
    assert fwd() == 1 and "65 buckets" in err()
    p.buckets = 8
    assert fwd() == 1 and "positions" in err()
    p.q_pos = p.k_pos = 256
    back = lambda rest: L.sgl_cross_attention_backward(ctypes.byref(p), one, rest, one, one, one, one, one, one, None,
                                                       0, None)
    assert back(None) == 3 and "workspace" in err()
    p.dtype, p.lk = 1, 100
    assert L.sgl_cross_attention_saves(ctypes.byref(p)) == 3
    assert back(None) == 1 and "rest" in err()
    assert back(one) == 3 and "workspace" in err()
    norm = lambda dt, r, d, n=3: L.sgl_gated_norm_backward(
        dt, r, d, one, 1, one, 1, one, 1, one, None, None, None, None, 1e-5, 0, None, None, one, one, one, one, n,
        None, 0, None)
    assert norm(0, 1, 9000) == 1 and "9000" in err()
    assert norm(0, 1, 8, 4) == 1 and "3 or 5" in err()
    assert norm(0, 1, 8) == 3 and "workspace" in err()


def test_attention_struct_layout_matches_header(tmp_path):
    """ctypes' Attention has the size and field offsets of struct sgl_attention."""
    import os
    import subprocess
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [f for f, _ in _capi.Attention._fields_]
    src = tmp_path / "layout.cpp"
    src.write_text(
        '#include <cstdio>\n#include <cstddef>\n#include "starrygl_mi355x.h"\nint main() {\n'
        '  printf("%zu %d %d %d", sizeof(sgl_attention), SGL_FP32, SGL_BF16, SGL_FP16);\n'
        + "".join(f'  printf(" %zu", offsetof(sgl_attention, {f}));\n' for f in fields) + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I" + os.path.join(repo, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    types = [_capi.DTYPES[t] for t in (torch.float32, torch.bfloat16, torch.float16)]
    want = [ctypes.sizeof(_capi.Attention), *types] + [getattr(_capi.Attention, f).offset for f in fields]
    assert got == want
