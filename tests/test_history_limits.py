"""What the history operators' C entries refuse by size, without a GPU: problems
of more threads than a launch has (a sequence's data need not exist, the checks
come before any access)."""
import ctypes

import pytest

from starry_unigraph.lib import _capi


def _attention(n, lq, lk, heads_q, heads_kv, dh=8):
    a = _capi.Attention(1, heads_q, heads_kv, dh, n, lq, lk)
    for f in ("q", "k", "v"):
        setattr(a, f, 4096)
    a.scale = 1.0
    return a


def _refused(rc):
    return rc != 0 and b"too many" in _capi.lib().sgl_last_error()


@pytest.mark.parametrize("n, lq, lk, hq, hkv", [
    (1 << 25, 1, 10, 1, 1),       # one wave a sequence
    (1 << 21, 1, 10, 64, 16),
    (1 << 23, 33, 10, 1, 1),      # workgroups a sequence
    (1 << 23, 1, 65, 1, 1),
    (1 << 20, 700, 10, 4, 2),
    (2, 1 << 30, 10, 4, 2),
    (2, 1 << 30, 10, 128, 1),     # (and more query heads than a key head takes)
])
def test_attention_of_too_many_rows(n, lq, lk, hq, hkv):
    a = _attention(n, lq, lk, hq, hkv)
    lib = _capi.lib()
    rc = lib.sgl_cross_attention_forward(ctypes.byref(a), 4096, None, None, None, 0, None)
    assert rc != 0
    if hq // hkv <= 64:
        assert _refused(rc)
        assert _refused(lib.sgl_cross_attention_backward(ctypes.byref(a), 4096, 4096, 4096, 4096, 4096, 4096, 4096,
                                                         None, None, 0, None))


@pytest.mark.parametrize("N, D", [(1 << 25, 128), (1 << 22, 1 << 10), ((1 << 31) - 2, 3)])
def test_scan_of_too_many_sequences(N, D):
    rc = _capi.lib().sgl_gated_scan_forward(0, N, 1, D, 4096, D, D, 4096, D, D, None, None, None, 0, 0, None, 4096,
                                            None, None, None, 0, None)
    assert _refused(rc)
