"""What a call of the losses over all candidates allocates does not grow with
the table (a teacher's routing alone counts blocks of 32 candidates), by the C
entries that give the sizes; no GPU."""
import ctypes

import pytest

from starry_unigraph.lib import _capi


def _bytes(dtype, dim, n, v, k=1, teacher=0):
    a = ctypes.byref(_capi.Candidates(dtype, dim, n, v, 16, 16, dim, dim, None, 1.0, 1.0))
    lib = _capi.lib()
    return (lib.sgl_candidates_workspace_bytes(a, k, teacher, 3, 0),
            lib.sgl_candidates_workspace_bytes(a, k, teacher, 3, 1), lib.sgl_candidates_keep_bytes(a, k, teacher, 3))


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim", [8, 64, 100, 172, 256])
@pytest.mark.parametrize("n", [1, 600, 4000, 24000])
def test_labels(dtype, dim, n):
    size, wide = 4 if dtype == 0 else 2, (dim + 63) // 64 * 64
    large, larger = _bytes(dtype, dim, n, 1_140_149), _bytes(dtype, dim, n, 20_000_000)
    assert larger == large
    # the rows' images (a row, four numbers and padding, tiles of 64), and two pieces of 256 candidates for each of 256
    # workgroups (or of 128 for each of 512) in float32
    tiles = (n + 63) // 64
    assert large[1] <= tiles * 64 * ((wide + 16) * size + 16) + 2 * 256 * 256 * (wide + 4) * 4 + 4096
    # the forward's pieces: every row once, and one outer tile of 256 more for each workgroup, three numbers each
    assert large[0] <= ((n + 255) // 256 + 512) * 256 * (wide + 3) * 4 + 4096


@pytest.mark.parametrize("n, k", [(600, 20), (1200, 64)])
def test_teacher(n, k):
    large, larger = _bytes(1, 172, n, 1_140_149, k, 1), _bytes(1, 172, n, 20_000_000, k, 1)
    tiles, blocks = (n + 63) // 64, (20_000_000 - 1_140_149) / 32
    assert larger[0] == large[0] and larger[2] == large[2]
    assert larger[1] - large[1] <= tiles * (blocks + 1) * 4 + 4096
