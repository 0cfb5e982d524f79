"""What ``embedding``, ``gated_mlp`` and ``orthogonalize_tensors`` refuse, on the host, before any launch (CPU tensors)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gptrig import _lib
from gptrig.nn import embedding

BF16, F32 = torch.bfloat16, torch.float32


def test_embedding_refusals():
    tokens, table = torch.zeros(3, dtype=torch.int32), torch.zeros((5, 8))
    for bad in (tokens.float(), tokens.short(), tokens.bool()):
        with pytest.raises(TypeError, match="int32 or int64"):
            embedding(bad, table)
    for bad in (table.half(), table.double(), table.int()):
        with pytest.raises(TypeError, match="bfloat16 or float32"):
            embedding(tokens, bad)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        embedding(tokens, table, dtype=torch.float16)
    for bad in (table[0], table[None], table[:0], table[:, :0]):
        with pytest.raises(ValueError, match="vocab, width"):
            embedding(tokens, bad)
    for bad in (float("nan"), float("inf"), 3.5e38, -1e300):
        with pytest.raises(ValueError, match="scale"):
            embedding(tokens, table, scale=bad)
    with pytest.raises(RuntimeError, match="GPU"):
        embedding(tokens, table)


def test_embedding_entry_points_check_their_arguments():
    lib = _lib.lib()
    at, odd = ctypes.c_void_p(1 << 12), ctypes.c_void_p((1 << 12) + 2)
    one = ctypes.c_float(1.0)
    fwd = lib.gptrig_scaled_embedding_fwd
    assert fwd(None, 0, at, 8, 1, at, 0, 3, 8, 5, one, None) == -1
    assert fwd(at, 0, at, 8, 2, at, 0, 3, 8, 5, one, None) == -3
    assert fwd(at, 0, at, 8, 1, at, -1, 3, 8, 5, one, None) == -3
    assert fwd(at, 0, at, -8, 1, at, 0, 3, 8, 5, one, None) == -2
    assert fwd(at, 0, at, 8, 1, at, 0, 2 ** 31, 8, 5, one, None) == -2
    assert fwd(at, 0, at, 8, 1, at, 0, 3, 0, 5, one, None) == -2
    assert fwd(at, 0, at, 8, 1, at, 0, 3, 8, 0, one, None) == -2
    assert fwd(odd, 0, at, 8, 1, at, 0, 3, 8, 5, one, None) == -2
    assert fwd(at, 0, odd, 8, 1, at, 0, 3, 8, 5, one, None) == -2
    assert fwd(at, 0, at, 8, 1, at, 0, 0, 8, 5, one, None) == 0
    bwd, size = lib.gptrig_scaled_embedding_bwd, _lib.query("gptrig_scaled_embedding_bwd_workspace_bytes", 3, 8, 5)
    assert size > 0
    assert bwd(at, 0, at, 8, 0, None, 1, 3, 8, 5, one, at, size, None) == -1
    assert bwd(at, 0, at, 8, 0, at, 1, 3, 8, 5, one, None, size, None) == -1
    assert bwd(at, 0, at, 8, 0, at, 1, 3, 8, 5, one, at, size - 1, None) == -6
    assert bwd(at, 0, at, 8, 0, odd, 1, 3, 8, 5, one, at, size, None) == -2
    assert bwd(at, 0, at, 8, 5, at, 1, 3, 8, 5, one, at, size, None) == -3


@pytest.mark.parametrize("n", [1, 1000, 8192, 8193, 65536, 131072, 10 ** 6, 2 ** 31 - 65537])
def test_embedding_workspace(n):
    """Two buffers of pairs, the histograms of at most 256 blocks, two partial rows a chunk of four pairs or more."""

    size = _lib.query("gptrig_scaled_embedding_bwd_workspace_bytes", n, 16, 1000)
    chunks = [-(-n // c) for c in (4, 32)]
    assert 16 * n + 128 * chunks[1] <= size <= 16 * n + 128 * chunks[0] + 256 * 1024 + 6 * 256
