"""What ``embedding``, ``gated_mlp`` and ``orthogonalize_tensors`` refuse, on the host, before any launch (CPU tensors)."""

from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from gptrig import _lib
from gptrig.nn import embedding, gated_mlp
from gptrig.optim import orthogonalize_tensors

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
    """Two buffers of pairs, the histograms of at most 256 blocks, two partial rows a chunk of four pairs or more, and
    its number."""

    size = _lib.query("gptrig_scaled_embedding_bwd_workspace_bytes", n, 16, 1000)
    chunks = [-(-n // c) for c in (4, 32)]
    assert 16 * n + 132 * chunks[1] <= size <= 16 * n + 132 * chunks[0] + 256 * 1024 + 7 * 256


def test_gated_mlp_refusals():
    x, w, v = (torch.zeros(s, dtype=BF16) for s in ((3, 16), (16, 48), (24, 8)))
    for bad in (x.float(), x.half()):
        with pytest.raises(TypeError, match="bfloat16, got x"):
            gated_mlp(bad, w, v)
    with pytest.raises(TypeError, match="gate_up_w"):
        gated_mlp(x, w.float(), v)
    with pytest.raises(TypeError, match="down_w"):
        gated_mlp(x, w, v.float())
    with pytest.raises(ValueError, match="activation"):
        gated_mlp(x, w, v, activation="relu")
    for args in ((x[:, :8], w, v), (x, w[:, :40], v), (x, w, v[:16]), (x, w[0], v), (x, w, v[0]), (x[0, 0], w, v),
                 (x, w[None], v)):
        with pytest.raises(ValueError, match="must be"):
            gated_mlp(*args)
    for shapes in (((3, 12), (12, 48), (24, 8)), ((3, 16), (16, 40), (20, 8)), ((3, 16), (16, 48), (24, 7)),
                   ((3, 0), (0, 48), (24, 8)), ((3, 16), (16, 0), (0, 8))):
        with pytest.raises(ValueError, match="multiples of 8"):
            gated_mlp(*(torch.zeros(s, dtype=BF16) for s in shapes))
    with pytest.raises(RuntimeError, match="GPU"):
        gated_mlp(x, w, v)


def test_gated_entry_points_check_their_arguments():
    lib = _lib.lib()
    at, odd = ctypes.c_void_p(1 << 12), ctypes.c_void_p((1 << 12) + 8)
    fwd = lib.gptrig_gated_mlp_fwd
    good = [at, 16, at, 48, at, 8, 0, at, at, at, 3, 16, 24, 8, None]

    def changed(**by):
        return [by.get(f"a{i}", a) for i, a in enumerate(good)]

    for i in (0, 2, 4, 8, 9):
        assert fwd(*changed(**{f"a{i}": None})) == -1
        assert fwd(*changed(**{f"a{i}": odd})) == -2
    assert fwd(*changed(a7=odd)) == -2
    assert fwd(*changed(a6=2)) == -4
    for i, bad in ((1, 8), (1, 20), (1, 1 << 23), (3, 40), (5, 0), (10, -1), (11, 12), (12, 20), (13, 4), (11, 0),
                   (12, 1 << 20), (13, 1 << 21)):
        assert fwd(*changed(**{f"a{i}": bad})) == -2, (i, bad)
    assert fwd(*changed(a10=0)) == 0
    size = _lib.query("gptrig_gated_mlp_bwd_workspace_bytes", 3, 16, 24, 8)
    bwd = lib.gptrig_gated_mlp_bwd
    call = [at, 8, at, 16, at, 48, at, 8, 0, at, at, at, at, at, 3, 16, 24, 8, at, size, None]
    for i in (0, 2, 4, 6, 9, 10, 18):
        assert bwd(*(None if j == i else a for j, a in enumerate(call))) == -1, i
    for i in (0, 2, 4, 6, 9, 10, 11, 12, 13, 18):
        assert bwd(*(odd if j == i else a for j, a in enumerate(call))) == -2, i
    assert bwd(*(size - 1 if j == 19 else a for j, a in enumerate(call))) == -6
    assert bwd(*(0 if j == 14 else a for j, a in enumerate(call))) == -2
    assert bwd(*(7 if j == 8 else a for j, a in enumerate(call))) == -4
    # Inside: the gradient of the projection's output, and float32 parts of at most 32 slices.
    for n, d, f in ((1, 64, 64), (65536, 768, 2048), (5001, 1000, 2664)):
        size = _lib.query("gptrig_gated_mlp_bwd_workspace_bytes", n, d, f, d)
        assert 4 * n * f <= size <= 4 * n * f + 32 * 12 * d * f + 1024


def test_orthogonalize_refusals():
    u = torch.zeros((4, 8))
    for bad in ([u.half()], [u.double()], [u, u.to(BF16)], [u.int()]):
        with pytest.raises(TypeError, match="all be float32 or all bfloat16"):
            orthogonalize_tensors(bad)
    for bad in (u[0], u[0, 0], torch.empty((65537, 1)), torch.empty((1, 65537))):
        with pytest.raises(ValueError, match=r"updates\[1\] must be matrices"):
            orthogonalize_tensors([u, bad])
    for steps in (0, -1, 1001):
        with pytest.raises(ValueError, match="steps"):
            orthogonalize_tensors([u], steps=steps)
    for c in ((1.0, 2.0), (1.0, 2.0, float("nan")), (1.0, 2.0, 3.0, 4.0), (float("inf"), 0.0, 0.0), (1e39, 0, 0)):
        with pytest.raises(ValueError, match="coefficients"):
            orthogonalize_tensors([u], coefficients=c)
    for eps in (-1e-7, float("nan"), float("inf"), 1e39):
        with pytest.raises(ValueError, match="eps"):
            orthogonalize_tensors([u], eps=eps)
    with pytest.raises(RuntimeError, match="no derivative"):
        orthogonalize_tensors([u, u.clone().requires_grad_()])
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            orthogonalize_tensors([u, forward_ad.make_dual(u.clone(), u)])
        with pytest.raises(RuntimeError, match="GPU"):
            orthogonalize_tensors([u])
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        orthogonalize_tensors([u.clone().requires_grad_()])
    with pytest.raises(RuntimeError, match="GPU"):
        orthogonalize_tensors([u])


def matrices(*rows):
    """Rows of gptrig_matrices: input, output, count, rows, columns."""

    return (ctypes.c_int64 * (4 * len(rows)))(*(v for a, b, n, r, c in rows for v in (a, b, n, r | c << 32)))


def test_orthogonalize_entry_points_check_their_arguments():
    lib = _lib.lib()
    at, f = 1 << 12, ctypes.c_float
    size = lib.gptrig_orthogonalize_workspace_bytes

    def call(table, count=1, type=1, steps=5, eps=1e-7, ws=at, nbytes=1 << 40):
        return lib.gptrig_orthogonalize(table, count, type, steps, f(1.0), f(1.0), f(1.0), f(eps), ws, nbytes, None)

    good = matrices((at, at, 2, 30, 50))
    assert call(None) == -1 and call(good, count=-1) == -2 and call(good, type=2) == -3
    assert call(good, steps=0) == -2 and call(good, eps=-1.0) == -2 and call(good, eps=float("nan")) == -2
    assert call(matrices((0, at, 2, 30, 50))) == -1 and call(matrices((at, 0, 2, 30, 50))) == -1
    assert call(matrices((at + 2, at, 2, 30, 50))) == -2 and call(matrices((at, at + 8, 2, 30, 50))) == -2
    for row in ((at, at, -1, 30, 50), (at, at, 2, 65537, 50), (at, at, 2, 30, 65537)):
        assert call(matrices(row)) == -2 and size(matrices(row), 1) == 0
    assert call(good, ws=None) == -1 and call(good, ws=at + 8) == -2
    assert call(good, nbytes=size(good, 1) - 1) == -6
    assert call(matrices((0, 0, 0, 30, 50), (0, 0, 3, 0, 50)), count=2, ws=None, nbytes=0) == 0
    assert call(None, count=0, ws=None, nbytes=0) == 0


def test_orthogonalize_workspace():
    """Three times X, A and B in 16 bits, rows padded to 32, two diagonals, and the sums: of one launch's
    tensors, which more matrices than fit 2 GiB do not make larger."""

    size = lambda *rows: _lib.lib().gptrig_orthogonalize_workspace_bytes(matrices(*rows), len(rows))  # noqa: E731
    assert size() == 0 and size((0, 0, 0, 5, 5)) == 0
    one = 3 * 2 * 30 * 64 + 2 * 2 * 30 * 32 + 2 * 4 * 32 + 8
    assert one <= size((0, 0, 1, 30, 50)) <= one + 8 * 255
    assert size((0, 0, 1, 30, 50)) == size((0, 0, 1, 50, 30))
    assert 7 * one <= size((0, 0, 3, 30, 50), (0, 0, 4, 50, 30)) <= 7 * one + 8 * 255
    assert 64 * one <= size(*[(0, 0, 1, 30, 50)] * 100) <= 64 * one + 8 * 255
    for rows in ([(0, 0, 1000, 2048, 2048)], [(0, 0, 1, 4096, 4096)] * 60, [(0, 0, 10 ** 9, 100, 100)]):
        assert (1 << 30) < size(*rows) <= (1 << 31) + 4096
    big = size((0, 0, 3, 65536, 65536))
    assert 10 * 2 ** 32 <= big <= 10 * 2 ** 32 + 2 ** 23
