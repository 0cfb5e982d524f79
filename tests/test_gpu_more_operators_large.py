"""``embedding``, ``gated_mlp`` and ``orthogonalize_tensors`` where element offsets pass 2^31."""

from __future__ import annotations

import pytest
import torch

from gptrig.nn import embedding, gated_mlp
from gptrig.optim import orthogonalize_tensors

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def test_embedding_of_many_wide_rows():
    """y and dy of 2.3e9 elements: each row of y, and the sums of whole numbers, which float32 holds."""

    n, d, vocab = 140001, 16384, 300
    tokens = torch.randint(-1, vocab, (n,), generator=generator(0), device=DEV, dtype=torch.int32)
    table = torch.randn((vocab, d), generator=generator(1), device=DEV, requires_grad=True)
    y = embedding(tokens, table, scale=3.0)
    dy = torch.empty((n, d), dtype=BF16, device=DEV)
    want = torch.zeros((vocab + 1, d), dtype=F64, device=DEV)
    for i in range(0, n, 20000):
        part = tokens[i:i + 20000].long() % (vocab + 1)  # (-1: the row behind the last)
        rows = torch.cat((table.detach(), torch.zeros((1, d), device=DEV)))[part]
        assert torch.equal(y[i:i + 20000], (rows * 3.0).to(BF16))
        dy[i:i + 20000] = torch.randint(-4, 5, rows.shape, generator=generator(i), device=DEV)
        want.index_add_(0, part, dy[i:i + 20000].to(F64))
    (grad,) = torch.autograd.grad(y, table, dy)
    assert torch.equal(grad, (3 * want[:vocab]).to(F32))


def test_embedding_of_a_large_table():
    vocab, d = 70000, 32768
    table = torch.empty((vocab, d), dtype=BF16, device=DEV).normal_(generator=generator(0)).requires_grad_()
    tokens = torch.tensor([0, vocab - 1, 69990, 65536, 69990, 65535, vocab], device=DEV)
    y = embedding(tokens, table)
    assert torch.equal(y[:6], table.detach()[tokens[:6]]) and (y[6] == 0).all()
    (grad,) = torch.autograd.grad(y, table, torch.ones_like(y))
    named = grad[tokens[:6]]
    assert torch.equal(named, torch.tensor([1.0, 1, 2, 1, 2, 1], device=DEV).to(BF16)[:, None].expand_as(named))
    grad[tokens[:6]] = 0
    assert not any(part.any() for part in grad.split(10000))


def test_gated_block_of_many_tokens():
    """Each token's rows in the bits of a call on its slice (of as many tiles as take the same kernels); the weights'
    gradients against the slices' sum, each rounded to bfloat16 once."""

    n, d, f = 2 ** 21 + 3, 64, 512
    x, dy = (torch.empty((n, d), dtype=BF16, device=DEV).normal_(generator=generator(i)) for i in (0, 1))
    w = (torch.randn((d, 2 * f), generator=generator(2), device=DEV) * d ** -0.5).to(BF16)
    v = (torch.randn((f, d), generator=generator(3), device=DEV) * f ** -0.5).to(BF16)

    def both(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, v)]
        y = gated_mlp(*leaves)
        return y.detach(), *torch.autograd.grad(y, leaves, dy)

    y, dx, dw, dv = both(x, dy)
    sums = [torch.zeros(t.shape, dtype=F64, device=DEV) for t in (dw, dv, dw, dv)]
    cuts = [*range(0, n - 70000, 65536), n]
    for begin, end in zip(cuts, cuts[1:]):
        part = both(x[begin:end], dy[begin:end])
        assert torch.equal(y[begin:end], part[0]) and torch.equal(dx[begin:end], part[1]), begin
        for i in (0, 1):
            sums[i] += part[2 + i]
            sums[2 + i] += part[2 + i].abs()
    for got, total, size in ((dw, sums[0], sums[2]), (dv, sums[1], sums[3])):
        # (Float32 sums of n terms are off by some 2^-24 n^1/2 = 2^-13 of their usual size.)
        assert ((got.to(F64) - total).abs() <= 2.0 ** -8 * (total.abs() + size) + 2.0 ** -11 * size).all()


def test_orthogonalize_a_large_matrix():
    """A permutation of 48000 rows with signs and a scale: each step takes its one singular value s = 48000^-1/2 to
    a s + b s^3 + c s^5.  X holds 22 bits of it, and its operands 11 of what a step adds."""

    n, (a, b, c) = 48000, (3.4445, -4.7750, 2.0315)
    place = torch.randperm(n, generator=generator(0), device=DEV)
    sign = torch.randint(0, 2, (n,), generator=generator(1), device=DEV) * 2.0 - 1
    u = torch.zeros((n, n), device=DEV)
    rows = torch.arange(n, device=DEV)
    u[rows, place] = 7.0 * sign
    (got,) = orthogonalize_tensors([u], steps=2)
    s = n ** -0.5
    for _ in range(2):
        s = a * s + b * s ** 3 + c * s ** 5
    assert ((got[rows, place].to(F64) - s * sign).abs() <= s * (2.0 ** -8 + 2.0 ** -10)).all()
    got[rows, place] = 0
    assert not any(part.any() for part in got.split(6000))
