"""``nn.embedding`` against the formula in 64 bits on the CPU.

Forward: one float32 product (the scale rounded to float32 before it) and the rounding to the output's type.
Gradient: a row's c terms are added in float32 in some fixed order, at most c - 1 roundings of partial sums that the
sum of the magnitudes bounds, then the scale (rounded), its product, and the rounding to the table's type.
"""

from __future__ import annotations

import math

import pytest
import torch

from gptrig.nn import embedding

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24
HALF = {BF16: 2.0 ** -8, F32: U}


def data(n, d, vocab, table_type=F32, out_type=BF16, wide=False, outside=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    tokens = (torch.exp(torch.rand(n, generator=g, dtype=F64) * math.log(vocab + 1)) - 1).floor().clamp(0, vocab - 1)
    tokens = tokens.to(torch.int64 if wide else torch.int32)
    if outside and n:
        tokens[torch.rand(n, generator=g) < 0.2] = -1
        tokens[torch.rand(n, generator=g) < 0.1] = vocab
        tokens[0] = 2 ** 40 if wide else 2 ** 31 - 1
        tokens[-1] = -(2 ** 32) if wide else -(2 ** 31)
    table = torch.randn((vocab, d), generator=g).to(table_type)
    dy = torch.randn((n, d), generator=g).to(out_type)
    return tokens, table, dy


def exact(tokens, table, dy, scale):
    """y, the gradient, and for each of its rows the sum of the terms' magnitudes and their number."""

    tokens = tokens.reshape(-1).to(torch.int64)
    vocab = table.shape[0]
    inside = (tokens >= 0) & (tokens < vocab)
    at = torch.where(inside, tokens, 0)
    y = table.to(F64)[at] * scale * inside[:, None]
    dy = dy.to(F64).reshape(-1, table.shape[1])[inside]
    grad, size = torch.zeros(table.shape, dtype=F64), torch.zeros(table.shape, dtype=F64)
    grad.index_add_(0, at[inside], dy)
    size.index_add_(0, at[inside], dy.abs())
    return y, grad * scale, size * abs(scale), torch.bincount(at[inside], minlength=vocab)[:, None]


def check(tokens, table, dy, scale, got_y, got_grad):
    y, grad, size, count = exact(tokens, table, dy, scale)
    got_y, got_grad = got_y.detach().cpu().reshape(y.shape), got_grad.cpu()
    assert ((got_y.to(F64) - y).abs() <= y.abs() * (2 * U + HALF[got_y.dtype]) * 1.01).all()
    off = (got_grad.to(F64) - grad).abs()
    assert (off <= ((count + 1) * U * size + grad.abs() * HALF[got_grad.dtype]) * 1.01).all()
    assert (got_grad[(count == 0).expand_as(got_grad)] == 0).all()


def both(tokens, table, dy, scale, dtype):
    leaf = table.to(DEV).requires_grad_()
    y = embedding(tokens.to(DEV), leaf, scale=scale, dtype=dtype)
    assert y.dtype == dtype and y.shape == (*tokens.shape, table.shape[1])
    return y, torch.autograd.grad(y, leaf, dy.to(DEV))[0]


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 8192, 8193, 20001])
@pytest.mark.parametrize("vocab", [1, 2, 255, 256, 1000])
def test_lengths_and_vocabularies(n, vocab):
    tokens, table, dy = data(n, 20, vocab, outside=n > 2)
    check(tokens, table, dy, 1.0, *both(tokens, table, dy, 1.0, BF16))


@pytest.mark.parametrize("vocab", [65535, 65536, 70001, 2 ** 24 + 3])
@pytest.mark.parametrize("n", [700, 12345])
def test_wide_keys(n, vocab):
    """Keys of two, three and four digits, spread evenly."""

    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, vocab, (n,), generator=g, dtype=torch.int32)
    tokens[n // 2:] = tokens[: n - n // 2].clone()
    tokens[0], tokens[1] = vocab - 1, 0
    table, dy = torch.randn((vocab, 4), generator=g), torch.randn((n, 4), generator=g)
    check(tokens, table, dy, 0.5, *both(tokens, table, dy, 0.5, F32))


@pytest.mark.parametrize("out_type", [BF16, F32])
@pytest.mark.parametrize("table_type", [BF16, F32])
@pytest.mark.parametrize("d", [1, 3, 4, 64, 255, 256, 260, 768, 1001])
def test_widths_and_types(d, table_type, out_type):
    tokens, table, dy = data(517, d, 300, table_type, out_type, wide=d % 2 == 1, outside=True, seed=d)
    check(tokens, table, dy, -1.7, *both(tokens, table, dy, -1.7, out_type))


@pytest.mark.parametrize("n", [300, 40000])
def test_one_row_takes_all(n):
    """A row whose sum crosses every chunk, and one of a few tokens at the end."""

    tokens = torch.full((n,), 5, dtype=torch.int64)
    tokens[-3:] = 6
    _, table, dy = data(n, 520, 9)
    check(tokens, table, dy, 2.0, *both(tokens, table, dy, 2.0, BF16))


def test_no_tokens():
    table = torch.randn((7, 12), device=DEV, requires_grad=True)
    y = embedding(torch.zeros((3, 0), dtype=torch.int32, device=DEV), table)
    assert y.shape == (3, 0, 12) and y.dtype == BF16
    (grad,) = torch.autograd.grad(y, table, torch.zeros_like(y))
    assert (grad == 0).all() and grad.shape == table.shape


def test_all_outside():
    tokens = torch.tensor([-1, 7, 100, -5], dtype=torch.int32)
    table, dy = torch.randn((7, 12)), torch.randn((4, 12))
    y, grad = both(tokens, table, dy, 1.0, F32)
    assert (y == 0).all() and (grad == 0).all()


def test_shapes_and_strides():
    """Tokens as a strided view, a table inside a wider one, gradients that repeat a row or run over columns first."""

    tokens, table, _ = data(600, 24, 50, wide=True, outside=True)
    tokens = tokens.view(20, 30)
    wide = torch.randn((50, 31), device=DEV)
    wide[:, 3:27] = table.to(DEV)
    for view in (wide[:, 3:27], wide.t().contiguous().t()[:, 3:27]):
        leaf = view.detach().requires_grad_()
        y = embedding(tokens.to(DEV).t(), leaf, scale=3.0, dtype=F32)
        for dy in (torch.randn((1, 1, 24)).expand(30, 20, 24), torch.randn((24, 30, 20)).permute(1, 2, 0),
                   torch.randn((30, 20, 25))[..., 1:]):
            (grad,) = torch.autograd.grad(y, leaf, dy.to(DEV), retain_graph=True)
            check(tokens.t(), table, dy, 3.0, y, grad)
    y = embedding(tokens.to(DEV)[3, 4], table.to(DEV))
    assert y.shape == (24,)


def test_gradient_by_differences():
    """y is linear in the table: the change that a small change of the table makes is the gradient's."""

    tokens, table, dy = data(300, 40, 60, out_type=F32)
    step = torch.randn(table.shape, generator=torch.Generator().manual_seed(5)).to(F64)
    _, grad = both(tokens, table, dy, 1.5, F32)
    with torch.no_grad():
        plus, minus = (embedding(tokens.to(DEV), (table.to(F64) + s * step).to(F32).to(DEV), scale=1.5, dtype=F32)
                       for s in (0.5, -0.5))
    by_difference = ((plus.cpu().to(F64) - minus.cpu().to(F64)) * dy.to(F64)).sum()
    size = (1.5 * (table.to(F64).abs() + step.abs())[tokens.long()] * dy.to(F64).abs()).sum()
    # Six roundings of 2^-24 of each term, and the gradient's own sums of at most 300.
    assert abs(by_difference - (grad.cpu().to(F64) * step).sum()) <= 306 * U * size


def test_same_bits():
    tokens, table, dy = data(30000, 256, 400)
    first = both(tokens, table, dy, 1.0, BF16)[1]
    for _ in range(3):
        assert torch.equal(first, both(tokens, table, dy, 1.0, BF16)[1])


def test_captured_and_replayed():
    tokens, table, dy = (t.to(DEV) for t in data(9000, 96, 500, outside=True))
    side = torch.cuda.Stream()
    leaf = table.clone().requires_grad_()

    def step():
        y = embedding(tokens, leaf, scale=2.0)
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]

    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    for seed in range(3):
        other, table2, dy2 = data(9000, 96, 500, outside=True, seed=seed + 10)
        tokens.copy_(other), dy.copy_(dy2)
        with torch.no_grad():
            leaf.copy_(table2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(other, table2, dy2, 2.0, *got)


def test_on_another_stream():
    tokens, table, dy = data(5000, 64, 100)
    tokens_d, dy_d = tokens.to(DEV), dy.to(DEV)
    leaf = table.to(DEV).requires_grad_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = embedding(tokens_d, leaf)
        (grad,) = torch.autograd.grad(y, leaf, dy_d)
    side.synchronize()
    check(tokens, table, dy, 1.0, y, grad)


def test_second_derivatives_are_refused():
    tokens, table, dy = data(10, 8, 5)
    leaf = table.to(DEV).requires_grad_()
    y = embedding(tokens.to(DEV), leaf)
    (grad,) = torch.autograd.grad(y, leaf, dy.to(DEV).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()
