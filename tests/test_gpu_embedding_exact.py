"""``nn.embedding``'s gradient where its sums have to be exact: whole numbers as gradients, whose sums float32 holds, so
that every term that is lost, added twice or given to another row shows.  The lengths reach each of the plan's forms:
chunks of 4 to 32 pairs, rows over thousands of chunks (which the join takes in many rounds), blocks of more than one
segment."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from gptrig.nn import embedding

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def wanted(tokens, dy, vocab, kind):
    tokens = tokens.long()
    inside = (tokens >= 0) & (tokens < vocab)
    sums = torch.zeros((vocab, dy.shape[1]), dtype=torch.int64)
    sums.index_add_(0, tokens[inside], dy.long()[inside])
    assert sums.abs().max() < 2 ** 24
    return sums.to(F32).to(kind)


def gradient(tokens, dy, vocab, kind, out_type):
    leaf = torch.zeros((vocab, dy.shape[1]), dtype=kind, device=DEV, requires_grad=True)
    y = embedding(tokens.to(DEV), leaf, dtype=out_type)
    return torch.autograd.grad(y, leaf, dy.to(out_type).to(DEV))[0].cpu()


def check(tokens, vocab, d, kind=F32, out_type=BF16, seed=0):
    dy = torch.randint(-8, 9, (len(tokens), d), generator=torch.Generator().manual_seed(seed))
    assert torch.equal(gradient(tokens, dy, vocab, kind, out_type), wanted(tokens, dy, vocab, kind))


@pytest.mark.parametrize("n", [1, 5, 300, 8192, 8193, 16384, 20001, 40000, 65536, 65543, 140000])
@pytest.mark.parametrize("vocab,wide", [(1, False), (9, True), (300, False), (66000, True)])
def test_sums_are_exact(n, vocab, wide):
    g = torch.Generator().manual_seed(n)
    tokens = torch.randint(-1, vocab + 1, (n,), generator=g, dtype=torch.int64 if wide else torch.int32)
    check(tokens, vocab, 20)


@pytest.mark.parametrize("n", [300, 8192, 40000, 65536, 131075])
@pytest.mark.parametrize("d", [4, 520, 1001])
def test_one_row_takes_all(n, d):
    tokens = torch.full((n,), 5, dtype=torch.int64)
    tokens[-3:] = 6
    check(tokens, 9, d, out_type=F32 if d == 4 else BF16)


@pytest.mark.parametrize("n", [524288, 524289, 1100003])
def test_blocks_of_more_than_one_segment(n):
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 70000, (n,), generator=g, dtype=torch.int32)
    tokens[torch.rand(n, generator=g) < 0.3] = 69999
    check(tokens, 70000, 4)


@pytest.mark.parametrize("out_type", [BF16, F32])
@pytest.mark.parametrize("kind", [BF16, F32])
def test_types(kind, out_type):
    tokens = torch.randint(0, 700, (65600,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    check(tokens, 700, 260, kind, out_type)


def test_runs_of_every_length():
    """Rows of 0 to 200 tokens, so that runs begin and end everywhere in a chunk; shuffled."""

    tokens = torch.repeat_interleave(torch.arange(500), torch.arange(500) % 201)
    tokens = tokens[torch.randperm(len(tokens), generator=torch.Generator().manual_seed(3))]
    check(tokens.to(torch.int32), 500, 64)


def test_transforms_are_refused():
    tokens, table = torch.zeros(6, dtype=torch.int32, device=DEV), torch.randn((5, 8), device=DEV)
    with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        embedding(tokens, forward_ad.make_dual(table, table))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: embedding(tokens, t), (table,), (table,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: embedding(tokens, t, dtype=F32).sum())(table)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda i: embedding(i, table))(tokens.view(2, 3))
