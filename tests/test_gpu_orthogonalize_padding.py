"""``optim.orthogonalize_tensors`` where what lies past a matrix's last row could pass float16.

All rows have the same length and are orthogonal but for one pair, the last row and one before it.  With b = -2 c D, D a
row's squared length, the factor of their entry of A cancels in B, while c D times it is past 65504: the entry that a
row of zeros behind the last would get with the last row's A.  One step, so that the result is bfloat16 of float32 sums.
"""

from __future__ import annotations

import pytest
import torch

from gptrig.optim import orthogonalize_tensors

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F64 = torch.float64
C = 2.0 ** 33


def matrix(m, n, partner):
    u = torch.eye(m, n)
    u[m - 1, m - 1] = u[m - 1, partner] = 0.5 ** 0.5
    return u


@pytest.mark.parametrize("m,n,count", [(70, 96, 1), (130, 160, 2), (130, 160, 200), (203, 210, 140)])
@pytest.mark.parametrize("turned", [False, True])
def test_rows_past_the_last(m, n, count, turned):
    """Each value against the formula's.  X's operand is off by e = 2^-11 at most, D by 2e and A's entry by 2e; of
    X' = (a + b D_i + c (D_i^2 + O O_ii)) X_i + B_ij X_j the first factor has terms of 2 c D^2, c D^2 and c D^2 / 2, off
    by 2e, 4e and 4e of themselves, and B_ij is c A (D_i + D_j - 2 D) and so off by 4e c D A: with |X| at most D^(1/2)
    and A at most D, (4 + 4 + 2 + 4) e = 14 e of c D^(5/2), and one more half step for the result (2^-8 of itself)."""

    partner = 3
    u = matrix(m, n, partner)
    d = 1.0 / m
    a, b, c = 1.0, -2 * C * d, C
    assert C * d * d / 2 ** 0.5 > 65504
    x = u.to(F64) / m ** 0.5
    gram = x @ x.T
    want = a * x + (b * gram + c * gram @ gram) @ x
    given = u.T.contiguous() if turned else u
    got = orthogonalize_tensors([given.expand(count, *given.shape).to(DEV)], steps=1, coefficients=(a, b, c), eps=0.0)[0]
    got = (got.transpose(-1, -2) if turned else got).cpu().to(F64)
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    assert (off <= 14 * 2.0 ** -11 * C * d ** 2.5 + 2.0 ** -8 * want.abs()).all(), off.max() / (C * d ** 2.5)


def test_on_another_stream():
    updates = [torch.randn(s, generator=torch.Generator().manual_seed(1)).to(DEV) for s in ((70, 100), (3, 200, 40))]
    wanted = orthogonalize_tensors(updates)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = orthogonalize_tensors(updates)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, wanted))


def test_transforms_are_refused():
    u = torch.randn((4, 20, 30), device=DEV)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: orthogonalize_tensors([t])[0], (u,), (u,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: orthogonalize_tensors([t])[0].float().sum())(u)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: orthogonalize_tensors([t])[0])(u)
