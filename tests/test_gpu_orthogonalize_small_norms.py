"""``optim.orthogonalize_tensors`` of matrices whose norm is far below ``eps``: x is small, A and B smaller still, and the
result about a^steps x.

x is held in two float16, the second at 2^11 times its size, so that a value below 2^-14 is held to 2^-36 absolutely
(float16 ends at 2^-24, half a step is 2^-25) and a larger one to 2^-22 of itself.  Each step adds that once and
multiplies what there is by a: ``direct``, element by element.

The products see x by its first float16, off by h = 2^-11 |x| + 2^-25 (m n)^1/2 (|.| the Frobenius norm, s the spectral
one).  So A = x x^T is off by 2 s h + h^2, and by its own rounding r(A) = 2^-11 |A| + 2^-25 m; B = b A + c A A by
(|b| + 2 c s^2) times that and r(B); and B x by |B| h + s times B's.  An error e of x itself comes through B x as (3 |b|
s^2 + 5 c s^4) |e|, the derivative of b x^3 + c x^5, while a e is in ``direct`` or multiplied here.  The float32 sums are
below 2^-20 of |x|.  All of that is ``other``.  The result is rounded to bfloat16 once.
"""

from __future__ import annotations

import pytest
import torch

from gptrig.optim import orthogonalize_tensors

pytestmark = pytest.mark.gpu

F64 = torch.float64
A, B, C = 3.4445, -4.7750, 2.0315


@pytest.mark.parametrize("norm", [1e-2, 1e-4, 1e-6, 1e-8, 1e-12, 1e-30])
@pytest.mark.parametrize("rows,cols", [(40, 72), (200, 96)])
@pytest.mark.parametrize("steps", [1, 5])
def test_norms_below_eps(rows, cols, norm, steps):
    eps = 1e-7
    u = torch.randn((rows, cols), generator=torch.Generator().manual_seed(rows))
    u = (u.to(F64) * (norm * eps / torch.linalg.norm(u.to(F64)))).float()
    x = u.to(F64) / (torch.linalg.norm(u.to(F64)) + eps)
    x = x.T if rows > cols else x
    size = (rows * cols) ** 0.5
    direct, other = 2.0 ** -36 + 2.0 ** -22 * x.abs().max(), 0.0
    for _ in range(steps):
        gram = x @ x.T
        more = B * gram + C * gram @ gram
        whole, s = torch.linalg.norm(x), torch.linalg.matrix_norm(x, 2)
        h = 2.0 ** -11 * whole + 2.0 ** -25 * size
        rounding = lambda t: 2.0 ** -11 * torch.linalg.norm(t) + 2.0 ** -25 * len(t)  # noqa: E731
        off_gram = 2 * s * h + h ** 2 + rounding(gram)
        off_more = (abs(B) + 2 * C * s ** 2) * off_gram + rounding(more)
        through = 3 * abs(B) * s ** 2 + 5 * C * s ** 4
        other = (A + through) * other + through * direct * size + torch.linalg.norm(more) * h + s * off_more
        other = other + 2.0 ** -20 * whole
        x = A * x + more @ x
        direct = A * direct + 2.0 ** -36 + 2.0 ** -22 * x.abs().max()
    x = x.T if rows > cols else x
    (got,) = orthogonalize_tensors([u.to("cuda:0")], steps=steps, eps=eps)
    off = (got.cpu().to(F64) - x).abs()
    limit = 2.0 ** -8 * x.abs() + direct + other
    assert (off <= limit).all(), (off / limit).max().item()
