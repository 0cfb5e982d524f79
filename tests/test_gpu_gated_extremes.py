"""``nn.gated_mlp`` at the ends of its values' range, against its formula in 64 bits on the CPU.

The bounds are those of the block's other tests (``bounds`` there), which are relative, and ``slack``: what float32 and
bfloat16 may flush below 2^-126 of g, u, dg and du and of each product on the way.
"""

from __future__ import annotations

import pytest
import torch
from test_gpu_gated_mlp import BF16, DEV, F64, NAMES, bounds, data, exact, kernels

from gptrig.nn import gelu

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -126
# A few tokens, and enough tiles of 256 x 256 in x W (153) and dy V^T (85) that the kernels of those tiles take them.
SIZES = [(40, 64, 72, 64), (4097, 64, 1032, 64)]


def slack(x, w, v, dy):
    x, w, v, dy = (t.to(F64).abs() for t in (x, w, v, dy))
    n, (f, _) = len(x), v.shape
    each = 4 * LEAST * (1 + dy @ v.T)  # of dg and du: a flushed u or g times dh, and their own
    both = torch.cat((each, each), 1)
    return [LEAST * (f + v.sum(0, keepdim=True).expand(n, -1)), both @ w.T + 2 * f * LEAST, x.T @ both + n * LEAST,
            LEAST * (n + dy.sum(0, keepdim=True).expand(f, -1))]


def off_by(a, b):
    return (a.cpu().to(F64) - b).abs()


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("which", ["x", "gate_up_w"])
@pytest.mark.parametrize("scale", [1e-33, 5e-35, 2e-35])
@pytest.mark.parametrize("sizes", SIZES)
def test_tiny_values(sizes, scale, which, kind):
    """g and u of some 1e-35: the gradient of what is not tiny is as small, and no less exact."""

    x, w, v, dy = data(*sizes)
    if which == "x":
        x = (x.to(F64) * scale).to(BF16)
    else:
        w = (w.to(F64) * scale).to(BF16)
    args = (x, w, v, dy)
    wanted, limits, more = exact(*args, kind), bounds(*args, kind), slack(*args)
    assert wanted[1 if which == "x" else 2].abs().max() > scale / 10
    for name, a, b, limit, least in zip(NAMES, kernels(*args, kind), wanted, limits, more):
        off = off_by(a, b)
        assert (off <= 1.1 * limit + least).all(), (name, (off / (1.1 * limit + least)).max().item())


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("column", [5, 64 + 37])
@pytest.mark.parametrize("sizes", [(n, d, 64 if n == 40 else f, o) for n, d, f, o in SIZES])
def test_a_feature_is_its_own(sizes, column, value, kind):
    """One infinity (or NaN) of the projection spoils one feature's g or u; the weights' gradients of all others, its
    neighbours in a run of 16 among them, are the formula's."""

    n, d, f, _ = sizes
    column = column if column < 64 else f + column - 64
    x, w, v, dy = data(*sizes)
    clean = (x, w.clone(), v, dy)
    clean[1][3, column] = 0
    w[3, column] = value
    x[:, 3] += (x[:, 3] == 0).to(BF16)
    wanted, limits = exact(*clean, kind), bounds(*clean, kind)
    got = kernels(x, w, v, dy, kind)
    others = torch.arange(f) != column % f
    for i, at in ((2, (slice(None), others.repeat(2))), (3, (others,))):
        off = off_by(got[i], wanted[i])[at]
        assert (off <= 1.1 * limits[i][at] + 1e-30).all(), (NAMES[i], (off / (limits[i][at] + 1e-30)).max().item())


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("which,scale", [("x", 1e6), ("x", 1e13), ("x", 1e14), ("x", 1e17), ("gate", 1e14), ("gate", 1e30)])
@pytest.mark.parametrize("sizes", [(40, 64, 64, 64), (4097, 64, 1032, 64)])
def test_far_gates(sizes, which, scale, kind):
    """Gates so far out that the cube in GELU's argument passes float32: its limits 0 and 1, no NaN."""

    x, w, v, dy = data(*sizes)
    if which == "x":
        x = (x.to(F64) * scale).to(BF16)
    else:
        f = len(v)
        w[:, :f] = (w[:, :f].to(F64) * scale).to(BF16)
    args = (x, w, v, dy)
    for name, a, b, limit in zip(NAMES, kernels(*args, kind), exact(*args, kind), bounds(*args, kind)):
        off = off_by(a, b)
        assert torch.isfinite(a).all() and (off <= 1.1 * limit + 1e-30).all(), name


def test_gelu_of_far_values():
    """``nn.gelu`` and its gradient, the same functions: 0 or x, 0 or 1."""

    size = torch.tensor([20.0, 1e4, 1e6, 1e12, 1.3e13, 1.6e13, 1e14, 1e18, 1.9e19, 1e20, 1e30, 3e38], dtype=F64).to(BF16)
    x = torch.cat((size, -size)).to(DEV).requires_grad_()
    y = gelu(x)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(y, torch.where(x > 0, x, 0)) and torch.equal(dx, (x > 0).to(BF16))
    x = torch.full((8,), float("nan"), dtype=BF16, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad(gelu(x), x, torch.ones_like(x))
    assert torch.isnan(dx).all()
