"""``nn.gated_mlp`` on the ways that its sizes choose: from which number of tiles of 256 x 256 on a product takes those
(68 for x W and dy V^T, 150 for h V and dx), with and without what the backward needs.

``model`` computes the block in 64 bits with the kernels' roundings: h, dg, du and the results to bfloat16, g and u to
float16 scaled by a power of two for each run of 16 features, where the backward finds them.  The kernels' own float32
sums differ from it by some 2^-22, which moves one value in some thousands over a border between two bfloat16 values:
their distance from the model is a small part of the model's from the exact result (a fiftieth to a tenth with float32
products on the CPU).  A quarter is allowed.  With g and u held in bfloat16 it would be 1.5 times as large as the model's
own, which the test finds in the model itself.
"""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from test_gpu_gated_mlp import BF16, DEV, F64, NAMES, act, bounds, check, data, exact, kernels

from gptrig.nn import gated_mlp

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def bf16(t):
    return t.to(F32).to(BF16).to(F64)


def kept(t):
    """Each run of 16 features (the last may be shorter) scaled to 2^14 .. 2^15, in float16."""

    n, f = t.shape
    t = torch.nn.functional.pad(t.to(F32).to(F64), (0, -f % 16)).view(n, -1, 16)
    power = torch.frexp(t.abs().amax(-1, keepdim=True)).exponent
    return torch.ldexp(torch.ldexp(t, 15 - power).to(F16).to(F64), power - 15).view(n, -1)[:, :f]


def model(x, w, v, dy, kind, kept=kept, product=lambda a, b: a @ b):
    x, w, v, dy = (t.to(F64) for t in (x, w, v, dy))
    g, u = product(x, w).chunk(2, 1)
    h = bf16(act(g, kind) * u)
    y = bf16(product(h, v))
    dh = product(dy, v.T)
    g, u = kept(g), kept(u)
    leaf = g.clone().requires_grad_()
    a = act(leaf, kind)
    (slope,) = torch.autograd.grad(a.sum(), leaf)
    dp = bf16(torch.cat((dh * u * slope, dh * a.detach()), 1))
    return [y, bf16(product(dp, w.T)), bf16(product(x.T, dp)), bf16(product(h.T, dy))]


def distance(a, b):
    return torch.linalg.norm(a.cpu().to(F64) - b)


# Tiles of x W, dy V^T, and of h V and dx: 64, 32, 24; 68, 34, 17; 153, 85, 17; 102, 51, 153; 153, 102, 153.
@pytest.mark.parametrize("n,d,f,kind", [(2000, 768, 1024, "silu"), (4300, 64, 512, "gelu"), (4097, 64, 1032, "silu"),
                                        (13000, 768, 136, "gelu"), (12900, 768, 264, "silu")])
def test_roundings(n, d, f, kind):
    args = data(n, d, f, d)
    wanted, held = exact(*args, kind), model(*args, kind)
    coarse = model(*args, kind, kept=bf16)
    for name, a, b, c, e in zip(NAMES, kernels(*args, kind), wanted, held, coarse):
        assert distance(a, c) <= 0.25 * distance(c, b), (name, (distance(a, c) / distance(c, b)).item())
        if name in ("x", "gate_up_w"):
            assert distance(e, c) > distance(c, b)


@pytest.mark.parametrize("n,d,f,kind", [(13000, 768, 136, "gelu"), (12900, 768, 264, "silu"), (13000, 768, 128, "silu")])
def test_large_tiles(n, d, f, kind):
    """Value by value; and without a gradient, where nothing is kept, the same bits."""

    args = data(n, d, f, d)
    check(kernels(*args, kind), exact(*args, kind), bounds(*args, kind))
    x, w, v = (t.to(DEV) for t in args[:3])
    y = gated_mlp(x, w, v, activation=kind)
    assert torch.equal(y, gated_mlp(x.requires_grad_(), w, v, activation=kind))


@pytest.mark.parametrize("n,f", [(300, 72), (4300, 512)])
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_nothing_kept(n, f, kind):
    x, w, v, _ = (t.to(DEV) for t in data(n, 64, f, 64))
    y = gated_mlp(x, w, v, activation=kind)
    assert torch.equal(y, gated_mlp(x.requires_grad_(), w, v, activation=kind))


def test_on_another_stream():
    args = data(700, 128, 136, 128)
    wanted = kernels(*args, "silu")
    leaves = [t.to(DEV).requires_grad_() for t in args[:3]]
    dy = args[3].to(DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = gated_mlp(*leaves)
        got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, wanted))


def test_transforms_are_refused():
    x, w, v, _ = (t.to(DEV) for t in data(10, 64, 72, 40))
    with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        gated_mlp(forward_ad.make_dual(x, x), w, v)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: gated_mlp(t, w, v), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gated_mlp(t, w, v).float().sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: gated_mlp(t, w, v))(x.view(2, 5, 64))
