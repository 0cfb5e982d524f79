"""``nn.gated_mlp`` against its formula in 64 bits on the CPU.

The bounds follow each value's errors through the formula (``bounds``): a float32 sum of k products is off by at most k
roundings of 2^-24 of the sum of their magnitudes, the activation and its derivative by 16 such of their own size (an
exponential, a quotient, products), a value held in bfloat16 by 2^-8 of itself; first-order terms, with a tenth for the
rest.  |act'| is below 1.13 and |act''| below 1.
"""

from __future__ import annotations

import math

import pytest
import torch

from gptrig.nn import gated_mlp

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F64 = torch.bfloat16, torch.float64
U, HALF = 2.0 ** -24, 2.0 ** -8
NAMES = ("y", "x", "gate_up_w", "down_w")


def act(g, kind):
    if kind == "silu":
        return g * torch.sigmoid(g)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def formula(x, w, v, kind):
    g, u = (x @ w).chunk(2, -1)
    return (act(g, kind) * u) @ v


def exact(x, w, v, dy, kind):
    leaves = [t.to(F64).requires_grad_() for t in (x, w, v)]
    y = formula(*leaves, kind)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy.to(F64))]


def bounds(x, w, v, dy, kind):
    x, w, v, dy = (t.to(F64) for t in (x, w, v, dy))
    n, d = x.shape
    f, d_out = v.shape
    p = x @ w
    ep = d * U * (x.abs() @ w.abs())
    g, u = p.chunk(2, 1)
    eg, eu = ep.chunk(2, 1)
    leaf = g.clone().requires_grad_()
    a = act(leaf, kind)
    (s,) = torch.autograd.grad(a.sum(), leaf)
    a = a.detach()
    h = a * u
    eh = h.abs() * (HALF + 16 * U) + 1.13 * u.abs() * eg + a.abs() * eu
    y = h @ v
    ey = eh @ v.abs() + f * U * (h.abs() @ v.abs()) + y.abs() * HALF
    dh = dy @ v.T
    edh = d_out * U * (dy.abs() @ v.abs().T)
    kg, ku = g.abs() * HALF + eg, u.abs() * HALF + eu  # as the backward finds them
    dg, du = dh * u * s, dh * a
    edg = (u * s).abs() * edh + (dh * s).abs() * ku + (dh * u).abs() * kg + dg.abs() * HALF + 16 * U * (dh * u).abs()
    edu = a.abs() * edh + 1.13 * dh.abs() * kg + du.abs() * (HALF + 16 * U)
    dp, edp = torch.cat((dg, du), 1), torch.cat((edg, edu), 1)
    ex = edp @ w.abs().T + 2 * f * U * (dp.abs() @ w.abs().T) + (dp @ w.T).abs() * HALF
    ew = x.abs().T @ edp + n * U * (x.abs().T @ dp.abs()) + (x.T @ dp).abs() * HALF
    ev = eh.T @ dy.abs() + n * U * (h.abs().T @ dy.abs()) + (h.T @ dy).abs() * HALF
    return [ey, ex, ew, ev]


def data(n, d, f, d_out, seed=0):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g)
    return (normal(n, d).to(BF16), (normal(d, 2 * f) * d ** -0.5).to(BF16), (normal(f, d_out) * f ** -0.5).to(BF16),
            normal(n, d_out).to(BF16))


def kernels(x, w, v, dy, kind):
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, v)]
    y = gated_mlp(*leaves, activation=kind)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy.to(DEV))]


def check(got, wanted, limits):
    for name, a, b, limit in zip(NAMES, got, wanted, limits):
        assert a.dtype == BF16 and a.shape == b.shape
        off = (a.cpu().to(F64) - b).abs()
        assert (off <= 1.1 * limit + 1e-30).all(), (name, (off / (limit + 1e-30)).max().item())


SIZES = [(8, 8, 8), (64, 64, 64), (136, 200, 72), (264, 128, 520), (768, 136, 256)]


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("n", [1, 2, 17, 64, 65, 200, 257, 700])
def test_sizes(n, sizes, kind):
    args = data(n, *sizes, seed=n)
    check(kernels(*args, kind), exact(*args, kind), bounds(*args, kind))


@pytest.mark.parametrize("n,d,f,kind", [(1000, 1000, 2664, "gelu"), (4097, 512, 1360, "silu"), (129, 768, 2048, "silu"),
                                        (5000, 264, 136, "silu"), (9001, 200, 2056, "gelu"), (2049, 1032, 520, "silu")])
def test_larger(n, d, f, kind):
    args = data(n, d, f, d)
    check(kernels(*args, kind), exact(*args, kind), bounds(*args, kind))


class Rounded(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.to(BF16).to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g.to(BF16).to(g.dtype)


@pytest.mark.parametrize("n,sizes,kind", [(300, (256, 344, 256), "silu"), (2000, (128, 512, 64), "gelu")])
def test_norms(n, sizes, kind):
    """The distance that the same roundings make in 64 bits, taken three times: two between kernels and that, one over."""

    args = data(n, *sizes)
    wanted = exact(*args, kind)
    leaves = [t.to(F64).requires_grad_() for t in args[:3]]
    r = Rounded.apply
    g, u = r(leaves[0] @ leaves[1]).chunk(2, -1)
    y = r(r(act(g, kind) * u) @ leaves[2])
    rounded = [y.detach(), *(r(t) for t in torch.autograd.grad(y, leaves, args[3].to(F64)))]
    for name, a, b, c in zip(NAMES, kernels(*args, kind), wanted, rounded):
        assert torch.linalg.norm(a.cpu().to(F64) - b) <= 3 * torch.linalg.norm(c - b), name


def test_large_gates():
    """Gates far on both sides: the activation's limits, no NaN."""

    x, w, v, dy = data(40, 64, 64, 64)
    for scale in (30.0, 1e4):
        args = ((x * scale).to(BF16), w, v, dy)
        for kind in ("silu", "gelu"):
            got = kernels(*args, kind)
            assert all(torch.isfinite(t).all() for t in got)
            check(got, exact(*args, kind), bounds(*args, kind))


def test_gradient_by_differences():
    """A change of all three along one direction, by differences of the formula."""

    args = data(50, 64, 72, 40, seed=3)
    g = torch.Generator().manual_seed(4)
    steps = [torch.randn(t.shape, generator=g, dtype=F64) for t in args[:3]]
    grads, limits = kernels(*args, "silu")[1:], bounds(*args, "silu")[1:]
    e = 1e-5
    ends = [(formula(*(t.to(F64) + s * e * step for t, step in zip(args, steps)), "silu") * args[3].to(F64)).sum()
            for s in (1, -1)]
    along = sum((a.cpu().to(F64) * s).sum() for a, s in zip(grads, steps))
    limit = sum((b * s.abs()).sum() for b, s in zip(limits, steps))
    assert abs((ends[0] - ends[1]) / (2 * e) - along) <= 1.1 * limit + 1e-6 * abs(along)


def test_shapes_and_strides():
    """Leading dimensions, slices of wider tensors, transposed and misaligned ones, a gradient that repeats a row."""

    x, w, v, dy = data(60, 64, 72, 40)
    wanted, limits = exact(x, w, v, dy, "silu"), bounds(x, w, v, dy, "silu")

    def inside(t, left, right):
        wide = torch.full((t.shape[0], left + t.shape[1] + right), float("nan"), dtype=BF16, device=DEV)
        wide[:, left:left + t.shape[1]] = t.to(DEV)
        return wide[:, left:left + t.shape[1]]

    for make in (lambda t: inside(t, 8, 16), lambda t: inside(t, 3, 2), lambda t: t.to(DEV).t().contiguous().t()):
        leaves = [make(t).detach().requires_grad_() for t in (x, w, v)]
        y = gated_mlp(leaves[0].view(60, 64), leaves[1], leaves[2])
        check([y.detach(), *torch.autograd.grad(y, leaves, make(dy))], wanted, limits)
    leaves = [x.to(DEV).view(3, 20, 64).requires_grad_(), w.to(DEV).requires_grad_(), v.to(DEV).requires_grad_()]
    y = gated_mlp(*leaves)
    assert y.shape == (3, 20, 40)
    row = dy[:1].expand(60, 40)
    got = [y.detach().view(60, 40), *torch.autograd.grad(y, leaves, row.to(DEV).view(3, 20, 40))]
    got[1] = got[1].view(60, 64)
    check(got, exact(x, w, v, row, "silu"), bounds(x, w, v, row, "silu"))
    one = gated_mlp(x.to(DEV)[7], w.to(DEV), v.to(DEV))
    assert one.shape == (40,)
    check([one[None]], [wanted[0][7:8]], [limits[0][7:8]])


def test_no_tokens():
    _, w, v, _ = data(1, 64, 72, 40)
    leaves = [torch.zeros((2, 0, 64), dtype=BF16, device=DEV, requires_grad=True), w.to(DEV).requires_grad_(),
              v.to(DEV).requires_grad_()]
    y = gated_mlp(*leaves)
    assert y.shape == (2, 0, 40)
    dx, dw, dv = torch.autograd.grad(y, leaves, torch.zeros_like(y))
    assert dx.shape == (2, 0, 64) and (dw == 0).all() and (dv == 0).all()


def test_each_gradient_alone():
    x, w, v, dy = (t.to(DEV) for t in data(70, 64, 72, 40))
    leaves = [t.clone().requires_grad_() for t in (x, w, v)]
    every = torch.autograd.grad(gated_mlp(*leaves), leaves, dy)
    for i in range(3):
        alone = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, v))]
        (grad,) = torch.autograd.grad(gated_mlp(*alone), alone[i], dy)
        assert torch.equal(grad, every[i])
    with torch.no_grad():
        assert torch.equal(gated_mlp(*leaves), gated_mlp(x, w, v))


def test_a_token_is_its_own():
    """NaN in one token's row stays in that token's rows; rows of other tokens keep their bits."""

    for n in (40, 700):
        x, w, v, dy = (t.to(DEV) for t in data(n, 64, 72, 40))
        clean = gated_mlp(x, w, v)
        x[n // 2] = float("nan")
        leaf = x.clone().requires_grad_()
        y = gated_mlp(leaf, w, v)
        (dx,) = torch.autograd.grad(y, leaf, dy)
        others = torch.arange(n, device=DEV) != n // 2
        assert torch.equal(y[others], clean[others]) and torch.isnan(y[n // 2]).all()
        assert torch.isfinite(dx[others]).all()


def test_same_bits():
    for n in (5000, 64):
        args = data(n, 256, 264, 128)
        first = kernels(*args, "silu")
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, kernels(*args, "silu")))


@pytest.mark.parametrize("n", [33, 900])
def test_captured_and_replayed(n):
    x, w, v, dy = (t.to(DEV) for t in data(n, 128, 136, 128))
    side = torch.cuda.Stream()
    leaves = [t.clone().requires_grad_() for t in (x, w, v)]

    def step():
        y = gated_mlp(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    for seed in range(3):
        args = data(n, 128, 136, 128, seed=seed + 5)
        with torch.no_grad():
            for leaf, t in zip((*leaves, dy), args):
                leaf.copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = kernels(*args, "silu")
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_second_derivatives_are_refused():
    x, w, v, dy = (t.to(DEV) for t in data(10, 64, 72, 40))
    x.requires_grad_()
    (grad,) = torch.autograd.grad(gated_mlp(x, w, v), x, dy.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()
