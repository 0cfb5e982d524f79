"""``gptrig.nn.layer_norm`` against the formula in 64 bits.

Tolerances, derived from the arithmetic: an output is rounded once to its type
(half a step, ``eps / 2`` of its value), after a float32 computation whose sums
over n terms are off by at most ``(chain + 32) 2^-24`` of the sum of magnitudes,
chain <= n / 32 + 64 being the longest run of additions (32 lanes or more share a
row, 32 or more sequences share the rows).
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def inputs(shape, dtype, params, bias, seed=0):
    g = torch.Generator().manual_seed(seed)
    d = shape[-1]
    x = (torch.randn(shape, generator=g) + torch.randn((*shape[:-1], 1), generator=g)).to(dtype)
    scale = (1 + 0.3 * torch.randn(d, generator=g)).to(params)
    b = torch.randn(d, generator=g).to(params) if bias else None
    dy = torch.randn(shape, generator=g).to(dtype)
    return tuple(None if t is None else t.to(DEV) for t in (x, scale, b, dy))


def reference(x, scale, b, dy, eps=1e-5):
    """y, dx, dscale, dbias and the bounds of each, in 64 bits."""

    d = x.shape[-1]
    x, s, dy = (t.to(F64).reshape(-1, d) if t.ndim != 1 or t is x else t.to(F64) for t in (x, scale, dy))
    dtype_rows = x.shape[0]
    mu = x.mean(1, keepdim=True)
    c = x - mu
    r = (c.square().mean(1, keepdim=True) + eps).rsqrt()
    h = c * r
    y = h * s + (0 if b is None else b.to(F64))
    g = dy * s
    a1, b1 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = r * (g - a1 - h * b1)
    k = (d / 32 + 96) * U  # of a row's sums
    size = x.abs().mean(1, keepdim=True) + x.abs()
    dh = k * (r * size + 2 * h.abs())  # the float32 error of h
    bounds = {
        "y": dh * s.abs() + 2 * U * (h * s).abs() + 2 * U * y.abs(),
        "dx": r * (k * (g.abs() + g.abs().mean(1, keepdim=True) + 4 * h.abs() * (g * h).abs().mean(1, keepdim=True))
                   + dh * b1.abs() + h.abs() * (g.abs() * dh).mean(1, keepdim=True)) + 4 * k * dx.abs(),
        "dscale": (dtype_rows / 32 + 96) * U * (dy * h).abs().sum(0) + (dy.abs() * dh).sum(0),
        "dbias": (dtype_rows / 32 + 96) * U * dy.abs().sum(0),
    }
    return {"y": y, "dx": dx, "dscale": (dy * h).sum(0), "dbias": dy.sum(0)}, bounds


def check(name, got, want, bound):
    want = want.reshape(got.shape)
    bound = bound.reshape(got.shape)
    bound = bound + half_step(got.dtype) * (want.abs() + bound) + torch.finfo(got.dtype).tiny
    off = (got.to(F64) - want).abs() - bound
    assert bool((off <= 0).all()), f"{name}: {float(off.max())} past its bound, {int((off > 0).sum())} values"


def compare(x, scale, b, dy):
    from gptrig.nn import layer_norm

    leaves = [t.detach().requires_grad_() for t in (x, scale, b) if t is not None]
    y = layer_norm(leaves[0], leaves[1], leaves[2] if b is not None else None)
    grads = torch.autograd.grad(y, leaves, dy)
    torch.cuda.synchronize()
    assert y.shape == x.shape and y.dtype == x.dtype
    want, bounds = reference(x, scale, b, dy)
    check("y", y.detach(), want["y"], bounds["y"])
    for name, got in zip(("dx", "dscale", "dbias"), grads):
        assert got.dtype == (x.dtype if name == "dx" else scale.dtype)
        check(name, got, want[name], bounds[name])


SHAPES = [(1, 1), (3, 2), (5, 7), (1, 768), (129, 768), (64, 100), (33, 250), (17, 1000), (9, 1001), (2, 3, 512), (7, 1025),
          (11, 2047), (5, 2049), (6, 4096), (3, 5000), (4, 8191), (3, 8192), (3, 8193), (2, 20000)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_matches_the_formula(shape, dtype):
    print(f"layer_norm {shape} {dtype}", flush=True)
    for params, bias in ((F32, True), (BF16, False)):
        compare(*inputs(shape, dtype, params, bias))


@pytest.mark.parametrize("rows,width,dtype", [(65536, 768, BF16), (20001, 1536, BF16), (8191, 1001, F32), (300, 9000, BF16)])
def test_many_rows(rows, width, dtype):
    print(f"layer_norm rows={rows} width={width} {dtype}", flush=True)
    compare(*inputs((rows, width), dtype, F32, True, seed=1))


@pytest.mark.parametrize("rows,width", [((1 << 25) + 9, 8), ((1 << 22) + 3, 5)])
def test_more_rows_than_a_launch_has_workgroups_for(rows, width):
    from gptrig.nn import layer_norm

    print(f"layer_norm rows={rows} width={width}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn((rows, width), generator=g, device=DEV).to(BF16)
    scale, b = torch.randn(width, generator=g, device=DEV), torch.randn(width, generator=g, device=DEV)
    leaf = x.requires_grad_()
    y = layer_norm(leaf, scale, b)
    dx, = torch.autograd.grad(y, leaf, y.detach())
    torch.cuda.synchronize()
    middle = rows - rows % (1 << 22)  # where a launch ends
    for part in (slice(0, 9), slice(middle - 9, middle + 9), slice(rows - 9, rows)):
        want, bounds = reference(x.detach()[part], scale, b, y.detach()[part])
        check("y", y.detach()[part], want["y"], bounds["y"])
        check("dx", dx[part], want["dx"], bounds["dx"])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_strides_and_alignment(dtype):
    """Rows of a wider buffer, an odd start, a transposed view, a repeated row and an expanded gradient."""

    from gptrig.nn import layer_norm

    wide = torch.randn((40, 3 * 200 + 1), device=DEV).to(dtype)
    scale, bias = torch.randn(200, device=DEV), torch.randn(200, device=DEV)
    for x in (wide[:, 200:400], wide[:, 1:201], wide[:, :200].t()[:, :].t(), wide[:1, 3:203].expand(40, 200),
              wide[:, :200].reshape(40, 10, 20).transpose(1, 2).reshape(40, 200), wide.t()[:200].t()):
        want = layer_norm(x.contiguous().clone(), scale, bias)
        assert torch.equal(layer_norm(x, scale, bias), want)
    x = wide[:, :200].detach().requires_grad_()
    layer_norm(x, scale, bias).sum().backward()
    z = wide[:, :200].contiguous().clone().requires_grad_()
    layer_norm(z, scale, bias).backward(torch.ones_like(z))
    assert torch.equal(x.grad, z.grad)
    odd = torch.randn(401, device=DEV)
    assert torch.equal(layer_norm(z, odd[1:201], odd[201:]), layer_norm(z, odd[1:201].clone(), odd[201:].clone()))


def test_no_rows_and_partial_gradients():
    from gptrig.nn import layer_norm

    x = torch.empty((0, 64), dtype=BF16, device=DEV, requires_grad=True)
    scale, bias = (torch.ones(64, device=DEV, requires_grad=True) for _ in range(2))
    layer_norm(x, scale, bias).sum().backward()
    assert x.grad.shape == (0, 64) and not scale.grad.any() and not bias.grad.any()
    x, s, b, dy = inputs((70, 96), BF16, F32, True)
    full = [t.detach().requires_grad_() for t in (x, s, b)]
    want = torch.autograd.grad(layer_norm(*full), full, dy)
    for i in range(3):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, s, b))]
        assert torch.equal(torch.autograd.grad(layer_norm(*some), some[i], dy)[0], want[i])


def test_gradient_against_differences():
    from gptrig.nn import layer_norm

    x, s, b, dy = inputs((13, 200), F32, F32, True, seed=3)
    leaves = [t.detach().requires_grad_() for t in (x, s, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    g = torch.Generator(device=DEV).manual_seed(5)
    step = 1e-5  # the quotient's own error: step^2 times a third derivative of order 1
    for i, grad in enumerate(grads):
        way = torch.randn(grad.shape, generator=g, device=DEV, dtype=F64)
        moved = []
        for sign in (1, -1):
            at = [t.to(F64) + (sign * step * way if j == i else 0) for j, t in enumerate((x, s, b))]
            c = at[0] - at[0].mean(1, keepdim=True)
            y = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * at[1] + at[2]
            moved.append((y * dy.to(F64)).sum())
        want = float((moved[0] - moved[1]) / (2 * step))
        got = float((grad.to(F64) * way).sum())
        # 1000 times 2^-24 of the terms (the float32 bounds above), and the quotient's error.
        assert abs(got - want) <= 1000 * U * float((grad.to(F64) * way).abs().sum()) + 1e-6


def test_a_row_with_infinities_keeps_to_itself():
    from gptrig.nn import layer_norm

    x, s, b, dy = inputs((50, 768), BF16, F32, True)
    bad = x.clone()
    bad[7, 3], bad[20, 700], bad[49] = float("inf"), float("nan"), float("-inf")
    clean = [t.detach().requires_grad_() for t in (x, s, b)]
    dirty = [t.detach().requires_grad_() for t in (bad, s, b)]
    y, z = layer_norm(*clean), layer_norm(*dirty)
    keep = torch.ones(50, dtype=torch.bool, device=DEV)
    keep[[7, 20, 49]] = False
    assert torch.equal(y[keep], z[keep]) and z[~keep].isnan().all()
    dx = torch.autograd.grad(z, dirty[0], dy)[0]
    assert torch.equal(dx[keep], torch.autograd.grad(y, clean[0], dy)[0][keep])


def test_large_offset_is_centred_first():
    """Values around 1000 with a spread of 1: the squares are of the differences from the mean."""

    g = torch.Generator().manual_seed(9)
    x = (1000 + torch.randn((20, 512), generator=g)).to(DEV)
    compare(x, torch.ones(512, device=DEV), torch.zeros(512, device=DEV), torch.randn((20, 512), device=DEV))


def test_other_stream_repeats_and_captured_graph():
    from gptrig.nn import layer_norm

    x, s, b, dy = inputs((1000, 768), BF16, F32, True)
    leaves = [t.detach().requires_grad_() for t in (x, s, b)]
    y = layer_norm(*leaves)
    want = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    del y
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = layer_norm(*leaves)
        got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        del y
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(*leaves)
        out = [y, *torch.autograd.grad(y, leaves, dy)]
    for k in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.roll(x, k, 0))
        graph.replay()
        torch.cuda.synchronize()
        fresh = [t.detach().clone().requires_grad_() for t in leaves]
        y = layer_norm(*fresh)
        again = [y.detach(), *torch.autograd.grad(y, fresh, dy)]
        torch.cuda.synchronize()
        assert all(torch.equal(p.detach(), q) for p, q in zip(out, again)), k
