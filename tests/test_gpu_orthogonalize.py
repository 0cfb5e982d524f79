"""``optim.orthogonalize_tensors`` against its formula in 64 bits on the CPU.

``stepped`` computes it a second time in 64 bits with the kernels' roundings: the operands, A and B (without their
diagonals) to float16, the rest of X to float16 at 2^11 times its size, the result to bfloat16.  Its distance from the
exact result is what the types lose; the kernels' own roundings differ from its in their errors, not in their number or
size, so two such distances lie between them, and a third over for the float32 sums.  A single value may be eight times the root mean square off (as far
as a sum of many roundings hardly ever gets), and half a step of bfloat16 of its own.
"""

from __future__ import annotations

import pytest
import torch

from gptrig.optim import orthogonalize_tensors

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
MUON = (3.4445, -4.7750, 2.0315)


def matrix(rows, cols, fall=0.0, seed=0, dtype=F32):
    """Singular values 1, ..., 10^-fall (fall 0: a normal matrix's)."""

    g = torch.Generator().manual_seed(seed)
    u = torch.randn((rows, cols), generator=g, dtype=F64)
    if fall:
        a, _, b = torch.linalg.svd(u, full_matrices=False)
        u = (a * 10.0 ** torch.linspace(0, -fall, min(rows, cols), dtype=F64)) @ b
    return u.to(dtype)


def stepped(u, steps=5, coefficients=MUON, eps=1e-7, rounded=False):
    a, b, c = coefficients
    r = (lambda t: t.to(F32).to(F16).to(F64)) if rounded else (lambda t: t)
    x = u.to(F64)
    x = x / (torch.linalg.norm(x) + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    hi, lo = r(x), r((x - r(x)) * 2048)
    for _ in range(steps):
        gram = hi @ hi.T
        d = gram.diagonal()
        o = r(gram - torch.diag(d))
        square = o @ o
        rest = (b + c * (d[:, None] + d)) * o + c * square
        more = a + b * d + c * (d * d + square.diagonal())
        x = more[:, None] * (hi + lo / 2048) + r(rest - torch.diag(rest.diagonal())) @ hi
        hi, lo = r(x), r((x - r(x)) * 2048)
    x = x.T if tall else x
    return x.to(F32).to(BF16).to(F64) if rounded else x


def check(got, u, **how):
    assert got.dtype == BF16 and got.shape == u.shape and got.is_contiguous()
    flat, got = u.reshape(-1, *u.shape[-2:]), got.cpu().to(F64).reshape(-1, *u.shape[-2:])
    for g, one in zip(got, flat):
        exact, rounded = stepped(one, **how), stepped(one, rounded=True, **how)
        loss = torch.linalg.norm(rounded - exact)
        assert torch.linalg.norm(g - exact) <= 3 * loss, (u.shape, torch.linalg.norm(g - exact) / loss)
        each = 8 * loss / exact.numel() ** 0.5 + 2.0 ** -8 * exact.abs()
        assert ((g - exact).abs() <= each).all(), (u.shape, ((g - exact).abs() / each).max())


def one(u, **how):
    return orthogonalize_tensors([u.to(DEV)], **how)[0]


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (7, 1), (2, 2), (5, 3), (8, 8), (9, 8), (31, 33), (64, 64),
                                       (64, 65), (65, 130), (128, 128), (130, 129), (1, 3000), (3, 700), (200, 1000),
                                       (1000, 96), (509, 701), (640, 640)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sizes(rows, cols, dtype):
    u = matrix(rows, cols, seed=rows + cols, dtype=dtype)
    check(one(u), u)


@pytest.mark.parametrize("fall", [1.0, 3.0, 6.0])
@pytest.mark.parametrize("rows,cols", [(128, 200), (300, 257)])
def test_falling_singular_values(rows, cols, fall):
    u = matrix(rows, cols, fall)
    check(one(u), u)


def test_low_rank():
    g = torch.Generator().manual_seed(1)
    u = torch.randn((150, 5), generator=g) @ torch.randn((5, 260), generator=g)
    check(one(u), u)


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e30, 3e37])
def test_scales(scale):
    """Squares of these pass float32 on either side; eps counts where the norm is near it."""

    u = matrix(40, 70) * scale
    check(one(u, eps=0.0), u, eps=0.0)
    check(one(u), u)


@pytest.mark.parametrize("shape", [(40, 72), (72, 40), (7, 9)])
def test_a_power_of_two_changes_nothing(shape):
    """Without eps: from multiples of the smallest float32 (the norm's inverse is none then) to its largest (the norm
    itself is none)."""

    g = torch.Generator().manual_seed(5)
    u = torch.randint(-127, 128, shape, generator=g).to(F32)
    want = one(u, eps=0.0)
    check(want, u, eps=0.0)
    for power in (-149, -130, 121):
        scaled = torch.ldexp(u.to(F64), torch.tensor(power)).to(F32)
        assert torch.equal(torch.ldexp(scaled.to(F64), torch.tensor(-power)), u.to(F64))
        assert torch.equal(one(scaled, eps=0.0), want), power


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_steps(steps):
    u = matrix(90, 140, 2.0)
    check(one(u, steps=steps), u, steps=steps)


def test_other_coefficients():
    """The cubic iteration, which converges: all singular values 1, to the operands' 11 bits."""

    how = dict(steps=14, coefficients=(1.5, -0.5, 0.0))
    u = matrix(96, 200, 1.0)
    got = one(u, **how)
    check(got, u, **how)
    values = torch.linalg.svdvals(got.cpu().to(F64))
    assert (values - 1).abs().max() < 0.01


def test_lists():
    """More tensors than a launch takes, of more shapes, with leading dimensions and empty ones between."""

    shapes = [(17 + i, 40 - i) for i in range(20)] + [(33, 20)] * 50 + [(2, 3, 24, 50), (0, 8, 8), (4, 50, 24), (5, 0),
                                                                        (0, 3), (24, 50)]
    updates = [torch.randn(s, generator=torch.Generator().manual_seed(i)) for i, s in enumerate(shapes)]
    got = orthogonalize_tensors([u.to(DEV) for u in updates])
    assert len(got) == len(updates)
    for a, u in zip(got, updates):
        if u.numel():
            check(a, u)
        else:
            assert a.shape == u.shape
    assert orthogonalize_tensors([]) == []
    assert orthogonalize_tensors([torch.zeros((0, 4), device=DEV)])[0].shape == (0, 4)


def test_wide_tiles():
    """Enough tiles of 128 x 128 that those are taken, with edges inside them."""

    updates = [matrix(200, 457, seed=i) for i in range(30)] + [matrix(331, 259, seed=50 + i) for i in range(24)]
    got = orthogonalize_tensors([u.to(DEV) for u in updates])
    for i in (0, 7, 29, 30, 41, 53):
        check(got[i], updates[i])
    alone = orthogonalize_tensors([updates[7].to(DEV)])[0]
    check(alone, updates[7])


def test_a_matrix_is_its_own():
    """Zeros stay zeros; a NaN or an infinity spoils its own matrix only."""

    g = torch.Generator().manual_seed(2)
    u = torch.randn((5, 70, 50), generator=g)
    clean = one(u)
    u[1] = 0
    u[3, 4, 5] = float("nan")
    u[4, 69, 49] = float("inf")
    got = one(u)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    assert (got[1] == 0).all()
    assert torch.isnan(got[3]).all() and torch.isnan(got[4]).any()


def test_strides():
    g = torch.Generator().manual_seed(3)
    wide = torch.randn((60, 4, 101), generator=g).to(DEV)
    for view in (wide[:, 1, 3:50], wide[:, 2, ::2], wide[:, 0].t(), wide.transpose(0, 1), wide[::3, :, 7:8]):
        (got,) = orthogonalize_tensors([view])
        assert torch.equal(got, orthogonalize_tensors([view.contiguous()])[0])
        check(got, view.cpu())


def test_inputs_stay():
    u = matrix(64, 80).to(DEV)
    before = u.clone()
    orthogonalize_tensors([u, u])
    assert torch.equal(u, before)


def test_same_bits():
    updates = [matrix(120, 300, seed=i).to(DEV) for i in range(3)]
    first = orthogonalize_tensors(updates)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, orthogonalize_tensors(updates)))


def test_captured_and_replayed():
    updates = [matrix(70, 100).to(DEV), matrix(3, 40).view(1, 3, 40).to(DEV)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        orthogonalize_tensors(updates)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = orthogonalize_tensors(updates)
    for seed in range(3):
        for i, u in enumerate(updates):
            u.copy_(matrix(*u.shape[-2:], seed=10 * seed + i))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, orthogonalize_tensors(updates)))
        check(got[0], updates[0].cpu())
