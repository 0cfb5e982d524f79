"""8-bit moments of ``gptrig.optim.adamw_tensors`` in captured graphs, whose replays read the seed on the device."""

from __future__ import annotations

import math

import pytest
import torch

from gptrig.optim import adamw_tensors

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F64, F8 = torch.float32, torch.float64, torch.float8_e4m3fn
B1, B2 = 0.9, 0.95


def lists(bits=8, sizes=(5000, 1001), seed=0):
    g = torch.Generator().manual_seed(seed)
    normal = lambda n, scale: torch.randn(n, generator=g) * scale  # noqa: E731
    out = dict(params=[normal(n, 1.0) for n in sizes], grads=[normal(n, 0.1) for n in sizes])
    if bits == 32:
        out.update(exp_avg=[normal(n, 0.1) for n in sizes], exp_avg_sq=[normal(n, 0.1).square() for n in sizes])
    else:
        blocks = [-(-n // 256) for n in sizes]
        out.update(exp_avg=[normal(n, 60.0).clamp(-448, 448).to(F8) for n in sizes],
                   exp_avg_sq=[normal(n, 60.0).abs().clamp(1, 448).to(F8) for n in sizes],
                   exp_avg_scale=[torch.rand(b, generator=g) * 1e-3 + 1e-3 for b in blocks],
                   exp_avg_sq_scale=[torch.rand(b, generator=g) * 1e-4 + 1e-4 for b in blocks])
    out = {k: [t.to(DEV) for t in v] for k, v in out.items()}
    out["hparams"] = torch.tensor([[1.0, 1e-8, 0.1]] * len(sizes), device=DEV)
    return out


def everything(state):
    return [t.view(torch.uint8) if t.dtype == F8 else t for k, v in state.items() if k not in ("grads", "hparams") for t in v]


def step(state, seed, number=4):
    adamw_tensors(**state, lr=0.01, beta1=B1, beta2=B2, step=number, seed=seed)


@pytest.mark.parametrize("bits", [8, 32])
def test_replays_read_the_seed(bits):
    """A graph that counts its seed up gives the bits of eager steps with those seeds, also past 2^32 and below 0."""

    a, b = lists(bits), lists(bits)
    seed = torch.tensor(0, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, seed)
        seed.add_(1)
    for first in (7, 2 ** 32 - 2, -2):
        seed.fill_(first)
        for k in range(4):
            print(f"adamw_tensors, seed on the device {first} + {k}, {bits} bits", flush=True)
            graph.replay()
            torch.cuda.synchronize()
            step(b, (first + k) % 2 ** 32)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(everything(a), everything(b))), (first, k)
    assert int(seed) == -2 + 4


def test_an_eager_call_takes_either():
    a, b = lists(), lists()
    step(a, torch.tensor([2 ** 32 + 12345], device=DEV))
    step(b, 12345)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(everything(a), everything(b)))


def test_moments_decay_over_replays():
    """Blocks whose largest v is held up by a gradient of its own (v = g^2), all others at 8 of 448 without a gradient:
    after n replays they are 8 b2^n on average.  A rounding's deviation is at most half a step, 1/4 from 4 on and 1/8
    below, so six deviations of the mean are at most 6 sqrt(n) / 4 / sqrt(elements).  (With one u for all replays the
    elements with u >= 0.4 stay at 8, and the mean is above 4.8.)"""

    blocks, n = 16, 20
    state = lists(sizes=(256 * blocks,))
    top = 0.5
    g, codes = torch.zeros(256 * blocks, device=DEV), torch.full((256 * blocks,), 8.0, device=DEV)
    g[::256], codes[::256] = top, 448.0
    state["grads"][0].copy_(g)
    state["exp_avg_sq"][0].copy_(codes.to(F8))
    state["exp_avg_sq_scale"][0].fill_(top * top / 448)
    seed = torch.tensor(3, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(state, seed)
        seed.add_(1)
    for _ in range(n):
        graph.replay()
    torch.cuda.synchronize()
    v = (state["exp_avg_sq"][0].to(F64).view(blocks, 256) * state["exp_avg_sq_scale"][0].to(F64)[:, None])[:, 1:]
    mean = float(v.mean()) / (top * top / 448)
    assert abs(mean - 8 * B2 ** n) <= 6 * math.sqrt(n) / 4 / math.sqrt(255 * blocks) + 1e-4, mean


def test_a_captured_number_is_warned_of():
    state = lists()
    with pytest.warns(UserWarning, match="every replay rounds"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step(state, 5)
