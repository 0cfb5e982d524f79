"""The token embedding, the gated block and the orthogonalised updates in a training step of a small model, next to the
operators that such a step takes beside them: layer_norm, the tiled loss and adamw_tensors.

As in the test of a block's step, the model is computed a second time in 64 bits, as it is and with a rounding wherever
the step holds a value or a gradient in bfloat16; three distances between those two bound the step's own (two by a
triangle through the exact result, one for what the kernels round inside).
"""

from __future__ import annotations

import math

import pytest
import torch

from gptrig.kernels import tiled_tied_cross_entropy
from gptrig.nn import embedding, gated_mlp, layer_norm
from gptrig.optim import adamw_tensors, adamw_tensors_state, orthogonalize_tensors

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
NAMES = ("table", "norm_scale", "gate_up_w", "down_w", "final_scale")
ORTHOGONAL = (2, 3)  # the matrices of the block, by their place in NAMES


class Rounded(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.to(BF16).to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g.to(BF16).to(g.dtype)


def setup(seed=0, tokens=300, width=128, hidden=344, vocab=500):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g)  # noqa: E731
    w = dict(table=normal(vocab, width) * width ** -0.5, norm_scale=1 + 0.2 * normal(width),
             gate_up_w=normal(width, 2 * hidden) * width ** -0.5, down_w=normal(hidden, width) * hidden ** -0.5,
             final_scale=1 + 0.2 * normal(width))
    ids = (torch.exp(torch.rand(tokens, generator=g) * math.log(vocab + 1)) - 1).floor().clamp(0, vocab - 1).int()
    ids[-20:] = -1  # padding
    targets = torch.randint(0, vocab, (tokens,), generator=g, dtype=torch.int32)
    return w, ids, targets


def loss(w, ids, targets, width=128):
    x = embedding(ids, w["table"], scale=math.sqrt(width))
    x = x + gated_mlp(layer_norm(x, w["norm_scale"]), w["gate_up_w"].to(BF16), w["down_w"].to(BF16))
    return tiled_tied_cross_entropy(layer_norm(x, w["final_scale"]), w["table"], targets,
                                    semantic_vocab_size=w["table"].shape[0])


def plain_norm(x, scale):
    x = x - x.mean(-1, keepdim=True)
    return x * (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * scale


def plain_loss(w, ids, targets, r, width=128):
    inside = (ids >= 0)[:, None]
    x = r(w["table"][ids.long().clamp(min=0)] * inside * math.sqrt(width))
    g, u = (r(plain_norm(x, w["norm_scale"])) @ r(w["gate_up_w"])).chunk(2, -1)
    x = r(x + r(r(torch.nn.functional.silu(g) * u) @ r(w["down_w"])))
    logits = r(plain_norm(x, w["final_scale"])) @ r(w["table"]).T
    return torch.nn.functional.cross_entropy(logits, targets.long())


def gradients(w, ids, targets):
    leaves = {n: t.to(DEV).requires_grad_() for n, t in w.items()}
    out = loss(leaves, ids.to(DEV), targets.to(DEV))
    return [out.detach(), *torch.autograd.grad(out, list(leaves.values()))]


def plain_gradients(w, ids, targets, r):
    leaves = {n: t.to(F64).requires_grad_() for n, t in w.items()}
    out = plain_loss(leaves, ids, targets, r)
    return [out.detach(), *torch.autograd.grad(out, list(leaves.values()))]


def test_gradients():
    w, ids, targets = setup()
    exact = plain_gradients(w, ids, targets, lambda t: t)
    rounded = plain_gradients(w, ids, targets, Rounded.apply)
    got = gradients(w, ids, targets)
    # (The loss is one number, whose rounded form may come near by chance: a rounding of 2^-8 of it.)
    assert abs(got[0].item() - exact[0].item()) <= 2.0 ** -8 * exact[0].item()
    for name, a, b, c in zip(NAMES, got[1:], exact[1:], rounded[1:]):
        off, lost = torch.linalg.norm(a.cpu().to(F64) - b), torch.linalg.norm(c - b)
        assert off <= 3 * lost, (name, (off / lost).item())


def step(params, momenta, state, hparams, ids, targets, number):
    """Momenta of all matrices of the block, orthogonalised; the rest by AdamW."""

    out = loss(dict(zip(NAMES, params)), ids, targets)
    grads = torch.autograd.grad(out, params)
    with torch.no_grad():
        for m, i in zip(momenta, ORTHOGONAL):
            m.mul_(0.95).add_(grads[i])
        updates = orthogonalize_tensors(momenta)
        for u, i in zip(updates, ORTHOGONAL):
            params[i].add_(u, alpha=-0.02)
        rest = [i for i in range(len(params)) if i not in ORTHOGONAL]
        adamw_tensors([params[i].detach() for i in rest], [grads[i] for i in rest], hparams=hparams, lr=0.01, beta1=0.9,
                      beta2=0.95, step=number, **state)
    return out.detach(), updates


def fresh(w):
    params = [t.to(DEV).requires_grad_() for t in w.values()]
    momenta = [torch.zeros_like(params[i]).detach() for i in ORTHOGONAL]
    state = adamw_tensors_state([p.detach() for i, p in enumerate(params) if i not in ORTHOGONAL])
    return params, momenta, state, torch.tensor([[1.0, 1e-8, 0.1], [1.0, 1e-8, 0.0], [1.0, 1e-8, 0.0]], device=DEV)


def test_training_steps():
    """Three steps: the updates of the momenta are near orthogonal, the same from the same, and every parameter moves."""

    w, ids, targets = setup(seed=1)
    every = []
    for _ in range(2):
        run = fresh(w)
        for number in range(1, 4):
            out, updates = step(*run, ids.to(DEV), targets.to(DEV), number)
            assert torch.isfinite(out)
            for u, m in zip(updates, run[1]):
                # Five steps leave singular values that were not tiny between 0.6 and 1.3: so the root mean square.
                size = torch.linalg.norm(u.to(F64)) / min(u.shape) ** 0.5
                assert u.shape == m.shape and 0.3 < size < 1.3
        every.append([p.detach().clone() for p in run[0]])
    assert all(not torch.equal(p.cpu(), q) for p, q in zip(every[0], w.values()))


def test_captured_step():
    """The step in one graph, replayed: the eager steps' bits wherever the step adds in a fixed order (the tiled loss
    adds its gradients of the hidden values and of the table so too at this size)."""

    w, ids, targets = setup(seed=2)
    ids, targets = ids.to(DEV), targets.to(DEV)
    eager, first = fresh(w), None
    losses = []
    for k in range(2):
        out, _ = step(*eager, ids, targets, 5)
        torch.cuda.synchronize()
        losses.append(out.item())
        first = [p.detach().clone() for p in eager[0]] if k == 0 else first
    second = [p.detach().clone() for p in eager[0]]
    del eager, out
    run = fresh(w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, _ = step(*run, ids, targets, 5)
    for wanted, value in zip((first, second), losses):
        graph.replay()
        torch.cuda.synchronize()
        assert out.item() == value
        assert all(torch.equal(a.detach(), b) for a, b in zip(run[0], wanted))
