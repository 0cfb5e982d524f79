"""LayerNorm, the scored attention and AdamW over a list of tensors as a training step of one block uses them.

The block is computed a second time in 64 bits, as it is and with a rounding to
bfloat16, of the value and of its gradient, wherever the step holds one in
bfloat16.  The distance between those two is what the types lose whatever the
order of the roundings; the kernels' own differ from it in their errors, not in
their number or size, so that two such distances lie between them and the exact
result (a triangle through the exact one) and a third covers P, dU and the
gradient of the projections' products, which the kernels round inside.
"""

from __future__ import annotations

import pytest
import torch

from gptrig.kernels import ScoredAttentionConfig, make_scored_attention
from gptrig.nn import layer_norm
from gptrig.optim import adamw_tensors, adamw_tensors_state

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
CAP = 20.0
NAMES = ("norm_scale", "norm_bias", "qkv_w", "out_w", "final_scale")
HPARAMS = ((1.0, 1e-8, 0.0), (1.0, 1e-8, 0.0), (0.5, 1e-8, 0.1), (0.5, 1e-9, 0.1), (2.0, 1e-8, 0.0))


class Rounded(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.to(BF16).to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g.to(BF16).to(g.dtype)


def block(w, x, seg, prefix, slopes, heads, kv_heads):
    """The step's forward pass on the kernels: float32 parameters, bfloat16 activations."""

    B, S, width = x.shape
    dim = width // heads
    h = layer_norm(x, w["norm_scale"], w["norm_bias"])
    qkv = torch.mm(h.view(B * S, width), w["qkv_w"].to(BF16)).view(B, S, heads + 2 * kv_heads, dim).transpose(1, 2)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
    o = make_scored_attention(ScoredAttentionConfig(score_cap=CAP))(q, k, v, seg, prefix_lengths=prefix,
                                                                    distance_slopes=slopes)
    y = x + torch.mm(o.transpose(1, 2).reshape(B * S, width), w["out_w"].to(BF16)).view(B, S, width)
    return layer_norm(y, w["final_scale"], eps=1e-6)


def plain_norm(x, scale, bias, eps):
    x = x - x.mean(-1, keepdim=True)
    y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * scale
    return y if bias is None else y + bias


def plain_block(w, x, seg, prefix, slopes, heads, kv_heads, r):
    """The same from the formulas in 64 bits, on the CPU; r: what happens to a value that the step rounds."""

    B, S, width = x.shape
    dim = width // heads
    h = r(plain_norm(x, w["norm_scale"], w["norm_bias"], 1e-5))
    qkv = r(h @ r(w["qkv_w"])).view(B, S, heads + 2 * kv_heads, dim).transpose(1, 2)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
    k, v = (t.repeat_interleave(heads // kv_heads, 1) for t in (k, v))
    i = torch.arange(S)
    apart = (i[:, None] - i[None, :]).abs()
    visible = (i[None, :] <= i[:, None]) | (i < prefix[:, None, None])
    visible = (visible & (seg[:, :, None] == seg[:, None, :]))[:, None]
    s = CAP * torch.tanh(q @ k.transpose(-1, -2) * dim ** -0.5 / CAP) - slopes[:, None, None] * apart
    o = r(torch.softmax(s.masked_fill(~visible, -torch.inf), -1) @ v)
    y = r(x + r(o.transpose(1, 2).reshape(B, S, width) @ r(w["out_w"])))
    return r(plain_norm(y, w["final_scale"], None, 1e-6))


def setup(seed=0, B=2, S=150, heads=6, kv_heads=2, dim=64):
    g = torch.Generator().manual_seed(seed)
    width = heads * dim
    normal = lambda *shape: torch.randn(shape, generator=g)
    w = dict(norm_scale=1 + 0.2 * normal(width), norm_bias=0.2 * normal(width),
             qkv_w=normal(width, (heads + 2 * kv_heads) * dim) * 1.5 * width ** -0.5,
             out_w=normal(width, width) * width ** -0.5, final_scale=1 + 0.2 * normal(width))
    x, target = normal(B, S, width).to(BF16), normal(B, S, width).to(BF16)
    seg = torch.cumsum(torch.rand((B, S), generator=g) < 0.02, 1).to(torch.int32)
    data = (x, seg, torch.tensor([40, 0], dtype=torch.int32), 2.0 ** -torch.arange(1.0, heads + 1))
    return w, data, target, (heads, kv_heads)


def gradients(w, data, target, sizes):
    w = {n: t.to(DEV).requires_grad_() for n, t in w.items()}
    out = block(w, *(t.to(DEV) for t in data), *sizes)
    return [out.detach(), *torch.autograd.grad(out, list(w.values()), target.to(DEV))]


def plain_gradients(w, data, target, sizes, r):
    w = {n: t.to(F64).requires_grad_() for n, t in w.items()}
    x, seg, prefix, slopes = data
    out = plain_block(w, x.to(F64), seg, prefix, slopes.to(F64), *sizes, r)
    return [out.detach(), *torch.autograd.grad(out, list(w.values()), target.to(F64))]


@pytest.mark.parametrize("sizes", [dict(), dict(B=1, S=67, heads=4, kv_heads=4, dim=32),
                                   dict(B=2, S=33, heads=2, kv_heads=1, dim=128)], ids=["64", "32", "128"])
def test_gradients(sizes):
    w, data, target, heads = setup(**sizes)
    data = (*data[:2], data[2][: data[0].shape[0]], data[3])
    got = gradients(w, data, target, heads)
    exact = plain_gradients(w, data, target, heads, lambda t: t)
    rounded = plain_gradients(w, data, target, heads, Rounded.apply)
    for name, a, b, c in zip(("out", *NAMES), got, exact, rounded):
        loss, off = torch.linalg.norm(c - b).item(), torch.linalg.norm(a.to("cpu", F64) - b).item()
        assert off <= 3 * loss, (name, off / torch.linalg.norm(b).item(), loss / torch.linalg.norm(b).item())


def values(state, i):
    """The moments of tensor i as float64 values."""

    out = []
    for name in ("exp_avg", "exp_avg_sq"):
        codes = state[name][i].to(F32).to(F64)
        if name + "_scale" in state:
            codes = codes * state[name + "_scale"][i].to(F64).repeat_interleave(256)[: codes.numel()].view(codes.shape)
        out.append(codes)
    return out


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(bits):
    """Three steps, each parameter against the formula on the step's own gradients and the moments before it."""

    w, data, target, heads = setup(seed=1)
    params = [t.to(DEV) for t in w.values()]
    state = adamw_tensors_state(params, bits)
    rows = torch.tensor(HPARAMS, device=DEV)
    lr, b1, b2 = 0.01, 0.9, 0.95
    for step in range(1, 4):
        grads = gradients(dict(zip(NAMES, params)), data, target, heads)[1:]
        before = [(p.to(F64), *values(state, i)) for i, p in enumerate(params)]
        adamw_tensors(params, grads, hparams=rows, lr=lr, beta1=b1, beta2=b2, step=step, **state)
        for p, g, (p0, m0, v0), row, name in zip(params, grads, before, rows.to(F64), NAMES):
            mult, eps, decay = row
            g = g.to(F64)
            root = ((b2 * v0 + (1 - b2) * g * g) / (1 - b2 ** step)).sqrt() + eps
            size = (b1 * m0 + (1 - b1) * g) / (1 - b1 ** step) / root
            want = p0 - lr * mult * (size + decay * p0)
            # 16 roundings of 2^-24 of the terms that the step adds up, one of the parameter.
            most = (b1 * m0.abs() + (1 - b1) * g.abs()) / (1 - b1 ** step) / root + decay * p0.abs()
            off = 2.0 ** -24 * (16 * lr * mult * most + want.abs())
            assert ((p.to(F64) - want).abs() <= off).all(), (step, name)


def test_captured_step():
    """Forward, backward and the update in one graph: every replay gives the eager step's bits."""

    w, data, target, heads = setup(seed=2)
    data, target = tuple(t.to(DEV) for t in data), target.to(DEV)
    rows = torch.tensor(HPARAMS, device=DEV)

    def step(params, state):
        out = block(dict(zip(NAMES, params)), *data, *heads)
        grads = torch.autograd.grad(out, params, target)
        with torch.no_grad():
            adamw_tensors([p.detach() for p in params], grads, hparams=rows, lr=0.01, beta1=0.9, beta2=0.95, step=7,
                          **state)

    def fresh():
        params = [t.to(DEV).requires_grad_() for t in w.values()]
        return params, adamw_tensors_state(params, 8)

    eager, eager_state = fresh()
    step(eager, eager_state)
    torch.cuda.synchronize()
    first = [p.detach().clone() for p in eager]
    step(eager, eager_state)
    torch.cuda.synchronize()
    params, state = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(params, state)
    for wanted in (first, eager):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(params, wanted))
