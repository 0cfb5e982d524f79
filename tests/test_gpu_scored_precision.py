"""What the scored attention keeps of ``o`` beyond its bfloat16, where the gradients hang on it.

All of a column's values are 1 or 1 + 2^-7 (or their negatives), neighbours in bfloat16, and the gradient of o has their
signs: dP - delta is then a hundredth of dP and of delta, and delta = o . do is wanted to far more than 8 bits.  Two
things of the forward serve it: o is divided by the sum of the same rounded P that its product took, so that their
roundings reach it by v - o and not by v; and 8 more bits of it go to the backward.  The bounds below count

  o:      2^-8 and the float32 error E of each P times |v - o|, 2^-18 for the float32 sums;
  delta:  that and 2^-15 of o (the kept bits stop at 2^-16, at the end of their range at 2^-15), 2^-24 a product;
  dU, dq, dk: delta's share, 2^-8 for the rounding of dU to bfloat16, the float32 errors of P and dP, their own rounding.

E, in a score, is (D + 16) 2^-24 of the magnitudes of its products, 2^-20 of the cap, 2^-22 of the bias and 2^-20 of its
exponential.  1 + 2^-6 stands for the products of two errors.  Each test also plants the two losses in the 64-bit
computation and finds them past the same bounds.
"""

from __future__ import annotations

import math

import pytest
import torch

from gptrig.kernels import ScoredAttentionConfig, make_scored_attention

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
R = 2.0 ** -8
MORE = 1 + 2.0 ** -6


def inputs(B, H, Hk, S, D, seed):
    g = torch.Generator().manual_seed(seed)
    sign = torch.where(torch.rand((1, 1, 1, D), generator=g) < 0.5, -1.0, 1.0)
    q = torch.randn((B, H, S, D), generator=g)
    k = 1 + 0.5 * torch.randn((B, Hk, S, D), generator=g)
    v = sign * (1 + 2.0 ** -7 * (torch.rand((B, Hk, S, D), generator=g) < 0.5))
    do = sign * torch.randn((B, H, S, D), generator=g).abs()
    return tuple(t.to(BF16).to(DEV) for t in (q, k, v, do))


class Exact:
    """The formula in 64 bits; ``gradients(o)``: with delta from this o."""

    def __init__(self, q, k, v, do, cap=None, slopes=None, seg=None, prefix=None):
        B, H, S, D = q.shape
        self.shape, self.join = (B, H, S, D), (B, k.shape[1], H // k.shape[1], S, D)
        self.scale = D ** -0.5
        self.q, self.do = q.to(F64), do.to(F64)
        self.k, self.v = (t.to(F64).repeat_interleave(H // k.shape[1], dim=1) for t in (k, v))
        mm = torch.matmul
        u = mm(self.q, self.t(self.k)) * self.scale
        E = (D + 16) * 2.0 ** -24 * mm(self.q.abs(), self.t(self.k.abs())) * self.scale + 2.0 ** -20
        self.t1 = torch.ones_like(u)
        if cap:
            t = torch.tanh(u / cap)
            u, self.t1 = cap * t, 1 - t * t
            E = E + 2.0 ** -20 * cap
        at = torch.arange(S, device=DEV)
        if slopes is not None:
            bias = slopes.to(F64)[:, None, None] * (at[:, None] - at[None, :]).abs()
            u, E = u - bias, E + 2.0 ** -22 * bias
        visible = (at[None, :] <= at[:, None])[None].expand(B, S, S)
        if prefix is not None:
            visible = visible | (at[None, None, :] < prefix[:, None, None])
        if seg is not None:
            visible = visible & (seg[:, :, None] == seg[:, None, :])
        u = u.masked_fill(~visible[:, None], -math.inf)
        self.raw = torch.exp(u - u.amax(-1, keepdim=True))
        self.P = self.raw / self.raw.sum(-1, keepdim=True)
        self.o = mm(self.P, self.v)
        self.dP = mm(self.do, self.t(self.v))
        # (Summed pair by pair: |v_j - o_i| is no product.)
        apart = torch.stack([(self.P[:, :, i:i + 1] * (R + E[:, :, i:i + 1])).transpose(-1, -2).mul(
            (self.v - self.o[:, :, i:i + 1]).abs()).sum(2) for i in range(S)], 2)
        self.wo = MORE * apart + 2.0 ** -18 * (self.o.abs() + mm(self.P, self.v.abs()))
        size = (self.do * self.o).abs().sum(-1, keepdim=True)
        wdelta = (self.do.abs() * (self.wo + 2.0 ** -15 * self.o.abs())).sum(-1, keepdim=True) + (D + 16) * 2.0 ** -24 * size
        PE = self.P * E
        PE = PE + self.P * PE.sum(-1, keepdim=True)
        left = self.dP - (self.do * self.o).sum(-1, keepdim=True)
        fP = (D + 16) * 2.0 ** -24 * mm(self.do.abs(), self.t(self.v.abs()))
        dU = (self.P * left * self.t1).abs()
        w = MORE * (R * dU + (PE * left.abs() + self.P * (fP + wdelta)) * self.t1 + 2.0 ** -20 * self.P * left.abs())
        self.bounds = {"o": self.wo + R * (self.o.abs() + self.wo)}
        for name, share in (("dq", self.scale * mm(w + 2.0 ** -18 * dU, self.k.abs())),
                            ("dk", self.heads(self.scale * mm(self.t(w + 2.0 ** -18 * dU), self.q.abs())))):
            self.bounds[name] = share + R * (self.gradients(self.o)[name].abs() + share)

    @staticmethod
    def t(x):
        return x.transpose(-1, -2).contiguous()

    def heads(self, x):
        return x.reshape(self.join).sum(2)

    def gradients(self, o):
        dU = self.P * (self.dP - (self.do * o).sum(-1, keepdim=True)) * self.t1 * self.scale
        return {"dq": torch.matmul(dU, self.k), "dk": self.heads(torch.matmul(self.t(dU), self.q))}

    def past(self, name, value):
        """The share of values outside their bound."""

        exact = self.o if name == "o" else self.gradients(self.o)[name]
        return float(((value.to(F64) - exact).abs() > self.bounds[name]).to(F64).mean())


def run(q, k, v, do, cap=None, slopes=None, seg=None, prefix=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = make_scored_attention(ScoredAttentionConfig(score_cap=cap))(*leaves, seg, prefix_lengths=prefix,
                                                                    distance_slopes=slopes)
    grads = torch.autograd.grad(o, leaves, do)
    torch.cuda.synchronize()
    return {"o": o.detach(), "dq": grads[0], "dk": grads[1], "dv": grads[2]}


CASES = {
    "plain-64": dict(sizes=(1, 2, 2, 200, 64)),
    "cap-64": dict(sizes=(1, 2, 1, 171, 64), cap=30.0),
    "bias-128": dict(sizes=(1, 2, 2, 150, 128), slopes=True),
    "cap-bias-128": dict(sizes=(1, 4, 2, 130, 128), cap=20.0, slopes=True),
    "documents-64": dict(sizes=(2, 2, 2, 129, 64), seg=12),
    "prefix-40": dict(sizes=(2, 2, 2, 100, 40), prefix=True),
    "many-64": dict(sizes=(33, 32, 32, 70, 64), cap=30.0),  # 128 rows a workgroup
    "many-128": dict(sizes=(33, 32, 16, 70, 128), seg=20),
}


@pytest.mark.parametrize("name", CASES)
def test_delta_from_more_than_bfloat16(name):
    print(f"scored attention, neighbouring values {name}", flush=True)
    case = dict(CASES[name])
    B, H, Hk, S, D = sizes = case.pop("sizes")
    if "slopes" in case:
        case["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEV, dtype=F32) / H)
    if "prefix" in case:
        case["prefix"] = torch.tensor([64, 7][:B], dtype=torch.int32, device=DEV)
    if "seg" in case:
        cuts = torch.rand((B, S), generator=torch.Generator().manual_seed(4)) < 1.0 / case["seg"]
        case["seg"] = torch.cumsum(cuts, 1).to(torch.int32).to(DEV)
    tensors = inputs(*sizes, seed=S)
    want = Exact(*tensors, **case)
    # What either loss would do, in the 64-bit computation: o as bfloat16, and o over the sum of the P before their rounding.
    short = want.gradients(want.o.to(BF16).to(F64))
    rounded = torch.matmul(want.raw.to(BF16).to(F64), want.v) / want.raw.sum(-1, keepdim=True)
    uneven = want.gradients(rounded)
    for n in ("dq", "dk"):
        assert want.past(n, short[n]) > 0.05 and want.past(n, uneven[n]) > 0.01, n
    assert want.past("o", rounded.to(BF16)) > 0.001
    got = run(*tensors, **case)
    for n in ("o", "dq", "dk"):
        assert want.past(n, got[n]) == 0, n


def test_powers_of_two_change_nothing():
    """v times 2^100 and do times 2^-100: the same delta and dP, so the same dq and dk bit for bit, dv by 2^-100."""

    q, k, v, do = inputs(1, 2, 2, 200, 64, seed=9)
    v = v.clone()
    v[..., ::3] *= 1.75
    want = run(q, k, v, do, cap=30.0)
    for power in (-100, 100):
        f = 2.0 ** power
        got = run(q, k, v * f, do / f, cap=30.0)
        assert torch.equal(got["dq"], want["dq"]) and torch.equal(got["dk"], want["dk"])
        assert torch.equal(got["o"], want["o"] * f) and torch.equal(got["dv"], want["dv"] / f)
