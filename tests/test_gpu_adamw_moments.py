"""8-bit moments of ``gptrig.optim.adamw_tensors`` where a float32 state would still hold them: gradients whose squares
are next to nothing.

With every gradient of a block equal to +-g its moments after the first step are +-(1 - b1) g and (1 - b2) g^2, the
largest of their blocks, so their codes are exact; a second step without a gradient then moves a parameter by
lr m / sqrt(v) (eps 0) with m = b1 (1 - b1) / (1 - b1^2) g and v = b2 (1 - b2) / (1 - b2^2) g^2.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F64 = torch.float32, torch.float64
U = 2.0 ** -24
LR, B1, B2 = 0.01, 0.9, 0.95
WAY = B1 / (1 + B1) / math.sqrt(B2 / (1 + B2))


def two_steps(g, eps):
    """The parameters after a step on gradients +-g and after one without any, and the gradients' signs."""

    from gptrig.optim import adamw_tensors, adamw_tensors_state

    n = 1024
    gen = torch.Generator().manual_seed(3)
    sign = torch.where(torch.rand(n, generator=gen) < 0.5, -1.0, 1.0).to(DEV)
    p = [torch.randn(n, generator=gen).to(DEV)]
    state = adamw_tensors_state(p, 8)
    hp = torch.tensor([[1.0, eps, 0.0]], device=DEV)
    out = []
    for step, grad in ((1, sign * g), (2, torch.zeros(n, device=DEV))):
        adamw_tensors(p, [grad], hparams=hp, lr=LR, beta1=B1, beta2=B2, step=step, **state)
        out.append(p[0].to(F64))
    return *out, sign.to(F64), state


@pytest.mark.parametrize("g", [1e-3, 1e-12, 1e-14, 1e-15, 1e-16, 3e-17])
def test_a_small_v_is_kept(g):
    """Down to a v of 2^-117: with eps 0 the second step is that of the formula.  A chain of fewer than 40 roundings of
    2^-24 of the move, two of the parameter."""

    print(f"adamw_tensors 8 bits g={g}", flush=True)
    assert (1 - B2) * g * g > 2.0 ** -117
    first, second, sign, state = two_steps(g, 0.0)
    assert (state["exp_avg_sq_scale"][0] > 0).all()
    off = (second - first + LR * WAY * sign).abs()
    assert (off <= 40 * U * LR * WAY + 2 * U * first.abs()).all(), float(off.max())


@pytest.mark.parametrize("g", [1e-17, 1e-18, 1e-20, 1e-24])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-8])
def test_a_v_kept_as_zero_divides_by_more_than_eps(g, eps):
    """Below that v is kept as zero and its momentum is not: the next step must not be the momentum over eps.  The v that
    it counts as is the most that can have been dropped, so the step is at most the formula's (the roundings as above)."""

    print(f"adamw_tensors 8 bits g={g} eps={eps}", flush=True)
    first, second, sign, state = two_steps(g, eps)
    assert not state["exp_avg_sq_scale"][0].any() and (state["exp_avg_scale"][0] > 0).all()
    move = (first - second) * sign
    slack = 40 * U * LR * WAY + 2 * U * first.abs()
    assert (move <= LR * WAY + slack).all() and (move >= -slack).all(), float(move.abs().max())
