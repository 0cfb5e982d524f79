"""How ``layer_norm``, ``adamw_tensors`` and the scored attention treat a call before anything is launched: the
launches are replaced by stand-ins on the CPU."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from gptrig import _lib, nn
from gptrig.kernels import make_scored_attention, scored_attention

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def no_launch(monkeypatch):
    """Both operators on CPU tensors, their outputs copies of an input."""

    monkeypatch.setattr(_lib, "require_one_device", lambda *tensors: None)
    monkeypatch.setattr(nn, "_layer_norm_forward",
                        lambda x, scale, bias, eps, keep: (x.clone(), x.clone(), scale.clone(), torch.zeros((2, 3))))
    monkeypatch.setattr(scored_attention, "_forward",
                        lambda q, k, v, *rest: (q, k, v, q.clone(), torch.zeros(8), None, True))


def calls():
    x, scale = torch.randn((3, 8)), torch.ones(8)
    q = torch.randn((1, 2, 4, 8)).to(BF16)
    return [(nn.layer_norm, [x, scale]), (nn.layer_norm, [x, scale, scale.clone()]),
            (make_scored_attention(), [q, q.clone(), q.clone()])]


@pytest.mark.parametrize("gradients", [True, False])
def test_forward_derivatives_are_refused(no_launch, gradients):
    """A tangent does not show in ``requires_grad``: without autograd's node the result would have none, a derivative
    of zero.  ``rms_norm`` and the causal attention refuse it in the same way."""

    for operator, tensors in calls():
        for i in range(len(tensors)):
            with forward_ad.dual_level(), torch.set_grad_enabled(gradients):
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(tensors)]
                with pytest.raises(NotImplementedError, match="jvp"):
                    operator(*dual)


def test_a_dual_level_without_tangents_changes_nothing(no_launch):
    for operator, tensors in calls():
        with forward_ad.dual_level():
            assert torch.equal(operator(*tensors), tensors[0])
        assert torch.equal(operator(*tensors), tensors[0])
        assert operator(*(t.clone().requires_grad_() for t in tensors)).requires_grad


def test_caps_that_float32_does_not_hold_are_refused():
    """A cap reaches the kernels as float32, where 0 is no cap at all; below 2^-126 it loses bits, from 2^-150 down all."""

    from gptrig.kernels import ScoredAttentionConfig

    for bad in (5e-324, 1e-300, 2.0 ** -150, 7e-46, 1e-42, 2.0 ** -127):
        with pytest.raises(ValueError, match="score_cap"):
            ScoredAttentionConfig(score_cap=bad)
    for cap in (2.0 ** -126, 1e-30, 0.01, 1000.0):
        assert ScoredAttentionConfig(score_cap=cap).score_cap == cap


def test_an_eps_that_float32_does_not_hold_is_refused(no_launch):
    """It reaches the kernels as float32: one that this rounds to 0 would make a constant row 0 / 0, one that it
    rounds to infinity every row 0."""

    x, scale = torch.randn((3, 8)), torch.ones(8)
    for bad in (1e-46, 5e-324, 2.0 ** -150, 3.5e38, 1e300):
        with pytest.raises(ValueError, match="eps"):
            nn.layer_norm(x, scale, eps=bad)
    for eps in (0, 0.0, 2.0 ** -149, 1e-12, 1.0, 3e38):
        assert torch.equal(nn.layer_norm(x, scale, eps=eps), x)


def test_a_seed_on_the_device_is_checked():
    import ctypes

    from gptrig.optim import adamw_tensors, adamw_tensors_state

    p = [torch.zeros(300)]
    call = dict(params=p, grads=[torch.zeros(300)], hparams=torch.zeros((1, 3)), lr=0.1, beta1=0.9, beta2=0.95, step=1,
                **adamw_tensors_state(p, 8))
    for bad in (torch.zeros((), dtype=torch.int32), torch.zeros(2, dtype=torch.int64), torch.zeros(()),
                torch.zeros(0, dtype=torch.int64)):
        with pytest.raises(ValueError, match="one int64"):
            adamw_tensors(**call, seed=bad)
    with pytest.raises(RuntimeError, match="GPU"):
        adamw_tensors(**call, seed=torch.zeros((), dtype=torch.int64))
    entry, at = _lib.lib().gptrig_adamw_tensors_device_seed, ctypes.c_void_p(1 << 12)
    row = (ctypes.c_int64 * 8)(*[k << 20 for k in range(1, 8)], 100)
    assert entry(row, 1, 1, 8, at, 0.1, 0.9, 0.95, 1, None, None, None) == -1
    assert entry(row, 1, 1, 8, at, 0.1, 0.9, 0.95, 1, None, ctypes.c_void_p((1 << 12) + 4), None) == -2
    assert entry(row, 1, 1, 16, at, 0.1, 0.9, 0.95, 1, None, at, None) == -4
    assert entry(row, 0, 1, 8, at, 0.1, 0.9, 0.95, 1, None, at, None) == 0
