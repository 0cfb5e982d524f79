"""``nn.embedding`` takes its scale as a number: a tensor that asks for a gradient would get none, and is refused."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from gptrig.nn import embedding


def test_a_scale_that_asks_for_a_gradient():
    tokens, table = torch.zeros(3, dtype=torch.int32), torch.zeros((5, 8))
    scale = torch.tensor(2.0, requires_grad=True)
    with pytest.raises(RuntimeError, match="no derivative in scale"):
        embedding(tokens, table, scale=scale)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no derivative in scale"):
        embedding(tokens, table, scale=forward_ad.make_dual(torch.tensor(2.0), torch.tensor(1.0)))
    # Numbers in any form, and tensors that ask for none, go on (to the refusal of host memory).
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        embedding(tokens, table, scale=scale)
    for number in (2, torch.tensor(2.0), torch.tensor([2.0], dtype=torch.bfloat16), scale.detach().numpy()):
        with pytest.raises(RuntimeError, match="GPU"):
            embedding(tokens, table, scale=number)
    for bad in (torch.tensor(float("nan")), torch.tensor(1e300, dtype=torch.float64), 10 ** 400):
        with pytest.raises(ValueError, match="finite float32"):
            embedding(tokens, table, scale=bad)


@pytest.mark.gpu
def test_the_scale_of_the_call():
    """A tensor that changes between the forward and the backward: both take the value at the call."""

    tokens = torch.tensor([1, 1, 4], dtype=torch.int32, device="cuda:0")
    table = torch.ones((5, 8), device="cuda:0", requires_grad=True)
    scale = torch.tensor(2.0)
    y = embedding(tokens, table, scale=scale)
    scale.fill_(3.0)
    (grad,) = torch.autograd.grad(y, table, torch.ones_like(y))
    assert (y == 2).all() and (grad[1] == 4).all() and (grad[4] == 2).all() and (grad[[0, 2, 3]] == 0).all()
