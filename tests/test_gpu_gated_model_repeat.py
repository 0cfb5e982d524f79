"""The training step of ``test_gpu_gated_model_step`` a second time: the same parameters, updates and losses, bit for bit.
Every operator of it adds in a fixed order at this size."""

from __future__ import annotations

import pytest
import torch
from test_gpu_gated_model_step import DEV, fresh, setup, step

pytestmark = pytest.mark.gpu


def test_the_same_steps_twice():
    w, ids, targets = setup(seed=1)
    every = []
    for _ in range(2):
        run, seen = fresh(w), []
        for number in range(1, 4):
            out, updates = step(*run, ids.to(DEV), targets.to(DEV), number)
            seen += [out, *updates, *(p.detach().clone() for p in run[0]), *(m.clone() for m in run[1])]
        every.append(seen)
    assert len(every[0]) == len(every[1]) == 30
    assert all(torch.equal(a, b) for a, b in zip(*every))
