"""Optimizer schedule and per-tensor AdamW hyper-parameters, mirroring
``recipes/reference/train.py:1219-1345``.

The update itself is the fused ``gptrig_adamw`` kernel over one arena; this
module resolves the host-side scalars (learning rate per step, bias corrections)
and the per-tensor table ``{lr_mult, epsilon, decay}`` the kernel reads.
``adamw_tensors`` is the same update over tensors that lie anywhere, with float32
or 8-bit moments.
"""

from __future__ import annotations

import array
import math
import operator
import warnings
from dataclasses import dataclass
from typing import Sequence

import numpy as np
import torch

from . import _lib


@dataclass(frozen=True)
class OptimizerConfig:
    """``run.optimizer`` of ``recipes/reference/config.yaml:98-108``."""

    learning_rate: float = 2.0 ** -8
    min_lr_ratio: float = 0.1
    warmup_steps: int = 0
    steps: int = 1
    weight_decay: float = 0.1
    adam_epsilon: float = 1.0e-8
    beta1: float = 0.9
    beta2: float = 0.95
    grad_clip: float = 0.0
    batch_multiplier: float = 1.0
    data_multiplier: float = 1.0


def _f32(x: float) -> float:
    return float(np.float32(x))


def learning_rate(step: int, cfg: OptimizerConfig) -> float:
    """``learning_rate`` (``train.py:1219-1236``) with float32 arithmetic."""

    s = _f32(step)
    warmup = min(1.0, _f32(s / float(cfg.warmup_steps))) if cfg.warmup_steps else 1.0
    span = max(1, cfg.steps - cfg.warmup_steps)
    progress = min(max(_f32((s - float(cfg.warmup_steps)) / float(span)), 0.0), 1.0)
    cosine = _f32(0.5 * (1.0 + _f32(math.cos(_f32(math.pi * progress)))))
    mult = _f32(cfg.min_lr_ratio + (1.0 - cfg.min_lr_ratio) * cosine)
    horizon = math.sqrt(cfg.batch_multiplier / cfg.data_multiplier)
    return _f32(_f32(_f32(cfg.learning_rate * horizon) * warmup) * mult)


def effective_adam_betas(cfg: OptimizerConfig) -> tuple[float, float]:
    """``effective_adam_betas`` (``train.py:1336-1345``)."""

    ratio = cfg.batch_multiplier / cfg.data_multiplier
    beta1 = 1.0 - (1.0 - cfg.beta1) * ratio
    beta2 = 1.0 - (1.0 - cfg.beta2) * ratio
    if not 0.0 <= beta1 < 1.0 or not 0.0 <= beta2 < 1.0:
        raise ValueError("fixed-TPP batch/data scaling produced invalid Adam momenta; use a closer transfer base")
    return beta1, beta2


def decays(path: str) -> bool:
    """``weight_decay_mask`` (``train.py:1252-1271``): decided by role name."""

    name = path.rsplit("/", 1)[-1]
    if name in {"token_embedding", "output_embedding"} or name.endswith("_w"):
        return True
    if name.endswith(("_b", "_bias", "_scale")):
        return False
    raise ValueError(f"weight-decay policy has no rule for parameter {name!r}")


def multipliers(path: str, parameterization: str, width: float, depth: float, alpha: float):
    """(lr, epsilon, decay) multipliers of ``optimizer_hyperparameter_trees``
    (``train.py:1274-1333``)."""

    if parameterization != "completep_fixed_tpp_v1":
        return 1.0, 1.0, 1.0
    name = path.rsplit("/", 1)[-1]
    if path.startswith("blocks/"):
        is_w = name.endswith("_w")
        lr = width ** -1 * depth ** (alpha - 1.0) if is_w else depth ** (alpha - 1.0)
        return lr, width ** -1 * depth ** -alpha, (width if is_w else 1.0)
    if name == "token_embedding":
        return 1.0, width ** -1, 1.0
    if name == "output_embedding":
        return width ** -1, 1.0, width
    if name == "final_ln_scale":
        return 1.0, 1.0, 1.0
    raise ValueError(f"no multiplier rule for {path!r}")


def tensor_hparams(paths, cfg: OptimizerConfig, parameterization: str, width: float, depth: float,
                   alpha: float) -> np.ndarray:
    """``[T, 3]`` float32 table of (lr_mult, epsilon, decay) per tensor
    (``train.py:1420-1435``)."""

    eps_h = math.sqrt(cfg.data_multiplier / cfg.batch_multiplier)
    dec_h = math.sqrt(cfg.batch_multiplier / cfg.data_multiplier)
    rows = []
    for path in paths:
        lr_m, eps_m, dec_m = multipliers(path, parameterization, width, depth, alpha)
        eps = cfg.adam_epsilon * eps_h * eps_m
        decay = cfg.weight_decay * dec_h * dec_m if decays(path) else 0.0
        rows.append((lr_m, eps, decay))
    return np.asarray(rows, dtype=np.float32)


# Consecutive values of a tensor that share a scale of the 8-bit moments.
STATE_BLOCK = 256
_STATE_TYPES = {torch.float32: 32, torch.float8_e4m3fn: 8}
_F32, _BF16 = {torch.float32}, {torch.bfloat16}
_DTYPE, _SHAPE = operator.attrgetter("dtype"), operator.attrgetter("shape")
E_OVERLAP = -7  # GPTRIG_E_OVERLAP


def adamw_tensors_state(params: Sequence[torch.Tensor], bits: int = 32) -> dict[str, list[torch.Tensor]]:
    """Zero moments for ``adamw_tensors`` under its argument names: float32, or
    float8_e4m3fn codes and their scales with ``bits=8``."""

    if bits not in (8, 32):
        raise ValueError(f"moments are held in 8 or 32 bits, got {bits}")
    names = ("exp_avg", "exp_avg_sq")
    if bits == 32:
        return {n: [torch.zeros(p.shape, dtype=torch.float32, device=p.device) for p in params] for n in names}
    state = {n: [torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn) for p in params]
             for n in names}
    state.update({n + "_scale": [torch.zeros(-(-p.numel() // STATE_BLOCK), dtype=torch.float32, device=p.device)
                                 for p in params] for n in names})
    return state


def _list_of(name: str, tensors, shapes: list, dtypes, device: int) -> torch.dtype:
    """Checks a list of tensors against the shapes and the GPU it must have; its type."""

    # (Maps over bound methods: with many small tensors the host's work is the step's.)
    if len(tensors) != len(shapes):
        raise ValueError(f"{name} has {len(tensors)} tensors, params {len(shapes)}")
    types = set(map(_DTYPE, tensors))
    if len(types) > 1 or not types <= dtypes:
        raise TypeError(f"{name} must all be one of {sorted(map(str, dtypes))}, got {sorted(map(str, types))}")
    if list(map(_SHAPE, tensors)) != shapes:
        i = next(i for i, t in enumerate(tensors) if t.shape != shapes[i])
        raise ValueError(f"{name}[{i}] must be {tuple(shapes[i])}, got {tuple(tensors[i].shape)}")
    if not all(map(torch.Tensor.is_contiguous, tensors)):
        i = next(i for i, t in enumerate(tensors) if not t.is_contiguous())
        raise ValueError(f"{name}[{i}] must be contiguous")
    if set(map(torch.Tensor.get_device, tensors)) != {device}:
        raise RuntimeError(f"{name} must all be on the device of params[0]")
    return types.pop()


def adamw_tensors(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avg: Sequence[torch.Tensor],
                  exp_avg_sq: Sequence[torch.Tensor], hparams: torch.Tensor, *, lr: float, beta1: float, beta2: float,
                  step: int, exp_avg_scale: Sequence[torch.Tensor] | None = None,
                  exp_avg_sq_scale: Sequence[torch.Tensor] | None = None, clip_scale: torch.Tensor | None = None,
                  shadow: Sequence[torch.Tensor] | None = None, seed: int | torch.Tensor | None = None) -> None:
    """One AdamW step, in place, over a list of contiguous float32 tensors.

    The update of ``GPTTrainer`` (``recipes/reference/train.py:1386-1445``), in a
    few launches however many tensors there are.  ``hparams``: float32 ``[tensors,
    3]`` on the device, the rows ``{lr_mult, epsilon, decay}`` of
    ``tensor_hparams``.  ``grads``: all float32 or all bfloat16.  ``exp_avg`` and
    ``exp_avg_sq``: both float32, or both float8_e4m3fn with the scales of their
    blocks of ``STATE_BLOCK`` values (``adamw_tensors_state`` makes either).  8-bit
    moments are rounded stochastically from ``seed`` (0 to 2^32 - 1; default
    ``step``), which every step needs another of; the same call gives the same
    result.  ``clip_scale``: a float32 scalar on the device that multiplies the
    gradients.  ``shadow``: bfloat16 tensors that receive the rounded parameters.
    A tensor that is written may overlap no other.  ``lr``, ``step`` and a ``seed``
    that is a number are fixed in a captured graph: its replays would round 8-bit moments
    the same way each time, so that some elements stand still and others decay for good.
    For a graph give ``seed`` as an int64 scalar on the device (its lower 32 bits count)
    that every replay finds changed, by ``seed.add_(1)`` in the graph or between replays.
    """

    if not params:
        raise ValueError("adamw_tensors needs at least one tensor")
    device = params[0].get_device()
    shapes = list(map(_SHAPE, params))
    counts = list(map(torch.Tensor.numel, params))
    _list_of("params", params, shapes, _F32, device)
    grad_type = _list_of("grads", grads, shapes, _F32 | _BF16, device)
    kind = _list_of("exp_avg", exp_avg, shapes, _STATE_TYPES.keys(), device)
    _list_of("exp_avg_sq", exp_avg_sq, shapes, {kind}, device)
    bits = _STATE_TYPES[kind]
    if (exp_avg_scale is None) != (bits == 32) or (exp_avg_sq_scale is None) != (bits == 32):
        raise ValueError("8-bit moments, and only those, come with exp_avg_scale and exp_avg_sq_scale")
    if bits == 8:
        blocks = [(-(-n // STATE_BLOCK),) for n in counts]
        _list_of("exp_avg_scale", exp_avg_scale, blocks, _F32, device)
        _list_of("exp_avg_sq_scale", exp_avg_sq_scale, blocks, _F32, device)
    if shadow is not None:
        _list_of("shadow", shadow, shapes, _BF16, device)
    if hparams.dtype != torch.float32 or hparams.shape != (len(params), 3) or not hparams.is_contiguous():
        raise ValueError(f"hparams must be contiguous float32 [{len(params)}, 3], got {hparams.dtype} "
                         f"{tuple(hparams.shape)}")
    if clip_scale is not None and (clip_scale.dtype != torch.float32 or clip_scale.numel() != 1):
        raise ValueError("clip_scale must be one float32 value")
    if not 0.0 <= beta1 < 1.0 or not 0.0 <= beta2 < 1.0:
        raise ValueError(f"beta1 and beta2 must be in [0, 1), got {beta1} and {beta2}")
    if not 1 <= step < 2 ** 31:
        raise ValueError(f"step counts from 1 and stays below 2^31, got {step}")
    on_device = isinstance(seed, torch.Tensor)
    if on_device:
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError("a seed on the device must be one int64 value")
    else:
        seed = step % 2 ** 32 if seed is None else seed
        if not 0 <= seed < 2 ** 32:
            raise ValueError(f"seed must be in [0, 2^32), got {seed}")
    _lib.require_one_device(params[0], hparams, clip_scale, seed if on_device else None)
    if bits == 8 and not on_device and torch.cuda.is_current_stream_capturing():
        warnings.warn("adamw_tensors captured with 8-bit moments and a seed that is a number: every replay rounds them "
                      "the same way; give the seed as an int64 tensor that changes between replays", stacklevel=2)
    # One row of gptrig_adamw_tensor a tensor: seven addresses and the count.
    table = [0] * (8 * len(params))
    for column, tensors in enumerate((params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, shadow)):
        if tensors is not None:
            table[column::8] = map(torch.Tensor.data_ptr, tensors)
    table[7::8] = counts
    table = array.array("q", table)
    try:
        _lib.call_on(device, "gptrig_adamw_tensors_device_seed" if on_device else "gptrig_adamw_tensors",
                     table.buffer_info()[0], len(params), 1 if grad_type == torch.float32 else 0, bits,
                     hparams.data_ptr(), float(lr), float(beta1), float(beta2), int(step), _lib.ptr(clip_scale),
                     seed.data_ptr() if on_device else seed)
    except _lib.StatusError as error:
        if error.status == E_OVERLAP:
            raise ValueError("a tensor that the step writes overlaps another") from error
        raise
    # (A graph that saved one of them must not run backward now.)
    torch.autograd.graph.increment_version(params)
    if shadow is not None:
        torch.autograd.graph.increment_version(shadow)
