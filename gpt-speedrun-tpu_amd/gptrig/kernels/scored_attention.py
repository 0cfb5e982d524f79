"""Attention whose scores are capped by a tanh or biased by distance, on gfx950.

Beside ``make_causal_attention``, which is the reference's operator:
``make_scored_attention(ScoredAttentionConfig)`` returns ``attention(q, k, v,
segment_ids=None, *, prefix_lengths=None, distance_slopes=None)`` over BHSD
tensors, with key and value heads that query heads may share.  For query i and
key j of one head

    u = softmax_scale * q_i . k_j
    score = score_cap * tanh(u / score_cap) - slope * |i - j|   (u without a cap)
    visible: (j <= i or j < prefix) and segment_i == segment_j

It runs the kernels of ``csrc/scored_attention_fwd.hip`` and
``csrc/scored_attention_bwd.hip``; head dims up to 128 and sequences of any length
are handled in-kernel.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Callable

import torch
from torch.autograd.function import once_differentiable

from .. import _lib

MAX_CAP = 1000.0  # float32 tells tanh scores of a larger cap apart less well than bfloat16 operands do
MIN_CAP = 2.0 ** -126  # the kernels take the cap as a float32; one that this rounds to 0 would be none


@dataclass(frozen=True)
class ScoredAttentionConfig:
    """``softmax_scale``: default ``head_dim ** -0.5``; ``score_cap``: default none."""

    softmax_scale: float | None = None
    score_cap: float | None = None

    def __post_init__(self) -> None:
        if self.softmax_scale is not None and not 0.0 < self.softmax_scale < math.inf:
            raise ValueError(f"softmax_scale must be positive and finite, got {self.softmax_scale}")
        if self.score_cap is not None and not MIN_CAP <= self.score_cap <= MAX_CAP:
            raise ValueError(f"score_cap must be in [2^-126, {MAX_CAP:g}], got {self.score_cap}")


def _validate(q, k, v, segment_ids, prefix_lengths, distance_slopes) -> None:
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError(
            f"q, k, and v must use BHSD rank-4 layout; got {tuple(q.shape)}, {tuple(k.shape)}, and {tuple(v.shape)}"
        )
    if 0 in q.shape or 0 in k.shape:
        raise ValueError(f"q/k/v dimensions must be nonzero, got {tuple(q.shape)} and {tuple(k.shape)}")
    B, H, S, D = q.shape
    if k.shape != v.shape or (k.shape[0], k.shape[2], k.shape[3]) != (B, S, D) or H % k.shape[1]:
        raise ValueError("k and v must be [batch, kv_heads, seq, head_dim] of q's batch, seq and head_dim, kv_heads "
                         f"dividing q's heads; got {tuple(q.shape)}, {tuple(k.shape)}, and {tuple(v.shape)}")
    if D > 128 or D % 8:
        raise ValueError(f"the kernel requires head_dim <= 128 and divisible by 8; got {D}")
    if not q.dtype == k.dtype == v.dtype == torch.bfloat16:
        raise TypeError(f"the HIP attention kernels take bfloat16 q/k/v; got {q.dtype}, {k.dtype}, {v.dtype}")
    if segment_ids is None and prefix_lengths is None and distance_slopes is None:
        return
    for name, t, shape in (("segment_ids", segment_ids, (B, S)), ("prefix_lengths", prefix_lengths, (B,))):
        if t is None:
            continue
        if t.dtype not in (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64):
            raise TypeError(f"{name} must be integers, got {t.dtype}")
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must be {list(shape)}; got {tuple(t.shape)}")
    if distance_slopes is not None:
        if distance_slopes.dtype != torch.float32:
            raise TypeError(f"distance_slopes must be float32, got {distance_slopes.dtype}")
        if tuple(distance_slopes.shape) != (H,):
            raise ValueError(f"distance_slopes must be [{H}], one a head; got {tuple(distance_slopes.shape)}")
        if distance_slopes.requires_grad:
            raise ValueError("distance_slopes are constants: no gradient is computed for them")


def _fits(t: torch.Tensor) -> bool:
    """Unit last stride, 8-element strides, 16-byte base, a (batch, head) slice within 32-bit offsets."""

    a, b, c, d = t.stride()
    return d == 1 and not (a | b | c) % 8 and not t.data_ptr() % 16 and (t.shape[2] + 64) * c < 1 << 30


def _view(t: torch.Tensor) -> torch.Tensor:
    """A BHSD view the kernels accept."""

    # (contiguous() returns the tensor itself where only its base or the strides of dimensions of size 1 are odd.)
    return t if _fits(t) else t.clone(memory_format=torch.contiguous_format)


_ARRAYS = {n: ctypes.c_int64 * (3 * n) for n in (4, 8)}


def _strides(*tensors: torch.Tensor):
    """The (batch, head, seq) strides of each tensor as the int64 array the entry points read."""

    return _ARRAYS[len(tensors)](*[s for t in tensors for s in t.stride()[:3]])


# (The host's work is most of a small call's time, and backwards run on a thread of
# their own, at half the speed: so contiguous tensors take the shorter ways below.)
def _plain(*tensors: torch.Tensor) -> bool:
    """Whether the kernels take them as they are, with default strides."""

    for t in tensors:
        if not t.is_contiguous() or t.data_ptr() & 15:
            return False
    return True


@functools.lru_cache(maxsize=512)
def _sizes(query: str, *sizes: int) -> int:
    return _lib.query(query, *sizes)


def _forward(q, k, v, segment_ids, prefix_lengths, slopes, scale: float, cap: float, keep: bool):
    """The views read, ``o``, for the backward (``None`` unless ``keep``) what its rounding cut off and then the
    logarithms of the scores' sums, in one buffer, the plan if the call has one, and whether the views are plain."""

    B, H, S, D = q.shape
    if _plain(q, k, v):
        o, strides = torch.empty_like(q), None
    else:
        q, k, v = _view(q), _view(k), _view(v)
        o = torch.empty((B, H, S, D), dtype=q.dtype, device=q.device)
        strides = _strides(q, k, v, o)
    kept = low = lse2 = None
    if keep:
        rows = B * H * S
        kept = torch.empty(rows * (D + 4), dtype=torch.uint8, device=q.device)
        low = kept.data_ptr()
        lse2 = low + rows * D
    plan = None
    if segment_ids is not None or prefix_lengths is not None:
        sizes = (B, H, k.shape[1], S, D)
        need = _sizes("gptrig_scored_attn_plan_bytes", *sizes)
        if need:
            plan = torch.empty(need, dtype=torch.uint8, device=q.device)
            _lib.call_on(q.get_device(), "gptrig_scored_attn_plan", _lib.ptr(segment_ids), _lib.ptr(prefix_lengths),
                         plan.data_ptr(), need, *sizes)
    _lib.call_on(q.get_device(), "gptrig_scored_attn_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(),
                 _lib.ptr(segment_ids), _lib.ptr(prefix_lengths), _lib.ptr(slopes), _lib.ptr(plan), o.data_ptr(),
                 low, lse2, B, H, k.shape[1], S, D, strides, scale, cap)
    return q, k, v, o, kept, plan, strides is None


class _ScoredAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, segment_ids, prefix_lengths, slopes, scale, cap):
        *kept, ctx.plain = _forward(q, k, v, segment_ids, prefix_lengths, slopes, scale, cap, True)
        ctx.save_for_backward(*kept, segment_ids, prefix_lengths, slopes)
        ctx.scalars = (scale, cap)
        return kept[3]

    @staticmethod
    def backward(ctx, do):
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, do)


def _backward(ctx, do):
    q, k, v, o, kept, plan, segment_ids, prefix_lengths, slopes = ctx.saved_tensors
    B, H, S, D = q.shape
    Hk = k.shape[1]
    if ctx.plain and _plain(do):
        dq, dk, dv, strides = torch.empty_like(q), torch.empty_like(k), torch.empty_like(k), None
    else:
        do = _view(do)
        dq = torch.empty((B, H, S, D), dtype=q.dtype, device=q.device)
        dk = torch.empty((B, Hk, S, D), dtype=q.dtype, device=q.device)
        dv = torch.empty_like(dk)
        strides = _strides(q, k, v, o, do, dq, dk, dv)
    size = _sizes("gptrig_scored_attn_bwd_workspace_bytes", B, H, Hk, S, D)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device)
    low = kept.data_ptr()
    _lib.call_on(q.get_device(), "gptrig_scored_attn_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                 do.data_ptr(), low, low + B * H * S * D, _lib.ptr(segment_ids), _lib.ptr(prefix_lengths),
                 _lib.ptr(slopes), _lib.ptr(plan), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), size,
                 B, H, Hk, S, D, strides, *ctx.scalars)
    return dq, dk, dv, None, None, None, None, None


_backward_once = once_differentiable(_backward)


def make_scored_attention(config: ScoredAttentionConfig = ScoredAttentionConfig()) -> Callable:
    """The attention of this module for one configuration.

    ``q`` ``[batch, heads, seq, head_dim]``, ``k`` and ``v`` ``[batch, kv_heads,
    seq, head_dim]`` bfloat16 of any strides, ``heads`` a multiple of ``kv_heads``
    (head h reads kv head ``h // (heads // kv_heads)``).  ``segment_ids``: integers
    ``[batch, seq]``, compared in their lower 32 bits; ``prefix_lengths``: integers ``[batch]``, the positions that
    every query of the sequence sees; ``distance_slopes``: float32 ``[heads]``,
    constants.  Differentiable once in q, k and v; the same call gives the same
    bits.  Pairs that are not visible add nothing, whatever they hold.
    """

    def attention(q, k, v, segment_ids=None, *, prefix_lengths=None, distance_slopes=None):
        _validate(q, k, v, segment_ids, prefix_lengths, distance_slopes)
        S = q.shape[2]
        if segment_ids is not None:
            segment_ids = segment_ids.to(torch.int32).contiguous()
        if prefix_lengths is not None:
            if prefix_lengths.dtype == torch.int64:
                prefix_lengths = prefix_lengths.clamp(0, S)
            prefix_lengths = prefix_lengths.to(torch.int32).contiguous()
        if distance_slopes is not None:
            distance_slopes = distance_slopes.contiguous()
        _lib.require_one_device(q, k, v, segment_ids, prefix_lengths, distance_slopes)
        if (S + 64) * q.shape[3] >= 1 << 30:
            raise ValueError(f"a head's tensors must stay below 2 GiB, got {tuple(q.shape)}")
        if q.shape[0] * q.shape[1] * (-(-S // 64)) > 1 << 22:
            raise ValueError(f"batch x heads x (seq / 64, rounded up) must be at most 2^22, got {tuple(q.shape)}")
        scale = q.shape[3] ** -0.5 if config.softmax_scale is None else config.softmax_scale
        call = (q, k, v, segment_ids, prefix_lengths, distance_slopes, float(scale), float(config.score_cap or 0.0))
        if _lib.needs_autograd(q, k, v):
            return _ScoredAttention.apply(*call)
        return _forward(*call, False)[3]

    return attention
