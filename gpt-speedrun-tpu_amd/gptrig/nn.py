"""Model primitives on gfx950, mirroring ``rig/nn.py``.

``rms_norm``, ``apply_rotary`` and ``gelu`` run the HIP kernels of
``csrc/elementwise.hip`` with hand-written backward passes, ``layer_norm``,
``embedding`` and ``gated_mlp`` (not in ``rig/nn.py``) those of
``csrc/layernorm.hip``, ``embedding.hip`` and ``gated_mlp.hip``; ``linear`` is a
plain library GEMM (hipBLASLt through torch) with the reference's bf16
rounding points.
"""

from __future__ import annotations

import functools
from typing import Any, Mapping

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _lib

BF16 = torch.bfloat16


def normal(rng: np.random.Generator, shape: tuple[int, ...], scale: float) -> np.ndarray:
    """``rig/nn.py:20-23``: float32 standard normal times a float32 scale."""

    return rng.standard_normal(shape, dtype=np.float32) * np.float32(scale)


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x.reshape(-1, x.shape[-1]).contiguous()


def rmsnorm_forward(x2: torch.Tensor, scale_bf16: torch.Tensor, out: torch.Tensor | None = None):
    rows, d = x2.shape
    y = torch.empty_like(x2) if out is None else out
    rstd = torch.empty(rows, dtype=torch.float32, device=x2.device)
    _lib.call("gptrig_rmsnorm_fwd", x2.data_ptr(), scale_bf16.data_ptr(), y.data_ptr(), rstd.data_ptr(), rows, d,
              _lib.stream())
    return y, rstd


def add_rmsnorm_forward(x2: torch.Tensor, branch: torch.Tensor, branch_scale: float, scale_bf16: torch.Tensor,
                        sum_out: torch.Tensor | None = None, out: torch.Tensor | None = None,
                        branch_bias: torch.Tensor | None = None):
    """``s = x + bf16(branch * branch_scale)`` then ``rms_norm(s)``: the block's
    residual add and the norm after it in one pass.  Returns ``(s, y, rstd)``.

    ``branch_bias`` (bf16 ``[d]``): ``branch`` is a linear's bf16 GEMM output
    without its bias, which is added here with its own rounding
    (``rig/nn.py:55-56``) before the residual add."""

    rows, d = x2.shape
    s = torch.empty_like(x2) if sum_out is None else sum_out
    y = torch.empty_like(x2) if out is None else out
    rstd = torch.empty(rows, dtype=torch.float32, device=x2.device)
    _lib.call("gptrig_add_bias_rmsnorm_fwd", x2.data_ptr(), branch.data_ptr(), _lib.ptr(branch_bias),
              float(branch_scale), scale_bf16.data_ptr(), s.data_ptr(), y.data_ptr(), rstd.data_ptr(), rows, d,
              _lib.stream())
    return s, y, rstd


def rmsnorm_backward(dy2, x2, scale_bf16, rstd, dscale: torch.Tensor | None = None, accumulate: bool = False,
                     dresidual: torch.Tensor | None = None, out: torch.Tensor | None = None):
    rows, d = x2.shape
    dx = torch.empty_like(x2) if out is None else out
    if dscale is None:
        dscale = torch.empty(d, dtype=torch.float32, device=x2.device)
        accumulate = False
    ws = _lib.workspace(_lib.query("gptrig_rmsnorm_bwd_workspace_bytes", rows, d), x2.device)
    _lib.call("gptrig_rmsnorm_bwd", dy2.data_ptr(), x2.data_ptr(), scale_bf16.data_ptr(), rstd.data_ptr(),
              _lib.ptr(dresidual), dx.data_ptr(), dscale.data_ptr(), int(accumulate), ws.data_ptr(), ws.numel(),
              rows, d, _lib.stream())
    return dx, dscale


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale):
        x2 = _rows(x)
        s = scale.to(BF16).contiguous()
        y, rstd = rmsnorm_forward(x2, s)
        ctx.save_for_backward(x2, s, rstd)
        ctx.meta = (x.shape, scale.dtype)
        return y.reshape(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, s, rstd = ctx.saved_tensors
        shape, sdtype = ctx.meta
        dx, dscale = rmsnorm_backward(_rows(dy.to(BF16)), x2, s, rstd)
        return dx.reshape(shape), dscale.to(sdtype)


def rms_norm(x: torch.Tensor, scale: torch.Tensor, dtype: Any = BF16) -> torch.Tensor:
    """``rig/nn.py:26-33``: ``bf16(bf16(x*rsqrt(mean(x^2)+1e-5)) * bf16(scale))``."""

    if dtype != BF16 or x.dtype != BF16:
        raise TypeError("the HIP rms_norm computes bfloat16 activations")
    _lib.require_device(x, scale)
    return _RMSNorm.apply(x, scale)


_TYPES = {BF16: 0, torch.float32: 1}  # GPTRIG_TYPE_* of include/gptrig.h
_LEAST_F32, _MOST_F32 = 2.0 ** -149, (2.0 - 2.0 ** -23) * 2.0 ** 127


def _strided_rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` as ``[rows, width]`` with unit stride along the width, without a copy where its strides allow it."""

    if x.ndim != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


@functools.lru_cache(maxsize=256)
def _layer_norm_workspace_bytes(rows: int, width: int, kind: int) -> int:
    return _lib.query("gptrig_layernorm_bwd_workspace_bytes", rows, width, kind)


def _layer_norm_forward(x, scale, bias, eps: float, keep: bool):
    """``y``, and what the backward needs (``None`` for the statistics unless ``keep``)."""

    x2 = _strided_rows(x)
    scale = scale.contiguous()
    bias = None if bias is None else bias.contiguous()
    rows, d = x2.shape
    y = torch.empty_like(x2) if x2.is_contiguous() else torch.empty((rows, d), dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if keep else None
    mean = stats.data_ptr() if keep else None
    if rows:
        _lib.call_on(x.get_device(), "gptrig_layernorm_fwd", x2.data_ptr(), x2.stride(0), _TYPES[x.dtype],
                     scale.data_ptr(), _lib.ptr(bias), _TYPES[scale.dtype], y.data_ptr(), mean,
                     mean + 4 * rows if keep else None, rows, d, eps)
    return y if x.ndim == 2 else y.reshape(x.shape), x2, scale, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, bias, eps):
        y, *kept = _layer_norm_forward(x, scale, bias, eps, True)
        ctx.save_for_backward(*kept)
        ctx.shape = x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_layer_norm_backward_once if torch.is_grad_enabled() else _layer_norm_backward)(ctx, dy)


def _layer_norm_backward(ctx, dy):
    x2, scale, stats = ctx.saved_tensors
    need_x, need_s, need_b, _ = ctx.needs_input_grad
    rows, d = x2.shape
    dev = x2.device
    if not rows:
        zero = torch.zeros(d, dtype=scale.dtype, device=dev)
        return (dy.reshape(ctx.shape) if need_x else None, zero if need_s else None, zero.clone() if need_b else None,
                None)
    dy2 = _strided_rows(dy)
    dx = None
    if need_x:
        dx = torch.empty_like(x2) if x2.is_contiguous() else torch.empty((rows, d), dtype=x2.dtype, device=dev)
    dscale = torch.empty_like(scale) if need_s else None
    dbias = torch.empty_like(scale) if need_b else None
    kind, ws, size = _TYPES[x2.dtype], None, 0
    if need_s or need_b:
        size = _layer_norm_workspace_bytes(rows, d, kind)
        ws = _lib.workspace(size, dev)
    mean = stats.data_ptr()
    _lib.call_on(x2.get_device(), "gptrig_layernorm_bwd", dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0),
                 kind, scale.data_ptr(), _TYPES[scale.dtype], mean, mean + 4 * rows, _lib.ptr(dx), _lib.ptr(dscale),
                 _lib.ptr(dbias), _lib.ptr(ws), size, rows, d)
    return dx if dx is None or len(ctx.shape) == 2 else dx.reshape(ctx.shape), dscale, dbias, None


_layer_norm_backward_once = once_differentiable(_layer_norm_backward)


def layer_norm(x: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None, *,
               eps: float = 1.0e-5) -> torch.Tensor:
    """Layer normalisation over the last dimension: ``(x - mean) / sqrt(variance +
    eps) * scale + bias``, computed in float32 and rounded once to ``x``'s type.

    ``x``: bfloat16 or float32 of any shape and strides; ``scale`` and ``bias``:
    ``[width]``, both float32 or both bfloat16.  Differentiable once in all three;
    the gradients of ``scale`` and ``bias`` are summed in float32, in a fixed order.
    """

    if x.dtype not in _TYPES:
        raise TypeError(f"the HIP layer_norm takes bfloat16 or float32 activations, got {x.dtype}")
    if scale.dtype not in _TYPES or (bias is not None and bias.dtype != scale.dtype):
        raise TypeError(f"scale and bias must both be float32 or both bfloat16, got {scale.dtype} and "
                        f"{None if bias is None else bias.dtype}")
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"x needs a last dimension to normalise over, got {tuple(shape)}")
    width = shape[-1]
    if scale.shape != (width,) or (bias is not None and bias.shape != (width,)):
        raise ValueError(f"scale and bias must be [{width}], got {tuple(scale.shape)} and "
                         f"{None if bias is None else tuple(bias.shape)}")
    if width > 1 << 30 or x.numel() // width >= 1 << 31:
        raise ValueError(f"at most 2^30 wide and fewer than 2^31 rows, got {tuple(shape)}")
    if not (eps == 0 or _LEAST_F32 <= eps <= _MOST_F32):
        raise ValueError(f"eps must be 0 or a positive float32, got {eps}")
    _lib.require_one_device(x, scale, bias)
    if _lib.needs_autograd(x, scale, bias):
        return _LayerNorm.apply(x, scale, bias, eps)
    return _layer_norm_forward(x, scale, bias, eps, False)[0]


@functools.lru_cache(maxsize=256)
def _embedding_workspace_bytes(tokens: int, width: int, vocab: int) -> int:
    return _lib.query("gptrig_scaled_embedding_bwd_workspace_bytes", tokens, width, vocab)


def _embedding_forward(tokens, table, scale: float, dtype):
    """``y``, and the tokens as the kernels read them."""

    tokens = tokens.contiguous()
    if table.stride(1) != 1 and table.shape[1] != 1:
        table = table.contiguous()
    vocab, width = table.shape
    y = torch.empty((*tokens.shape, width), dtype=dtype, device=table.device)
    if tokens.numel():
        _lib.call_on(table.get_device(), "gptrig_scaled_embedding_fwd", tokens.data_ptr(),
                     int(tokens.dtype == torch.int64), table.data_ptr(), table.stride(0), _TYPES[table.dtype],
                     y.data_ptr(), _TYPES[dtype], tokens.numel(), width, vocab, scale)
    return y, tokens


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, dtype):
        y, tokens = _embedding_forward(tokens, table, scale, dtype)
        ctx.save_for_backward(tokens)
        ctx.meta = (table.shape, table.dtype, scale)
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_embedding_backward_once if torch.is_grad_enabled() else _embedding_backward)(ctx, dy)


def _embedding_backward(ctx, dy):
    (tokens,) = ctx.saved_tensors
    (vocab, width), kind, scale = ctx.meta
    n, dev = tokens.numel(), dy.device
    dtable = torch.empty((vocab, width), dtype=kind, device=dev)
    dy2 = _strided_rows(dy) if n else dy
    size = _embedding_workspace_bytes(n, width, vocab)
    ws = _lib.workspace(size, dev)
    _lib.call_on(dev.index, "gptrig_scaled_embedding_bwd", tokens.data_ptr(), int(tokens.dtype == torch.int64),
                 dy2.data_ptr(), dy2.stride(0) if n else width, _TYPES[dy.dtype], dtable.data_ptr(), _TYPES[kind], n,
                 width, vocab, scale, ws.data_ptr(), size)
    return dtable, None, None, None


_embedding_backward_once = once_differentiable(_embedding_backward)


def embedding(tokens: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0, dtype: Any = BF16) -> torch.Tensor:
    """``scale * table[tokens]`` in ``dtype``: the product in float32, rounded once.

    ``tokens``: int32 or int64 of any shape; a token outside ``[0, vocab)``, such
    as -1 for padding, gives a row of zeros and takes no part in the gradient.
    ``table``: float32 or bfloat16 ``[vocab, width]``, any row stride; ``dtype``:
    bfloat16 or float32; ``scale``: a number (read at the call; one that asks for a
    gradient is refused).  Differentiable once in ``table``: the gradient has its
    shape and type, each row the float32 sum of its tokens' gradients in a fixed
    order, so that the same call gives the same bits.  (``train.GPTTrainer`` keeps a
    lookup of its own, the reference's: tokens clamped, the gradient added with
    atomics.)
    """

    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    if table.dtype not in _TYPES or dtype not in _TYPES:
        raise TypeError(f"the HIP embedding takes and gives bfloat16 or float32, got {table.dtype} and {dtype}")
    if table.ndim != 2 or not table.shape[0] or not table.shape[1]:
        raise ValueError(f"table must be [vocab, width], got {tuple(table.shape)}")
    if table.shape[0] >= 2 ** 31 - 1 or table.shape[1] > 1 << 24 or tokens.numel() >= 2 ** 31 - 65536:
        raise ValueError(f"at most 2^31 - 2 rows of 2^24 columns and fewer than 2^31 - 65536 tokens, got "
                         f"{tuple(table.shape)} and {tuple(tokens.shape)}")
    if isinstance(scale, torch.Tensor) and _lib.needs_autograd(scale):
        raise RuntimeError("embedding has no derivative in scale: give it a number, or multiply the result")
    if not -_MOST_F32 <= scale <= _MOST_F32:
        raise ValueError(f"scale must be a finite float32, got {scale}")
    scale = float(scale)
    _lib.require_one_device(table, tokens)
    if _lib.needs_autograd(table):
        return _Embedding.apply(table, tokens, scale, dtype)
    return _embedding_forward(tokens, table, scale, dtype)[0]


_ACTIVATIONS = {"silu": 0, "gelu": 1}  # GPTRIG_SILU, GPTRIG_GELU
_MOST_WIDTH, _MOST_STRIDE = 1 << 20, 1 << 22


def _operand(x: torch.Tensor) -> torch.Tensor:
    """``x`` as ``[rows, width]`` in the layout that the matrix products read (unit stride along the width, rows that do
    not overlap, 16-byte alignment), without a copy where it has that."""

    if x.ndim != 2:
        x = x.reshape(-1, x.shape[-1])
    rows, width = x.shape
    if x.stride(1) == 1 and x.data_ptr() % 16 == 0:
        ld = x.stride(0)
        if ld == width or rows > 1 and ld > width and ld % 8 == 0 and ld <= _MOST_STRIDE:
            return x
    return torch.empty((rows, width), dtype=x.dtype, device=x.device).copy_(x)


@functools.lru_cache(maxsize=256)
def _gated_kept_bytes(n: int, f: int) -> int:
    return _lib.query("gptrig_gated_mlp_kept_bytes", n, f)


@functools.lru_cache(maxsize=256)
def _gated_workspace_bytes(n: int, d: int, f: int, d_out: int) -> int:
    return _lib.query("gptrig_gated_mlp_bwd_workspace_bytes", n, d, f, d_out)


def _gated_forward(x, gate_up_w, down_w, activation: int, keep: bool):
    """``y``, and what the backward needs (``None`` for the projection's output unless ``keep``)."""

    x2, w, v = _operand(x), _operand(gate_up_w), _operand(down_w)
    n, d = x2.shape
    f, d_out = v.shape
    dev = x2.device
    h = torch.empty((n, f), dtype=BF16, device=dev)
    kept = _lib.workspace(_gated_kept_bytes(n, f), dev) if keep else None
    y = torch.empty((n, d_out), dtype=BF16, device=dev)
    if n:
        _lib.call_on(x2.get_device(), "gptrig_gated_mlp_fwd", x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0),
                     v.data_ptr(), v.stride(0), activation, _lib.ptr(kept), h.data_ptr(), y.data_ptr(), n, d, f,
                     d_out)
    return y if x.ndim == 2 else y.view(*x.shape[:-1], d_out), x2, w, v, kept, h


class _GatedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_up_w, down_w, activation):
        y, *kept = _gated_forward(x, gate_up_w, down_w, activation, True)
        ctx.save_for_backward(*kept)
        ctx.meta = (x.shape, activation)
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_gated_backward_once if torch.is_grad_enabled() else _gated_backward)(ctx, dy)


def _gated_backward(ctx, dy):
    x, w, v, kept, h = ctx.saved_tensors
    shape, activation = ctx.meta
    need_x, need_w, need_v, _ = ctx.needs_input_grad
    n, d = x.shape
    f, d_out = v.shape
    dev = x.device
    if not n:
        return (torch.zeros(shape, dtype=BF16, device=dev) if need_x else None,
                torch.zeros((d, 2 * f), dtype=BF16, device=dev) if need_w else None,
                torch.zeros((f, d_out), dtype=BF16, device=dev) if need_v else None, None)
    dy = _operand(dy)
    dx = torch.empty((n, d), dtype=BF16, device=dev) if need_x else None
    dw = torch.empty((d, 2 * f), dtype=BF16, device=dev) if need_w else None
    dv = torch.empty((f, d_out), dtype=BF16, device=dev) if need_v else None
    size = _gated_workspace_bytes(n, d, f, d_out)
    ws = _lib.workspace(size, dev)
    _lib.call_on(x.get_device(), "gptrig_gated_mlp_bwd", dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0),
                 w.data_ptr(), w.stride(0), v.data_ptr(), v.stride(0), activation, kept.data_ptr(), h.data_ptr(),
                 _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(dv), n, d, f, d_out, ws.data_ptr(), size)
    return None if dx is None else dx.view(shape), dw, dv, None


_gated_backward_once = once_differentiable(_gated_backward)


def gated_mlp(x: torch.Tensor, gate_up_w: torch.Tensor, down_w: torch.Tensor, *,
              activation: str = "silu") -> torch.Tensor:
    """A gated feed-forward block: ``(act(x @ gate) * (x @ up)) @ down_w`` with
    ``gate_up_w = [gate | up]``, ``act`` ``"silu"`` or ``"gelu"`` (tanh form).

    ``x``: bfloat16 ``[..., d]`` of any strides; ``gate_up_w`` ``[d, 2 * hidden]``
    and ``down_w`` ``[hidden, d_out]`` in bfloat16; widths are multiples of 8.  The
    sums are float32; the hidden values are held in bfloat16, for the backward both
    halves of the projection in 11 bits.  Differentiable once in all three, the
    gradients in bfloat16 and the same at every call.
    """

    for name, t in (("x", x), ("gate_up_w", gate_up_w), ("down_w", down_w)):
        if t.dtype != BF16:
            raise TypeError(f"the HIP gated_mlp computes bfloat16, got {name} of {t.dtype}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if not x.ndim or gate_up_w.ndim != 2 or down_w.ndim != 2 or gate_up_w.shape[0] != x.shape[-1] or (
            gate_up_w.shape[1] != 2 * down_w.shape[0]):
        raise ValueError(f"x, gate_up_w and down_w must be [..., d], [d, 2 * hidden] and [hidden, d_out], got "
                         f"{tuple(x.shape)}, {tuple(gate_up_w.shape)} and {tuple(down_w.shape)}")
    widths = (x.shape[-1], *down_w.shape)
    if any(w == 0 or w % 8 for w in widths) or max(widths[0], 2 * widths[1], widths[2]) > _MOST_WIDTH:
        raise ValueError(f"widths must be multiples of 8, and d, 2 * hidden and d_out at most 2^20, got {widths}")
    if x.numel() // widths[0] > 1 << 26:
        raise ValueError(f"at most 2^26 tokens, got {x.numel() // widths[0]}")
    _lib.require_one_device(x, gate_up_w, down_w)
    if _lib.needs_autograd(x, gate_up_w, down_w):
        return _GatedMLP.apply(x, gate_up_w, down_w, _ACTIVATIONS[activation])
    return _gated_forward(x, gate_up_w, down_w, _ACTIVATIONS[activation], False)[0]


_ROPE_TABLES: dict = {}


def rope_tables(seq: int, head_dim: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 cos/sin ``[seq, head_dim/2]`` built on the device (``rig/nn.py:43-47``)."""

    key = (seq, head_dim, str(device))
    if key not in _ROPE_TABLES:
        c = torch.empty((seq, head_dim // 2), dtype=BF16, device=device)
        s = torch.empty_like(c)
        _lib.call("gptrig_rope_table", c.data_ptr(), s.data_ptr(), seq, head_dim, _lib.stream())
        _ROPE_TABLES[key] = (c, s)
    return _ROPE_TABLES[key]


def rope_inplace(buf: torch.Tensor, row_stride: int, rows: int, seq: int, heads: int, head_dim: int,
                 backward: bool = False) -> None:
    c, s = rope_tables(seq, head_dim, buf.device)
    _lib.call("gptrig_rope_bwd" if backward else "gptrig_rope_fwd", buf.data_ptr(), int(row_stride), rows, seq,
              heads, head_dim, c.data_ptr(), s.data_ptr(), _lib.stream())


def bias_rope_inplace(buf: torch.Tensor, bias: torch.Tensor, seq: int, heads: int, head_dim: int) -> None:
    """In place on a ``[rows, cols]`` bf16 projection output without its bias:
    every column gets ``bf16(x + bias)`` (``rig/nn.py:55-56``), then the first
    ``heads * head_dim`` columns are rotated (``rig/nn.py:36-52``)."""

    rows, cols = buf.shape
    c, s = rope_tables(seq, head_dim, buf.device)
    _lib.call("gptrig_bias_rope_fwd", buf.data_ptr(), int(buf.stride(0)), rows, cols, bias.data_ptr(), seq, heads,
              head_dim, c.data_ptr(), s.data_ptr(), _lib.stream())


def _rotated(x: torch.Tensor, backward: bool) -> torch.Tensor:
    """The rotation of a bf16 BTHD tensor of any strides into a new contiguous one."""

    B, S, H, D = x.shape
    if x.numel() >= 2 ** 34:  # past the out-of-place pass's 32-bit chunk index
        y = x.contiguous().clone()
        rope_inplace(y, H * D, B * S, S, H, D, backward=backward)
        return y
    strides = x.stride()[:3]
    if x.stride(3) != 1 or any(s % 8 for s in strides) or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
        strides = (S * H * D, H * D, D)  # (dimensions of size 1 may keep any stride)
    y = torch.empty((B, S, H, D), dtype=x.dtype, device=x.device)
    if y.numel():
        c, s = rope_tables(S, D, x.device)
        _lib.call("gptrig_rope_copy", x.data_ptr(), *strides, y.data_ptr(), B, S, H, D, int(backward),
                  c.data_ptr(), s.data_ptr(), _lib.stream())
    return y


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return _rotated(x, False)

    @staticmethod
    def backward(ctx, dy):
        return _rotated(dy.to(BF16), True)


def apply_rotary(x: torch.Tensor) -> torch.Tensor:
    """``rig/nn.py:36-52``: interleaved base-10,000 RoPE on a BTHD tensor."""

    if x.shape[-1] % 2:
        raise ValueError("rotary attention requires an even head dimension")
    if x.dtype != BF16:
        raise TypeError("the HIP rotary kernel takes bfloat16")
    if x.shape[-1] % 8:
        raise ValueError("the HIP rotary kernel needs head_dim % 8 == 0")
    _lib.require_device(x)
    return _Rotary.apply(x)


class _Gelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        xc = x.contiguous()
        y = torch.empty_like(xc)
        _lib.call("gptrig_gelu_fwd", xc.data_ptr(), y.data_ptr(), xc.numel(), _lib.stream())
        ctx.save_for_backward(xc)
        return y

    @staticmethod
    def backward(ctx, dy):
        (xc,) = ctx.saved_tensors
        g = dy.to(BF16).contiguous()
        dx = torch.empty_like(xc)
        _lib.call("gptrig_gelu_bwd", g.data_ptr(), xc.data_ptr(), dx.data_ptr(), xc.numel(), _lib.stream())
        return dx


def gelu(x: torch.Tensor) -> torch.Tensor:
    """``jax.nn.gelu(approximate=True)`` (``recipes/reference/train.py:1171``)."""

    if x.dtype != BF16:
        raise TypeError("the HIP gelu kernel takes bfloat16")
    _lib.require_device(x)
    return _Gelu.apply(x)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, dtype: Any = BF16) -> torch.Tensor:
    """``rig/nn.py:55-56``: ``x @ W.astype(dtype) + b.astype(dtype)`` (a plain
    library GEMM; bf16 product rounded, then the bf16 bias add)."""

    return torch.matmul(x.to(dtype), weight.to(dtype)) + bias.to(dtype)


def parameter_count(params: Any) -> int:
    """``rig/nn.py:59-60``."""

    if isinstance(params, Mapping):
        return sum(parameter_count(v) for v in params.values())
    if isinstance(params, (list, tuple)):
        return sum(parameter_count(v) for v in params)
    return int(params.numel() if isinstance(params, torch.Tensor) else np.asarray(params).size)
