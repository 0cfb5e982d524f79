"""What ``layer_norm``, ``adamw_tensors`` and the scored attention refuse, on the host, before any launch (CPU tensors)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gptrig import _lib
from gptrig.nn import layer_norm
from gptrig.optim import adamw_tensors, adamw_tensors_state

BF16, F32 = torch.bfloat16, torch.float32


def test_layer_norm_refusals():
    x, s = torch.zeros((2, 8)), torch.ones(8)
    for bad in (x.half(), x.double(), x.int()):
        with pytest.raises(TypeError, match="bfloat16 or float32"):
            layer_norm(bad, s)
    with pytest.raises(TypeError, match="both"):
        layer_norm(x, s, torch.zeros(8, dtype=BF16))
    with pytest.raises(TypeError, match="both"):
        layer_norm(x, s.half())
    for bad in (torch.ones(7), torch.ones((1, 8)), torch.ones(())):
        with pytest.raises(ValueError, match=r"must be \[8\]"):
            layer_norm(x, bad)
        with pytest.raises(ValueError, match=r"must be \[8\]"):
            layer_norm(x, s, bad)
    for bad in (torch.zeros(()), torch.zeros((3, 0))):
        with pytest.raises(ValueError, match="last dimension"):
            layer_norm(bad, s)
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            layer_norm(x, s, eps=eps)
    with pytest.raises(RuntimeError, match="GPU"):
        layer_norm(x, s)


def step(n=2, bits=32, **change):
    shapes = [(3, 4), (300,)][:n]
    p = [torch.zeros(s) for s in shapes]
    args = dict(params=p, grads=[torch.zeros(s) for s in shapes], hparams=torch.zeros((n, 3)), lr=0.1, beta1=0.9, beta2=0.95,
                step=1, **adamw_tensors_state(p, bits))
    args.update(change)
    adamw_tensors(**args)


def test_adamw_tensors_refusals():
    with pytest.raises(RuntimeError, match="GPU"):
        step()
    with pytest.raises(RuntimeError, match="GPU"):
        step(bits=8)
    with pytest.raises(ValueError, match="at least one"):
        step(params=[])
    with pytest.raises(ValueError, match="grads has 1"):
        step(grads=[torch.zeros((3, 4))])
    with pytest.raises(ValueError, match=r"grads\[1\] must be"):
        step(grads=[torch.zeros((3, 4)), torch.zeros(299)])
    with pytest.raises(ValueError, match=r"grads\[0\] must be contiguous"):
        step(grads=[torch.zeros((4, 3)).t(), torch.zeros(300)])
    with pytest.raises(TypeError, match="grads must all"):
        step(grads=[torch.zeros((3, 4)), torch.zeros(300, dtype=BF16)])
    with pytest.raises(TypeError, match="params must all"):
        step(params=[torch.zeros((3, 4), dtype=BF16), torch.zeros(300, dtype=BF16)])
    with pytest.raises(TypeError, match="exp_avg must all"):
        step(exp_avg=[torch.zeros((3, 4), dtype=BF16), torch.zeros(300, dtype=BF16)])
    with pytest.raises(TypeError, match="exp_avg_sq must all"):
        step(exp_avg_sq=adamw_tensors_state([torch.zeros((3, 4)), torch.zeros(300)], 8)["exp_avg_sq"])
    with pytest.raises(ValueError, match="come with"):
        step(bits=8, exp_avg_scale=None)
    with pytest.raises(ValueError, match="come with"):
        step(exp_avg_scale=[torch.zeros(1), torch.zeros(2)])
    with pytest.raises(ValueError, match=r"exp_avg_sq_scale\[1\] must be \(2,\)"):
        step(bits=8, exp_avg_sq_scale=[torch.zeros(1), torch.zeros(1)])
    with pytest.raises(TypeError, match="shadow"):
        step(shadow=[torch.zeros((3, 4)), torch.zeros(300)])
    for bad in (torch.zeros((2, 2)), torch.zeros((1, 3)), torch.zeros((2, 3), dtype=torch.float64), torch.zeros((3, 2)).t()):
        with pytest.raises(ValueError, match="hparams"):
            step(hparams=bad)
    for bad in (torch.zeros(2), torch.zeros(1, dtype=torch.float64)):
        with pytest.raises(ValueError, match="clip_scale"):
            step(clip_scale=bad)
    for name in ("beta1", "beta2"):
        for bad in (1.0, -0.1, float("nan")):
            with pytest.raises(ValueError, match="beta1"):
                step(**{name: bad})
    for bad in (0, 2 ** 31, 2 ** 32 + 1):
        with pytest.raises(ValueError, match="counts from 1"):
            step(step=bad)
    for bad in (-1, 2 ** 32):
        with pytest.raises(ValueError, match="seed"):
            step(seed=bad)
    p = torch.zeros(300)
    with pytest.raises(ValueError, match="8 or 32"):
        adamw_tensors_state([p], 16)


def test_entry_points_refuse_on_the_host():
    lib = _lib.lib()
    at = ctypes.c_void_p(1 << 12)
    odd = ctypes.c_void_p((1 << 12) + 1)
    fwd = lib.gptrig_layernorm_fwd
    assert fwd(None, 8, 0, at, None, 1, at, None, None, 2, 8, 1e-5, None) == -1
    assert fwd(at, 8, 2, at, None, 1, at, None, None, 2, 8, 1e-5, None) == -3
    assert fwd(at, 8, 0, at, None, 1, at, at, None, 2, 8, 1e-5, None) == -1
    for ld, rows, d in ((-1, 2, 8), (8, -1, 8), (8, 2, 0), (8, 1 << 31, 8), (8, 2, (1 << 30) + 1)):
        assert fwd(at, ld, 0, at, None, 1, at, None, None, rows, d, 1e-5, None) == -2
    assert fwd(at, 8, 0, at, None, 1, at, None, None, 2, 8, float("nan"), None) == -2
    assert fwd(odd, 8, 0, at, None, 1, at, None, None, 2, 8, 1e-5, None) == -2
    assert fwd(at, 8, 0, at, None, 1, at, None, None, 0, 8, 1e-5, None) == 0
    bwd = lib.gptrig_layernorm_bwd
    need = lib.gptrig_layernorm_bwd_workspace_bytes(100, 64, 0)
    assert need >= 2 * 64 * 4
    assert bwd(at, 64, at, 64, 0, at, 1, at, at, None, at, None, None, 0, 100, 64, None) == -1
    assert bwd(at, 64, at, 64, 0, at, 1, at, at, None, at, None, at, need - 1, 100, 64, None) == -6
    assert bwd(at, 64, at, 64, 0, at, 1, at, at, None, None, None, None, 0, 100, 64, None) == 0
    adamw = lib.gptrig_adamw_tensors
    row = (ctypes.c_int64 * 8)(1 << 12, 1 << 12, 1 << 12, 1 << 12, 0, 0, 0, 100)
    assert adamw(None, 1, 1, 32, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -1
    assert adamw(row, 1, 1, 8, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -1  # no scales
    assert adamw(row, 1, 2, 32, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -3
    assert adamw(row, 1, 1, 16, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -4
    assert adamw(row, 1, 1, 32, at, 0.1, 1.0, 0.95, 1, None, 0, None) == -2
    assert adamw(row, 1, 1, 32, at, 0.1, 0.9, 0.95, 0, None, 0, None) == -2
    assert adamw(row, 0, 1, 32, at, 0.1, 0.9, 0.95, 1, None, 0, None) == 0
    assert lib.gptrig_status_string(-7) == b"buffers that the call writes overlap"
    rows = (ctypes.c_int64 * 16)(*[k << 20 for k in range(1, 8)], 1000, *[k << 20 for k in range(11, 18)], 1000)
    for state, first, second in ((32, 0, 8), (32, 0, 2), (32, 3, 11), (8, 4, 5), (8, 10, 13), (32, 6, 0), (8, 6, 14)):
        for shift in (0, 4):
            bad = (ctypes.c_int64 * 16)(*rows)
            bad[second] = bad[first] + shift
            assert adamw(bad, 2, 1, state, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -7, (state, first, second, shift)
    for state, first, second in ((32, 0, 1), (32, 9, 2), (8, 1, 13), (8, 14, 1)):  # (gradients are read, not written)
        for shift in (0, 4):
            bad = (ctypes.c_int64 * 16)(*rows)
            bad[second] = bad[first] + shift
            assert adamw(bad, 2, 1, state, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -7, (state, first, second, shift)
    # A gradient that reaches over several arrays, the written one not next to it by its address.
    bad = (ctypes.c_int64 * 16)(*rows)
    bad[1], bad[9], bad[8] = 100 << 20, (100 << 20) + 4, (100 << 20) + 3992
    assert adamw(bad, 2, 1, 32, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -7
    rows[7] = (1 << 35) + 1
    assert adamw(rows, 2, 1, 32, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -2
    many = (ctypes.c_int64 * (8 * 200))(*[v for i in range(200) for v in (*[(i * 8 + k + 1) << 20 for k in range(7)], 10)])
    many[8 * 199] = many[8 * 3 + 2] + 36
    assert adamw(many, 200, 1, 32, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -7
    row[0] += 2
    assert adamw(row, 1, 1, 32, at, 0.1, 0.9, 0.95, 1, None, 0, None) == -2


def test_scored_attention_refusals():
    from gptrig.kernels import ScoredAttentionConfig, make_scored_attention

    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="softmax_scale"):
            ScoredAttentionConfig(softmax_scale=bad)
        with pytest.raises(ValueError, match="score_cap"):
            ScoredAttentionConfig(score_cap=bad)
    with pytest.raises(ValueError, match="score_cap"):
        ScoredAttentionConfig(score_cap=1001.0)
    attention = make_scored_attention(ScoredAttentionConfig(score_cap=30.0))
    q = torch.zeros((2, 4, 16, 64), dtype=BF16)
    k = torch.zeros((2, 2, 16, 64), dtype=BF16)
    with pytest.raises(ValueError, match="rank-4"):
        attention(q[0], k, k)
    for bad in (k[:1], k[:, :, :8], k[..., :32], torch.zeros((2, 3, 16, 64), dtype=BF16), torch.zeros((2, 8, 16, 64), dtype=BF16)):
        with pytest.raises(ValueError, match="kv_heads"):
            attention(q, bad, bad)
    with pytest.raises(ValueError, match="kv_heads"):
        attention(q, k, k[:, :1])
    with pytest.raises(ValueError, match="nonzero"):
        attention(q[:, :, :0], k[:, :, :0], k[:, :, :0])
    for D in (136, 60):
        t = torch.zeros((1, 1, 4, D), dtype=BF16)
        with pytest.raises(ValueError, match="head_dim"):
            attention(t, t, t)
    with pytest.raises(TypeError, match="bfloat16"):
        attention(q.half(), k.half(), k.half())
    with pytest.raises(TypeError, match="bfloat16"):
        attention(q, k, k.float())
    for bad in (torch.zeros((2, 16)), torch.zeros((2, 16), dtype=torch.bool)):
        with pytest.raises(TypeError, match="segment_ids"):
            attention(q, k, k, bad)
    with pytest.raises(ValueError, match="segment_ids"):
        attention(q, k, k, torch.zeros((2, 15), dtype=torch.int32))
    with pytest.raises(TypeError, match="prefix_lengths"):
        attention(q, k, k, prefix_lengths=torch.zeros(2))
    with pytest.raises(ValueError, match="prefix_lengths"):
        attention(q, k, k, prefix_lengths=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(TypeError, match="distance_slopes"):
        attention(q, k, k, distance_slopes=torch.zeros(4, dtype=BF16))
    with pytest.raises(ValueError, match="distance_slopes"):
        attention(q, k, k, distance_slopes=torch.zeros(2))
    with pytest.raises(ValueError, match="constants"):
        attention(q, k, k, distance_slopes=torch.zeros(4, requires_grad=True))
    with pytest.raises(RuntimeError, match="GPU"):
        attention(q, k, k)
    wide = torch.zeros((1, 1, 1, 8), dtype=BF16).expand(1 << 20, 5, 1, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        attention(wide, wide, wide)


def test_scored_attention_entry_points_refuse_on_the_host():
    lib = _lib.lib()
    at, odd = ctypes.c_void_p(1 << 12), ctypes.c_void_p((1 << 12) + 8)

    def fwd(q=at, o=at, B=1, H=4, Hk=2, S=16, D=64, strides=None, scale=0.125, cap=0.0):
        return lib.gptrig_scored_attn_fwd(q, at, at, None, None, None, None, o, None, None, B, H, Hk, S, D, strides, scale, cap, None)

    assert fwd(q=None) == -1 and fwd(q=odd) == -2
    assert fwd(Hk=3) == -2 and fwd(Hk=0) == -2 and fwd(S=0) == -2 and fwd(B=-1) == -2
    assert fwd(D=60) == -2 and fwd(D=136) == -4
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert fwd(scale=scale) == -2
    for cap in (-1.0, 1001.0, float("nan"), 1e-42):
        assert fwd(cap=cap) == -2
    assert fwd(B=1 << 20, H=5, Hk=5, S=1) == -2 and fwd(B=1 << 30, S=1) == -2 and fwd(B=1 << 14, S=(1 << 14) + 1) == -2
    assert fwd(S=1 << 24) == -2  # a head's slice past 2 GiB
    for change in (4, -64):
        st = (ctypes.c_int64 * 12)(*[4096, 1024, 64] * 4)
        st[2] = change
        assert fwd(strides=st) == -2
    assert lib.gptrig_scored_attn_plan_bytes(1, 4, 2, 16, 64) == 0
    need = lib.gptrig_scored_attn_plan_bytes(4, 12, 12, 2000, 64)
    assert need >= 2 * 4 * 16 * 4
    plan = lib.gptrig_scored_attn_plan
    assert plan(at, at, at, need, 1, 4, 2, 16, 64, None) == -2 and plan(at, at, None, need, 4, 12, 12, 2000, 64, None) == -1
    assert plan(at, at, at, need - 1, 4, 12, 12, 2000, 64, None) == -6 and plan(at, at, odd, need, 4, 12, 12, 2000, 64, None) == -2
    big = ctypes.c_size_t(1 << 40)
    need = lib.gptrig_scored_attn_bwd_workspace_bytes(1, 4, 2, 16, 64)
    assert need >= 4 * 16 * 4

    def bwd(ws=at, size=big, lse=at, dv=at, low=at):
        return lib.gptrig_scored_attn_bwd(at, at, at, at, at, low, lse, None, None, None, None, at, at, dv, ws, size, 1, 4, 2, 16, 64, None,
                                          0.125, 0.0, None)

    assert bwd(ws=None) == -1 and bwd(lse=None) == -1 and bwd(low=None) == -1 and bwd(low=odd) == -2 and bwd(dv=None) == -1
    assert bwd(size=need - 1) == -6 and bwd(ws=odd) == -2
