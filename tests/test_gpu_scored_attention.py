"""``gptrig.kernels.make_scored_attention`` against the formula in 64 bits.

Tolerances, derived from the arithmetic.  bfloat16 roundings are off by at most
2^-8 of the value, with a deviation of at most 2^-8 / sqrt(3): of P for its product
with v (and do), of dU for its products with k and q, and of each result; delta = o .
do is computed from the rounded o.  Float32 errors: a score by ``E`` = (D + 16) 2^-24
of the magnitudes of its products, 2^-20 of the cap and 2^-22 of the bias, and 2^-20
of its exponential.  Every value has to be within the sum of the worst cases
(``worst``), and the 2-norm of a tensor's error within twice its deviation
(``deviation``) and the float32 share, which one pair too many in each row would
break.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
R = 2.0 ** -8
V3 = R * R / 3


def attend(cap=None, scale=None):
    from gptrig.kernels import ScoredAttentionConfig, make_scored_attention

    return make_scored_attention(ScoredAttentionConfig(softmax_scale=scale, score_cap=cap))


def inputs(B, H, Hk, S, D, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    make = lambda h: (torch.randn((B, h, S, D), generator=g) * size).to(BF16).to(DEV)  # noqa: E731
    return make(H), make(Hk), make(Hk), torch.randn((B, H, S, D), generator=g).to(BF16).to(DEV)


def visible(B, S, seg=None, prefix=None):
    at = torch.arange(S, device=DEV)
    vis = (at[None, :] <= at[:, None]).expand(B, S, S)
    if prefix is not None:
        vis = vis | (at[None, None, :] < prefix[:, None, None])
    if seg is not None:
        vis = vis & (seg[:, :, None] == seg[:, None, :])
    return vis[:, None]


def reference(q, k, v, do, cap=None, scale=None, seg=None, prefix=None, slopes=None):
    """{name: (value, worst, variance, float32 share)} of o, dq, dk and dv."""

    B, H, S, D = q.shape
    Hk = k.shape[1]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    q, do = q.to(F64), do.to(F64)
    k, v = (t.to(F64).repeat_interleave(G, dim=1) for t in (k, v))
    mm = torch.matmul
    u = mm(q, k.transpose(-1, -2).contiguous()) * scale
    size = mm(q.abs(), k.abs().transpose(-1, -2).contiguous()) * scale
    E = (D + 16) * 2.0 ** -24 * size + 2.0 ** -20
    t1 = torch.ones_like(u)
    s = u
    if cap:
        t = torch.tanh(u / cap)
        s, t1 = cap * t, 1 - t * t
        E = E + 2.0 ** -20 * cap
    if slopes is not None:
        at = torch.arange(S, device=DEV, dtype=F64)
        bias = slopes.to(F64)[:, None, None] * (at[:, None] - at[None, :]).abs()
        s = s - bias
        E = E + 2.0 ** -22 * bias.abs()
    s = s.masked_fill(~visible(B, S, seg, prefix), -math.inf)
    P = torch.softmax(s, -1)
    PE = P * E
    PE = PE + P * PE.sum(-1, keepdim=True)  # the float32 error of P
    o = mm(P, v)
    fo = mm(PE, v.abs()) + 2.0 ** -20 * mm(P, v.abs())
    wo = R * (mm(P, v.abs()) + o.abs()) * (1 + 4 * R) + fo
    vo = V3 * (mm(P * P, v * v) + o * o)
    out = {"o": (o, wo, vo, fo)}
    vt = v.transpose(-1, -2).contiguous()
    dP = mm(do, vt)
    delta = (do * o).sum(-1, keepdim=True)
    fdelta = (D + 16) * 2.0 ** -24 * (do * o).abs().sum(-1, keepdim=True) + (fo * do.abs()).sum(-1, keepdim=True)
    wdelta = (wo * do.abs()).sum(-1, keepdim=True) + fdelta
    vdelta = (vo * do * do).sum(-1, keepdim=True)
    fP = (D + 16) * 2.0 ** -24 * mm(do.abs(), vt.abs())
    dU = P * (dP - delta) * t1
    edge = 2.0 ** -20 * P * (dP - delta).abs()  # of 1 - tanh^2, and the subtraction
    f = (PE * (dP - delta).abs() + P * (fP + fdelta)) * t1 + edge
    w = R * dU.abs() * (1 + 4 * R) + f + P * t1 * wdelta
    kk, qq = k, q
    tr = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    dq = scale * mm(dU, kk)
    out["dq"] = (dq, scale * mm(w, kk.abs()) * (1 + 4 * R) + R * dq.abs() * (1 + R),
                 scale ** 2 * (V3 * mm(dU * dU, kk * kk) + vdelta * mm(P * t1, kk).square()) + V3 * dq * dq,
                 scale * mm(f, kk.abs()) + 2.0 ** -18 * scale * mm(dU.abs(), kk.abs()))
    dk = scale * mm(tr(dU), qq)
    dv = mm(tr(P), do)
    join = lambda x: x.reshape(B, Hk, G, S, D).sum(2)  # noqa: E731
    dk, dv = join(dk), join(dv)
    out["dk"] = (dk, join(scale * mm(tr(w), qq.abs())) * (1 + 4 * R) + R * dk.abs() * (1 + R),
                 join(scale ** 2 * (V3 * mm(tr(dU * dU), qq * qq) + mm(tr((P * t1).square()), vdelta * qq * qq)))
                 + V3 * dk * dk, join(scale * (mm(tr(f), qq.abs()) + 2.0 ** -18 * mm(tr(dU.abs()), qq.abs()))))
    fv = join(mm(tr(PE), do.abs()) + 2.0 ** -18 * mm(tr(P), do.abs()))
    out["dv"] = (dv, join(mm(tr(R * P), do.abs())) * (1 + 4 * R) + fv + R * dv.abs() * (1 + R),
                 join(V3 * mm(tr(P * P), do * do)) + V3 * dv * dv, fv)
    return out


def check(name, got, want):
    value, worst, variance, share = want
    assert got.shape == value.shape and got.dtype == BF16, name
    off = (got.to(F64) - value).abs()
    assert bool((off <= worst + 1e-30).all()), f"{name}: {float((off - worst).max())} past the worst case"
    limit = 2 * float(variance.sum().sqrt()) + float(share.norm())
    assert float(off.norm()) <= limit + 1e-30, f"{name}: 2-norm {float(off.norm())} against {limit}"


def run(q, k, v, do, cap=None, scale=None, seg=None, prefix=None, slopes=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = attend(cap, scale)(*leaves, seg, prefix_lengths=prefix, distance_slopes=slopes)
    grads = torch.autograd.grad(o, leaves, do)
    torch.cuda.synchronize()
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)))


def compare(q, k, v, do, **options):
    got, want = run(q, k, v, do, **options), reference(q, k, v, do, **options)
    for name in got:
        check(name, got[name], want[name])
    return got


def documents(B, S, mean, seed=5):
    g = torch.Generator().manual_seed(seed)
    return torch.cumsum(torch.rand((B, S), generator=g) < 1.0 / mean, 1).to(torch.int32).to(DEV)


def slopes_of(H):
    return 2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEV, dtype=F32) / H)


@pytest.mark.parametrize("S", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 200, 257, 500])
@pytest.mark.parametrize("D", [64, 128])
def test_lengths(S, D):
    print(f"scored attention S={S} D={D}", flush=True)
    compare(*inputs(2, 2, 2, S, D, seed=S), cap=20.0)
    compare(*inputs(1, 2, 1, S, D, seed=S + 1), slopes=slopes_of(2))


OPTIONS = [dict(), dict(cap=30.0), dict(slopes=True), dict(cap=5.0, slopes=True), dict(seg=40), dict(cap=50.0, seg=9),
           dict(slopes=True, seg=70), dict(cap=15.0, slopes=True, seg=1), dict(prefix=True), dict(cap=30.0, prefix=True),
           dict(slopes=True, prefix=True), dict(cap=10.0, slopes=True, prefix=True, seg=60), dict(prefix=True, seg=100)]


def resolve(options, B, H, S):
    o = dict(options)
    if "slopes" in o:
        o["slopes"] = slopes_of(H)
    if "seg" in o:
        o["seg"] = documents(B, S, o["seg"])
    if "prefix" in o:
        o["prefix"] = torch.tensor([0, S, 37, S // 2, 129, -4, S + 100][:B], dtype=torch.int32, device=DEV)
    return o


@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("D", [64, 128])
def test_every_mask_and_score(options, D):
    print(f"scored attention {options} D={D}", flush=True)
    B, H, S = 4, 4, 300
    compare(*inputs(B, H, 2, S, D, seed=3), **resolve(options, B, H, S))


@pytest.mark.parametrize("D", [8, 24, 40, 56, 72, 80, 96, 120])
def test_head_dims(D):
    print(f"scored attention D={D}", flush=True)
    compare(*inputs(2, 3, 3, 150, D, seed=D), **resolve(dict(cap=20.0, slopes=True, prefix=True), 2, 3, 150))


@pytest.mark.parametrize("H,Hk", [(1, 1), (8, 1), (6, 2), (6, 3), (12, 4)])
def test_shared_heads(H, Hk):
    print(f"scored attention H={H} Hk={Hk}", flush=True)
    compare(*inputs(2, H, Hk, 190, 64, seed=H), cap=30.0)
    compare(*inputs(1, H, Hk, 270, 128, seed=H), slopes=slopes_of(H), seg=documents(1, 270, 50))


@pytest.mark.parametrize("options", [dict(slopes=True, seg=700), dict(cap=30.0, prefix=True), dict(cap=50.0, slopes=True)],
                         ids=lambda o: "-".join(o))
def test_long(options):
    print(f"scored attention long {options}", flush=True)
    compare(*inputs(1, 2, 1, 4133, 64, seed=8), **resolve(options, 1, 2, 4133))
    o = resolve(options, 1, 1, 5000)
    if "prefix" in o:
        o["prefix"] = torch.tensor([3001], device=DEV)
    compare(*inputs(1, 1, 1, 5000, 128, seed=9), **o)


@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("D", [64, 128])
def test_many_workgroups(options, D):
    """Enough of them that each owns 128 rows (with fewer, as in the other tests, 64)."""

    print(f"scored attention, many workgroups {options} D={D}", flush=True)
    B, H, S = 33, 16, 290
    o = dict(options)
    if "prefix" in o:
        o["prefix"] = torch.arange(-3, 10 * B - 3, 10, dtype=torch.int32, device=DEV)
    if "seg" in o:
        o["seg"] = documents(B, S, o["seg"])
    if "slopes" in o:
        o["slopes"] = slopes_of(H)
    compare(*inputs(B, H, H if D == 64 else 8, S, D, seed=21), **o)


@pytest.mark.parametrize("D", [40, 64, 72, 128])
@pytest.mark.parametrize("B, H, Hk", [(8, 32, 8), (10, 24, 8), (2, 12, 3)])
def test_shared_heads_in_parts(B, H, Hk, D):
    """Groups of query heads whose key gradients come in several parts, of one head or of two."""

    S = 600 if B > 2 else 1100
    print(f"scored attention, shared heads in parts B={B} H={H}/{Hk} S={S} D={D}", flush=True)
    compare(*inputs(B, H, Hk, S, D, seed=23), cap=25.0, seg=documents(B, S, 300), slopes=slopes_of(H))


def test_large_scores_and_extreme_caps():
    q, k, v, do = inputs(1, 2, 2, 180, 64, seed=4, size=6.0)
    for cap, scale in ((2.0, None), (0.01, None), (1000.0, None), (40.0, 3.0), (None, 1.0), (None, 0.001)):
        print(f"cap={cap} scale={scale}", flush=True)
        compare(q, k, v, do, cap=cap, scale=scale)


def test_slopes_of_any_sign():
    q, k, v, do = inputs(1, 4, 2, 260, 64, seed=6)
    for slopes in ([0.0, -0.05, 3.0, 1e-4], [-1.0, 100.0, 0.0, -0.3]):
        compare(q, k, v, do, slopes=torch.tensor(slopes, device=DEV))
        compare(q, k, v, do, slopes=torch.tensor(slopes, device=DEV), cap=10.0, prefix=torch.tensor([111], device=DEV))


def test_strides():
    """Slices of one projection, the [batch, seq, heads] order, keys expanded over heads, a broadcast gradient."""

    B, H, S, D = 2, 3, 150, 64
    g = torch.Generator().manual_seed(1)
    packed = torch.randn((B, S, 3, H, D), generator=g).to(BF16).to(DEV)
    do = torch.randn((B, S, H, D), generator=g).to(BF16).to(DEV).transpose(1, 2)
    views = [packed[:, :, i].transpose(1, 2) for i in range(3)]
    want = run(*(t.contiguous() for t in views), do.contiguous(), cap=20.0)
    for vs in (views, [t.transpose(1, 2).contiguous().transpose(1, 2) for t in views]):
        got = run(*vs, do, cap=20.0)
        assert all(torch.equal(got[n], want[n]) for n in want)
    one = torch.randn((B, 1, S, D), generator=g).to(BF16).to(DEV)
    expanded = run(views[0], one.expand(B, H, S, D), one.expand(B, H, S, D), do)
    assert torch.equal(expanded["o"], run(views[0], one, one, do)["o"])
    odd = torch.randn(B * H * S * D + 1, generator=g).to(BF16).to(DEV)[1:].view(B, H, S, D)
    assert torch.equal(run(odd, odd, odd, do)["o"], run(*[odd.clone()] * 3, do)["o"])
    leaf = views[0].contiguous().requires_grad_()
    attend()(leaf, views[1], views[2]).sum().backward()
    ones = run(views[0], views[1], views[2], torch.ones((B, H, S, D), dtype=BF16, device=DEV))
    assert torch.equal(leaf.grad, ones["dq"])


def test_hidden_infinities_add_nothing():
    """A padded tail of garbage, and a document of it between others: the other
    rows and their gradients are bit for bit those of clean values."""

    for D in (64, 128):
        for Hk in (4, 2):
            q, k, v, do = inputs(2, 4, Hk, 300, D, seed=11)
            seg = torch.zeros((2, 300), dtype=torch.int32, device=DEV)
            seg[:, 90:150], seg[:, 150:] = 1, 2
            cases = [(dict(cap=20.0), slice(171, None)), (dict(slopes=slopes_of(4)), slice(257, None)),
                     (dict(seg=seg), slice(90, 150)), (dict(seg=seg, cap=9.0, slopes=slopes_of(4)), slice(90, 150)),
                     (dict(prefix=torch.tensor([60, 171], device=DEV)), slice(171, None)),
                     (dict(prefix=torch.tensor([90, 20], device=DEV), seg=seg), slice(90, 150))]
            for options, where in cases:
                clean = run(q, k, v, do, **options)
                keep = torch.ones(300, dtype=torch.bool, device=DEV)
                keep[where] = False
                for bad in (float("nan"), float("inf"), float("-inf")):
                    print(f"hidden {bad} D={D} Hk={Hk} {list(options)} {where}", flush=True)
                    dirty = [t.clone() for t in (q, k, v, do)]
                    for t in dirty:
                        t[:, :, where] = bad
                    got = run(*dirty, **options)
                    # (Without documents the tail's queries see every key before them, so what they
                    # spoil in dk and dv is theirs by the formula.)
                    for n in clean if "seg" in options else ("o", "dq"):
                        same = torch.equal(got[n][:, :, keep], clean[n][:, :, keep])
                        assert same, (n, bad, options.keys())


def test_visible_infinities_show():
    q, k, v, do = inputs(1, 2, 1, 200, 64, seed=12)
    v[0, 0, 70, 5], v[0, 0, 75, 6], v[0, 0, 75, 9] = float("inf"), float("-inf"), float("nan")
    v[0, 0, 130, 5] = float("-inf")
    o = run(q, k, v, do)["o"]
    clean = run(q, k, torch.nan_to_num(v, 0.0, 0.0, 0.0), do)["o"]
    col = lambda j: o[0, :, :, j]  # noqa: E731
    assert torch.isfinite(o[:, :, :70]).all() and torch.equal(o[:, :, :70], clean[:, :, :70])
    assert (col(5)[:, 70:130] == float("inf")).all() and col(5)[:, 130:].isnan().all()
    assert torch.isfinite(col(6)[:, :75]).all() and (col(6)[:, 75:] == float("-inf")).all() and col(9)[:, 75:].isnan().all()
    rest = [j for j in range(64) if j not in (5, 6, 9)]
    assert torch.equal(o[..., rest], clean[..., rest])
    q, k, v, do = inputs(1, 1, 1, 200, 64, seed=13)
    k[0, 0, 40, 3] = float("nan")
    got = run(q, k, v, do)
    assert got["o"][:, :, 40:].isnan().all() and torch.isfinite(got["o"][:, :, :40]).all()
    assert got["dq"][:, :, 40:].isnan().all() and torch.isfinite(got["dq"][:, :, :40]).all()


def test_plain_scores_agree_with_the_causal_attention():
    from gptrig.kernels import make_causal_attention

    q, k, v, do = inputs(2, 4, 4, 333, 64, seed=14)
    seg = documents(2, 333, 60)
    want = reference(q, k, v, do, seg=seg)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = make_causal_attention()(*leaves, seg)
    got = run(q, k, v, do, seg=seg)
    for name, other in zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))):
        assert bool(((got[name].to(F64) - other.to(F64)).abs() <= 2 * want[name][1]).all()), name


def test_gradients_against_differences():
    """Of the formula in 64 bits: the quotient is off by step^2 times a third
    derivative (of order 1 here), the kernel by its worst case."""

    B, H, Hk, S, D = 1, 4, 2, 70, 64
    q, k, v, do = inputs(B, H, Hk, S, D, seed=15)
    options = resolve(dict(cap=8.0, slopes=True, prefix=True, seg=40), B, H, S)
    got, want = run(q, k, v, do, **options), reference(q, k, v, do, **options)
    g = torch.Generator(device=DEV).manual_seed(2)

    def loss(*qkv):
        qq, kk, vv = qkv[0], *(t.repeat_interleave(H // Hk, dim=1) for t in qkv[1:])
        s = 8.0 * torch.tanh(torch.matmul(qq, kk.transpose(-1, -2)) * D ** -0.5 / 8.0)
        at = torch.arange(S, device=DEV, dtype=F64)
        s = s - options["slopes"].to(F64)[:, None, None] * (at[:, None] - at[None, :]).abs()
        s = s.masked_fill(~visible(B, S, options["seg"], options["prefix"]), -math.inf)
        return float((torch.matmul(torch.softmax(s, -1), vv) * do.to(F64)).sum())

    base = [t.to(F64) for t in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(base[i].shape, generator=g, device=DEV, dtype=F64)
        step = 1e-5
        ends = [loss(*(t + sign * step * way if j == i else t for j, t in enumerate(base))) for sign in (1, -1)]
        quotient = (ends[0] - ends[1]) / (2 * step)
        limit = float((want[name][1] * way.abs()).sum()) * 0.1 + 1e-5  # (the roundings' signs are not all the same)
        assert abs(quotient - float((got[name].to(F64) * way).sum())) <= limit, name


def test_repeats_other_streams_and_captured_graph():
    q, k, v, do = inputs(2, 6, 2, 400, 64, seed=16)
    options = resolve(dict(cap=30.0, slopes=True, seg=100, prefix=True), 2, 6, 400)
    want = run(q, k, v, do, **options)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, do, **options)
    assert all(torch.equal(got[n], want[n]) for n in want)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    attention = attend(30.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = attention(*leaves, options["seg"], prefix_lengths=options["prefix"], distance_slopes=options["slopes"])
        out = dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do))))
    for shift in range(3):
        moved = [torch.roll(t, shift, 2) for t in (q, k, v)]
        with torch.no_grad():
            for leaf, t in zip(leaves, moved):
                leaf.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        again = run(*moved, do, **options)
        assert all(torch.equal(out[n].detach(), again[n]) for n in again), shift


def test_partial_gradients_and_no_grad():
    q, k, v, do = inputs(1, 2, 2, 130, 64, seed=17)
    want = run(q, k, v, do, cap=20.0)
    for i, name in enumerate(("dq", "dk", "dv")):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        assert torch.equal(torch.autograd.grad(attend(20.0)(*leaves), leaves[i], do)[0], want[name])
    with torch.no_grad():
        assert torch.equal(attend(20.0)(q, k, v), want["o"])
    assert torch.equal(attend(20.0)(q, k, v, torch.zeros((1, 130), dtype=torch.int64, device=DEV)), want["o"])


@pytest.mark.parametrize("options", [dict(prefix=True), dict(seg=90, cap=20.0), dict(prefix=True, seg=150, slopes=True)],
                         ids=lambda o: "-".join(o))
def test_the_order_of_blocks_changes_nothing(options, monkeypatch):
    from gptrig.kernels import scored_attention as module

    print(f"scored attention, planned order {options}", flush=True)
    B, H, S = 5, 12, 1000
    o = resolve(options, B, H, S)
    if "seg" in o:
        o["seg"][1] = torch.randint(0, 4, (S,), device=DEV)  # (ids in no order)
    tensors = inputs(B, H, 4, S, 64, seed=31)
    assert module._sizes("gptrig_scored_attn_plan_bytes", B, H, 4, S, 64) > 0
    got = compare(*tensors, **o)
    leaves = [t.detach().clone().requires_grad_() for t in tensors[:3]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(o.get("cap"))(*leaves, o.get("seg"), prefix_lengths=o.get("prefix"),
                                   distance_slopes=o.get("slopes"))
        again = dict(zip(("o", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, tensors[3]))))
    for shift in range(3):
        if "prefix" in o:
            o["prefix"].copy_(torch.roll(o["prefix"], shift))
        if "seg" in o:
            o["seg"].copy_(torch.roll(o["seg"], shift, 0))
        graph.replay()
        torch.cuda.synchronize()
        with monkeypatch.context() as m:
            m.setattr(module, "_sizes", lambda name, *sizes: 0 if "plan" in name else module._lib.query(name, *sizes))
            plain = run(*tensors, **o)
        assert all(torch.equal(again[n].detach(), plain[n]) for n in plain), shift
        if not shift:
            assert all(torch.equal(got[n], plain[n]) for n in plain)
