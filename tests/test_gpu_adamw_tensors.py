"""``gptrig.optim.adamw_tensors`` against the formula in 64 bits.

Tolerances: the float32 update is a chain of fewer than 16 roundings of 2^-24
each (the moments of 4), so a parameter is off by at most half a step of its own
plus ``lr_t 16 2^-24 (|step| + |decay p|)``.  An 8-bit code is the exact one
wherever ``y / step + u`` is further from a whole number than its float32 error
(y / step < 16, 12 roundings: below 2^-16), elsewhere at most one code away.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64, F8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
U = 2.0 ** -24
LR, B1, B2 = 0.01, 0.9, 0.95


def bits_of(seed, tensor, n):
    """The 32 random bits of a tensor's n values, from the definition of the hash."""

    low = np.uint64(0xFFFFFFFF)

    def mix(x):
        x = np.asarray(x, np.uint64) & low
        x ^= x >> np.uint64(16)
        x = x * np.uint64(0x6A09E667) & low
        x ^= x >> np.uint64(15)
        x = x * np.uint64(0xBB67AE85) & low
        return x ^ (x >> np.uint64(16))

    phi = np.uint64(0x9E3779B9)
    key = mix(mix(seed) + np.uint64(tensor) * phi)
    return mix(np.arange(n, dtype=np.uint64) * phi + key)


def codes_of(x, u, floor):
    """Exact codes (before the rounding's float32 error), scales, the size of each code's step and its distance
    from a tie."""

    n = x.size
    blocks = -(-n // 256)
    size = np.abs(np.concatenate([x, np.zeros(blocks * 256 - n)])).reshape(blocks, 256)
    finite = np.where(np.isfinite(size), size, 0)
    top = finite.max(1, keepdims=True)
    scale = np.where(top < 2.0 ** -100, 0, top / 448)
    y = np.where(scale > 0, np.minimum(size / np.where(scale > 0, scale, 1), 448), 0).reshape(-1)[:n]
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(y, 1e-300))), -6) - 3)
    at = y / step + u
    code = np.floor(at) * step
    near = np.abs(at - np.round(at))
    if floor:
        code = np.where((np.abs(x) > 0) & (scale.repeat(256, 1).reshape(-1)[:n] > 0), np.maximum(code, 2.0 ** -9), code)
    return np.copysign(code, x), scale.reshape(-1), step, near


def values(code, scale):
    n = code.numel()
    return (code.to(F64).reshape(-1) * scale.to(F64).repeat_interleave(256)[:n]).cpu().numpy()


class Lists:
    def __init__(self, shapes, bits, grads=F32, shadow=False, seed=0, unaligned=False, started=True):
        g = torch.Generator().manual_seed(seed)

        def put(t):
            t = t.to(DEV)
            if not unaligned:
                return t
            room = torch.empty(t.numel() + 3, dtype=torch.uint8 if t.dtype == F8 else t.dtype, device=DEV)
            room = room.view(t.dtype) if t.dtype == F8 else room
            return room[3:].view(t.shape).copy_(t)

        def normal(shape, scale):
            return torch.randn(shape, generator=g) * scale

        self.bits = bits
        self.p = [put(normal(s, 1.0)) for s in shapes]
        self.g = [put(normal(s, 0.1).to(grads)) for s in shapes]
        if bits == 32:
            self.m = [put(normal(s, 0.1 * started)) for s in shapes]
            self.v = [put(normal(s, 0.1 * started).square()) for s in shapes]
            self.ms = self.vs = None
        else:
            self.m = [put((normal(s, 60.0 * started).clamp(-448, 448)).to(F8)) for s in shapes]
            self.v = [put((normal(s, 60.0 * started).abs().clamp(0, 448)).to(F8)) for s in shapes]
            blocks = [-(-math.prod(s) // 256) for s in shapes]
            self.ms = [put((torch.rand(b, generator=g) + 0.5) * 1e-3 * started) for b in blocks]
            self.vs = [put((torch.rand(b, generator=g) + 0.5) * 1e-4 * started) for b in blocks]
        self.shadow = [put(torch.zeros(s, dtype=BF16)) for s in shapes] if shadow else None
        rows = [(1.0 + 0.5 * (i % 3), 1e-8 * (1 + i % 2), 0.1 * (i % 2)) for i in range(len(shapes))]
        self.hp = torch.tensor(rows, dtype=F32, device=DEV).reshape(len(shapes), 3)

    def step(self, step=3, clip=None, seed=None, lr=LR, b1=B1, b2=B2):
        from gptrig.optim import adamw_tensors

        adamw_tensors(self.p, self.g, self.m, self.v, self.hp, lr=lr, beta1=b1, beta2=b2, step=step,
                      exp_avg_scale=self.ms, exp_avg_sq_scale=self.vs, clip_scale=clip, shadow=self.shadow, seed=seed)

    def moments(self, i):
        if self.bits == 32:
            return (t[i].to(F64).reshape(-1).cpu().numpy() for t in (self.m, self.v))
        return values(self.m[i], self.ms[i]), values(self.v[i], self.vs[i])

    def everything(self):
        flat = [*self.p, *self.m, *self.v, *(self.ms or []), *(self.vs or []), *(self.shadow or [])]
        return [t.to(F64).reshape(-1) if t.dtype == F8 else t.reshape(-1) for t in flat]


def expected(L, clip, step):
    """The new parameters and moments in 64 bits, from the present lists."""

    out = []
    for i, p in enumerate(L.p):
        m, v = L.moments(i)
        g = L.g[i].to(F64).reshape(-1).cpu().numpy() * (1.0 if clip is None else float(clip))
        p = p.to(F64).reshape(-1).cpu().numpy()
        lr_mult, eps, decay = (float(x) for x in L.hp[i].cpu())
        m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
        way = m / (1 - B1 ** step) / (np.sqrt(v / (1 - B2 ** step)) + eps)
        lr = LR * lr_mult
        size_m = np.abs(m) + (1 - B1) * np.abs(g)
        bound = U * np.abs(p) + 16 * U * lr * (np.abs(way) + np.abs(decay * p)) + 16 * U * lr * size_m / (
            1 - B1 ** step) / (np.sqrt(v / (1 - B2 ** step)) + eps)
        new = p - lr * (way + decay * p)
        out.append((new, bound + U * np.abs(new), m, 4 * U * size_m, v, 4 * U * v))
    return out


def verify(L, want, seed):
    for i, (p, pb, m, mb, v, vb) in enumerate(want):
        got = L.p[i].to(F64).reshape(-1).cpu().numpy()
        assert (np.abs(got - p) <= pb).all(), (i, np.max(np.abs(got - p) - pb))
        if L.shadow is not None:
            assert torch.equal(L.shadow[i], L.p[i].to(BF16)), i
        if L.bits == 32:
            for kept, x, b in ((L.m, m, mb), (L.v, v, vb)):
                assert (np.abs(kept[i].to(F64).reshape(-1).cpu().numpy() - x) <= b + 1e-45).all(), i
            continue
        bits = bits_of(seed, i, p.size)
        for kept, scales, x, shift, floor in ((L.m, L.ms, m, 0, False), (L.v, L.vs, v, 16, True)):
            u = ((bits >> np.uint64(shift) & np.uint64(0xFFFF)).astype(np.float64) + 0.5) / 65536
            code, scale, step, near = codes_of(x, u, floor)
            got_scale = scales[i].to(F64).cpu().numpy()
            assert (np.abs(got_scale - scale) <= 8 * U * scale).all(), i
            got = kept[i].to(F64).reshape(-1).cpu().numpy()
            off = np.abs(got - code)
            # (m is a difference where its terms cancel: its own bound counts towards the tie.)
            tie = near <= 2.0 ** -16 + 16 * np.where(np.abs(x) > 0, (mb if shift == 0 else vb) / np.maximum(np.abs(x), 1e-300), 0)
            assert (off[~tie] == 0).all(), (i, int((off[~tie] > 0).sum()))
            assert (off[tie] <= 2 * step[tie]).all(), i


SHAPES = [(1,), (3,), (255,), (256,), (257,), (0,), (1000,), (31, 33), (4095,), (4096,), (4097,), (300, 301), (2, 3, 5)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grads,shadow,clip,unaligned",
                         [(F32, False, None, False), (BF16, True, 0.37, False), (F32, True, 2.0, True), (BF16, False, None, True)])
def test_matches_the_formula(bits, grads, shadow, clip, unaligned):
    print(f"adamw_tensors bits={bits} grads={grads} shadow={shadow} clip={clip} unaligned={unaligned}", flush=True)
    L = Lists(SHAPES, bits, grads, shadow, unaligned=unaligned)
    factor = None if clip is None else torch.tensor(clip, device=DEV)
    before = [t.clone() for t in L.g]
    want = expected(L, factor, 3)
    L.step(3, factor, seed=1234567)
    verify(L, want, 1234567)
    assert all(torch.equal(a, b) for a, b in zip(before, L.g))


@pytest.mark.parametrize("bits", [32, 8])
def test_from_zero_moments_and_several_steps(bits):
    from gptrig.optim import adamw_tensors_state

    L = Lists([(700,), (64, 65)], bits, started=False)
    state = adamw_tensors_state(L.p, bits)
    L.m, L.v = state["exp_avg"], state["exp_avg_sq"]
    L.ms, L.vs = state.get("exp_avg_scale"), state.get("exp_avg_sq_scale")
    for step in range(1, 5):
        want = expected(L, None, step)
        L.step(step)  # the seed is the step
        verify(L, want, step)


def test_more_tensors_than_a_launch_takes():
    L = Lists([(5 + i,) if i % 7 else (0,) for i in range(111)] + [(70000,)], 8, BF16, True)
    want = expected(L, None, 9)
    L.step(9, seed=2 ** 32 - 1)
    verify(L, want, 2 ** 32 - 1)


def test_codes_are_right_on_average():
    """The mean over N seeds of what a moment is kept as, against the moment: the
    roundings are independent with a deviation of at most half a step, so six
    deviations of the mean are 3 steps / sqrt(N)."""

    n, seeds = 512, 400
    L = Lists([(n,)], 8)
    L.v[0].copy_(torch.rand(n, device=DEV) * 400 + 1)
    keep = [t.clone() for t in (L.m[0].view(torch.uint8), L.v[0].view(torch.uint8), L.ms[0], L.vs[0], L.p[0])]
    _, _, m, _, v, _ = expected(L, None, 3)[0]
    mean = np.zeros((2, n))
    for seed in range(seeds):
        for t, k in zip((L.m[0].view(torch.uint8), L.v[0].view(torch.uint8), L.ms[0], L.vs[0], L.p[0]), keep):
            t.copy_(k)
        L.step(3, seed=seed)
        mean += np.stack([values(L.m[0], L.ms[0]), values(L.v[0], L.vs[0])]) / seeds
    for got, x, scales in ((mean[0], m, L.ms[0]), (mean[1], v, L.vs[0])):
        s = scales.to(F64).cpu().numpy().repeat(256)
        _, _, step, _ = codes_of(x, 0.0, False)
        assert (np.abs(got - x) <= 3 * step * s / math.sqrt(seeds) + 1e-6 * np.abs(x)).all()


def test_empty_tiny_and_infinite_blocks():
    L = Lists([(1024,)], 8, started=False)
    L.g[0][:256] = 0                      # nothing
    L.g[0][256:512] = 1e-18               # v below 2^-100, m above
    L.g[0][600], L.g[0][601] = float("inf"), float("nan")
    p = L.p[0].clone()
    L.step(1, seed=5)
    m, v = (t[0].to(F32) for t in (L.m, L.v))
    assert not m[:256].any() and not v[:256].any() and not L.ms[0][0] and not L.vs[0][0]
    assert m[256:512].all() and not L.vs[0][1]
    assert torch.isfinite(L.ms[0]).all() and torch.isfinite(L.vs[0]).all()
    bad = torch.zeros(1024, dtype=torch.bool, device=DEV)
    bad[600:602] = True
    assert m[bad].isnan().all() and v[bad].isnan().all()
    for t in (L.p[0], m, v):
        assert torch.isfinite(t[~bad]).all()
    assert L.p[0][bad].isnan().all()
    assert torch.equal(L.p[0][:256], p[:256])  # (the first tensor does not decay)
    # A v of zero beside a momentum is never what a step leaves.
    assert ((v > 0) | (m == 0) | bad)[512:].all()


def test_the_same_call_gives_the_same_and_the_seed_matters():
    runs = []
    for seed in (7, 7, 8):
        L = Lists([(5000,), (333, 3)], 8, shadow=True, seed=2)
        L.step(4, seed=seed)
        runs.append(L.everything())
    assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1]))
    assert not all(torch.equal(a, b) for a, b in zip(runs[0], runs[2]))
    assert torch.equal(runs[0][0], runs[2][0])  # the step itself does not see the rounding


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed_on_another_stream(bits):
    L, M = (Lists([(5000,), (77, 13)], bits, BF16, True, seed=3) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        L.step(2, seed=11)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        M.step(2, seed=11)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(L.everything(), M.everything())), k
        for a, b in zip(L.g, M.g):
            a.mul_(0.5), b.mul_(0.5)


def test_backward_through_a_changed_parameter_is_refused():
    L = Lists([(64,)], 32)
    w = L.p[0].requires_grad_()
    loss = (w * w).sum()
    L.p = [w.detach()]
    L.step(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_the_same_tensor_twice_is_refused():
    L = Lists([(300,), (300,)], 32)
    before = L.p[0].clone()
    L.p[1] = L.p[0]
    with pytest.raises(ValueError, match="overlap"):
        L.step(1)
    M = Lists([(300,), (300,)], 8)
    M.vs[1] = M.ms[1]
    with pytest.raises(ValueError, match="overlap"):
        M.step(1)
    torch.cuda.synchronize()
    assert torch.equal(L.p[0], before)
    N = Lists([(300,), (300,)], 32)
    N.g[1] = N.p[0]
    with pytest.raises(ValueError, match="overlap"):
        N.step(1)


def test_a_shared_gradient_and_a_saved_shadow():
    L, M = Lists([(300,), (300,)], 32, shadow=True), Lists([(300,), (300,)], 32, shadow=True)
    L.g[1], M.g[1] = L.g[0], M.g[0].clone()
    w = torch.ones(300, dtype=BF16, device=DEV, requires_grad=True)
    loss = (w * L.shadow[0]).sum()
    L.step(1), M.step(1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(L.p + L.shadow, M.p + M.shadow))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
