"""LayerNorm, attention with capped or biased scores, and AdamW over lists of
tensors, as cases that can be timed and compared.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes what a training program holds before the call, ``run`` is one
pass: in elementary float32 torch operations, or, with ``own``, through
gptrig's entry points.  ``work`` is what the pass cannot do without, ``exact``
the same outputs in 64 bits.

Imported with the repository's root as the working folder.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
BF16, F32, F64, F8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
TYPES = {"bf16": BF16, "f32": F32}
VOCAB = 50304  # storage rows of the embedding, as in the benchmark's model
QUANT = 256  # values that share a scale of the 8-bit states
ALIGN = 64  # every tensor of a list starts on such an element of its buffer


def listed() -> list[dict]:
    return [
        # The norm of one prompt, forward only: the smallest call, where its launch counts.
        norm("norm-prompt", rows=129, width=768, backward=False),
        # One block's norm in training, at the tokens of a micro-batch of the 125M model.
        norm("norm-train", rows=65536, width=768),
        # Float32 activations of a width that is no multiple of a vector, without a bias.
        norm("norm-float32-odd", rows=8191, width=1001, dtype="f32", bias=False),
        # Evaluating one short sequence with capped scores.
        attention("attention-prompt", batch=1, heads=12, seq=129, dim=64, cap=30.0, backward=False),
        # The attention layer of the 125M model with capped scores, in training.
        attention("attention-capped", batch=16, heads=12, seq=1024, dim=64, cap=30.0),
        # Prefix language modelling with a distance bias, over a window that is no multiple of any tile.
        attention("attention-prefix-bias", batch=4, heads=12, seq=2000, dim=64, slopes=True, prefix=True),
        # Heads of 128 that share keys and values in groups of four, capped and biased.
        attention("attention-grouped-wide", batch=4, heads=16, kv_heads=4, seq=2048, dim=128, cap=50.0, slopes=True),
        # Long-context training on packed documents with a distance bias, q, k and v as slices of one projection.
        attention("attention-documents-8k", batch=1, heads=12, seq=8192, dim=64, slopes=True, documents=1500,
                  packed=True),
        # The update of a small model's tensors, where the launch and the host count.
        adamw("adamw-small", width=256, layers=2, vocab=1000, bits=32),
        # The update of a model of 230M parameters, float32 states.
        adamw("adamw-32", width=960, layers=12, vocab=VOCAB, bits=32),
        # The same with 8-bit states.
        adamw("adamw-8", width=960, layers=12, vocab=VOCAB, bits=8),
        # Odd sizes, bf16 gradients, a bf16 copy of the parameters and a clip factor, 8-bit states.
        adamw("adamw-8-odd", width=509, layers=6, vocab=20011, bits=8, grads="bf16", shadow=True, clip=True),
    ]


def norm(name, rows, width, dtype="bf16", bias=True, params="f32", backward=True) -> dict:
    return dict(name=name, op="norm", rows=rows, width=width, dtype=dtype, bias=bias, params=params, backward=backward)


def attention(name, batch, heads, seq, dim, kv_heads=0, cap=0.0, slopes=False, prefix=False, documents=0,
              packed=False, backward=True) -> dict:
    """cap 0: none; kv_heads 0: as many as heads; documents: their mean length, 0 for one."""

    return dict(name=name, op="attention", batch=batch, heads=heads, kv_heads=kv_heads or heads, seq=seq, dim=dim,
                cap=cap, slopes=slopes, prefix=prefix, documents=documents, packed=packed, backward=backward)


def adamw(name, width, layers, vocab, bits, grads="f32", shadow=False, clip=False) -> dict:
    return dict(name=name, op="adamw", width=width, layers=layers, vocab=vocab, bits=bits, grads=grads, shadow=shadow,
                clip=clip)


def spread(rng, low, high) -> int:
    """A whole number between low and high, even over their logarithm."""

    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    op = rng.choice(("norm", "attention", "attention", "adamw"))
    if op == "norm":
        width = rng.choice((256, 512, 768, 1024, 1536, spread(rng, 64, 8192)))
        rows = spread(rng, 1, 2 ** 25 // width)
        case = norm("", rows, width, rng.choice(("bf16", "bf16", "f32")), rng.random() < 0.7,
                    rng.choice(("f32", "bf16")), rng.random() < 0.7)
    elif op == "attention":
        groups = rng.choice((1, 1, 2, 4))
        kv_heads = rng.choice((1, 2, 3, 4, 6))
        seq = spread(rng, 1, 8192)
        batch = spread(rng, 1, max(1, min(16, 2 ** 29 // (kv_heads * groups * seq * seq))))
        case = attention("", batch, kv_heads * groups, seq, rng.choice((64, 64, 128, 128, 8 * rng.randint(4, 16))),
                         kv_heads, rng.choice((0.0, 15.0, 30.0, 50.0)), rng.random() < 0.5, rng.random() < 0.4,
                         rng.choice((0, 0, spread(rng, 16, 3000))), groups == 1 and rng.random() < 0.5,
                         rng.random() < 0.7)
    else:
        width = spread(rng, 64, 1024)
        case = adamw("", width, rng.randint(1, 12), spread(rng, 500, VOCAB), rng.choice((8, 8, 32)),
                     rng.choice(("f32", "f32", "bf16")), rng.random() < 0.5, rng.random() < 0.5)
    del case["name"]
    return case


# -- what a program has in hand ---------------------------------------------------


def generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def prepare(case, seed):
    return {"norm": prepare_norm, "attention": prepare_attention, "adamw": prepare_adamw}[case["op"]](case, seed)


def prepare_norm(case, seed):
    g = generator(seed)
    rows, d, dtype, params = case["rows"], case["width"], TYPES[case["dtype"]], TYPES[case["params"]]
    # Activations of a residual stream: a mean and a spread of their own for each row.
    x = torch.randn((rows, d), generator=g, device=DEVICE) * (0.5 + torch.rand((rows, 1), generator=g, device=DEVICE))
    x += torch.randn((rows, 1), generator=g, device=DEVICE)
    scale = 1 + 0.2 * torch.randn(d, generator=g, device=DEVICE)
    bias = 0.2 * torch.randn(d, generator=g, device=DEVICE) if case["bias"] else None
    dy = torch.randn((rows, d), generator=g, device=DEVICE) if case["backward"] else None
    back = case["backward"]
    return dict(case=case, x=x.to(dtype).requires_grad_(back), scale=scale.to(params).requires_grad_(back),
                bias=None if bias is None else bias.to(params).requires_grad_(back),
                dy=None if dy is None else dy.to(dtype))


def prepare_attention(case, seed):
    g = generator(seed)
    B, H, Hk, S, D = (case[k] for k in ("batch", "heads", "kv_heads", "seq", "dim"))
    if case["packed"]:  # [batch, seq, 3, heads, dim], as one projection leaves it
        qkv = torch.randn((B, S, 3, H, D), generator=g, device=DEVICE).to(BF16)
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    else:
        q = torch.randn((B, H, S, D), generator=g, device=DEVICE).to(BF16)
        k = torch.randn((B, Hk, S, D), generator=g, device=DEVICE).to(BF16)
        v = torch.randn((B, Hk, S, D), generator=g, device=DEVICE).to(BF16)
    back = case["backward"]
    state = dict(case=case, do=None, segments=None, prefix=None, slopes=None)
    state.update(zip("qkv", (t.detach().requires_grad_(back) for t in (q, k, v))))
    if back:
        state["do"] = torch.randn((B, H, S, D), generator=g, device=DEVICE).to(BF16)
    if case["documents"]:
        cuts = torch.rand((B, S), generator=g, device=DEVICE) < 1.0 / case["documents"]
        state["segments"] = torch.cumsum(cuts.to(torch.int32), dim=1).to(torch.int32)
    if case["prefix"]:
        state["prefix"] = torch.randint(0, S + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32)
    if case["slopes"]:
        state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEVICE, dtype=F32) / H)
    return state


def shapes(case) -> list[tuple[int, ...]]:
    d, vocab = case["width"], case["vocab"]
    block = [(d,), (d, 3 * d), (3 * d,), (d, d), (d,), (d,), (d, 4 * d), (4 * d,), (4 * d, d), (d,)]
    return [(vocab, d)] + block * case["layers"] + [(d,), (vocab, d)]


def views(flat, all_shapes, unit=1):
    """The tensors of a list inside one buffer, of ``unit`` values each an element (1) or a scale (QUANT)."""

    if unit == 1:
        sizes = [math.prod(s) for s in all_shapes]
        starts = np.cumsum([0] + [-(-n // ALIGN) * ALIGN for n in sizes])
        return [flat[a:a + n].view(s) for a, n, s in zip(starts.tolist(), sizes, all_shapes)]
    sizes = [-(-math.prod(s) // unit) for s in all_shapes]
    starts = np.cumsum([0] + sizes)
    return [flat[a:a + n] for a, n in zip(starts.tolist(), sizes)]


def prepare_adamw(case, seed):
    g = generator(seed)
    every = shapes(case)
    total = sum(-(-math.prod(s) // ALIGN) * ALIGN for s in every)
    scales = sum(-(-math.prod(s) // QUANT) for s in every)

    def normal(scale):
        return torch.randn(total, generator=g, device=DEVICE).mul_(scale)

    flat = {"p": normal(0.02)}
    grad = normal(1e-3).to(TYPES[case["grads"]])
    if case["bits"] == 32:
        flat["m"] = normal(1e-3)
        flat["v"] = normal(1e-3).square_()
    else:
        flat["m"] = normal(60.0).clamp_(-448, 448).to(F8)
        flat["v"] = normal(60.0).abs_().clamp_(2.0 ** -9, 448).to(F8)
        flat["ms"] = torch.rand(scales, generator=g, device=DEVICE) * 1e-5 + 1e-6
        flat["vs"] = torch.rand(scales, generator=g, device=DEVICE) * 1e-8 + 1e-9
    if case["shadow"]:
        flat["shadow"] = flat["p"].to(BF16)
    lists = {k: views(t, every, QUANT if k in ("ms", "vs") else 1) for k, t in flat.items()}
    # Learning-rate multiplier, epsilon and decay of each tensor: vectors (norms, biases) do not decay.
    rows = [(1.0 if len(s) > 1 else 2.0, 1e-8, 0.1 if len(s) > 1 else 0.0) for s in every]
    return dict(case=case, flat=flat, lists=lists, grads=views(grad, every), hparams=torch.tensor(rows, device=DEVICE),
                clip=torch.full((1,), 0.7, device=DEVICE) if case["clip"] else None, seed=seed % 2 ** 31)


LR, BETA1, BETA2, STEP = 2.0 ** -8, 0.9, 0.95, 100


# -- one pass ----------------------------------------------------------------------


def run(state):
    return {"norm": run_norm, "attention": run_attention, "adamw": run_adamw}[state["case"]["op"]](state)


def package():
    path = os.path.join(os.getcwd(), "gpt-speedrun-tpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)


def run_norm(s):
    names = ("x", "scale", "bias") if s["bias"] is not None else ("x", "scale")
    if own:
        package()
        from gptrig.nn import layer_norm

        y = layer_norm(s["x"], s["scale"], s["bias"])
        if s["dy"] is None:
            return {"y": y}
        return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, [s[n] for n in names], s["dy"])))}
    x, w = s["x"].detach().to(F32), s["scale"].detach().to(F32)
    d = x.shape[1]
    centred = x - x.sum(1, keepdim=True) / d
    r = torch.rsqrt(centred.square().sum(1, keepdim=True) / d + 1e-5)
    h = centred * r
    y = h * w
    if s["bias"] is not None:
        y = y + s["bias"].detach().to(F32)
    out = {"y": y.to(s["x"].dtype)}
    if s["dy"] is None:
        return out
    dy = s["dy"].to(F32)
    g = dy * w
    out["x"] = (r * (g - g.sum(1, keepdim=True) / d - h * ((g * h).sum(1, keepdim=True) / d))).to(s["x"].dtype)
    out["scale"] = (dy * h).sum(0, dtype=F64).to(s["scale"].dtype)
    if s["bias"] is not None:
        out["bias"] = dy.sum(0, dtype=F64).to(s["bias"].dtype)
    return out


def run_attention(s):
    c = s["case"]
    if own:
        package()
        from gptrig.kernels import ScoredAttentionConfig, make_scored_attention

        o = make_scored_attention(ScoredAttentionConfig(score_cap=c["cap"] or None))(
            s["q"], s["k"], s["v"], s["segments"], prefix_lengths=s["prefix"], distance_slopes=s["slopes"])
        if s["do"] is None:
            return {"o": o}
        return {"o": o.detach(), **dict(zip("qkv", torch.autograd.grad(o, [s[n] for n in "qkv"], s["do"])))}
    B, H, Hk, S, D = (c[k] for k in ("batch", "heads", "kv_heads", "seq", "dim"))
    scale, cap = D ** -0.5, c["cap"]
    q = s["q"].detach().to(F32).reshape(B * H, S, D)
    k, v = (s[n].detach().to(F32).repeat_interleave(H // Hk, dim=1).reshape(B * H, S, D) for n in "kv")
    score = torch.bmm(q, k.transpose(1, 2).contiguous()) * scale
    slope = None
    if cap:
        t = torch.tanh(score / cap)
        score = cap * t
        slope = 1 - t * t
        del t
    score = score.view(B, H, S, S)
    at = torch.arange(S, device=DEVICE)
    if s["slopes"] is not None:
        score -= s["slopes"][:, None, None] * (at[:, None] - at[None, :]).abs().to(F32)
    hidden = (at[None, :] > at[:, None])[None]
    if s["prefix"] is not None:
        hidden = hidden & (at[None, None, :] >= s["prefix"][:, None, None])
    if s["segments"] is not None:
        hidden = hidden | (s["segments"][:, :, None] != s["segments"][:, None, :])
    score.masked_fill_(hidden[:, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = torch.exp(score)
    del score
    p /= p.sum(-1, keepdim=True)
    p = p.view(B * H, S, S)
    o = torch.bmm(p, v)
    out = {"o": o.view(B, H, S, D).to(BF16)}
    if s["do"] is None:
        return out
    do = s["do"].to(F32).view(B * H, S, D)
    dv = torch.bmm(p.transpose(1, 2), do)
    dp = torch.bmm(do, v.transpose(1, 2).contiguous())
    dp -= (do * o).sum(-1, keepdim=True)
    dp *= p
    del p
    if slope is not None:
        dp *= slope
    dp *= scale
    dk = torch.bmm(dp.transpose(1, 2), q)
    out["q"] = torch.bmm(dp, k).view(B, H, S, D).to(BF16)
    out["k"], out["v"] = (x.view(B, Hk, H // Hk, S, D).sum(2).to(BF16) for x in (dk, dv))
    return out


def random_bits(seed, tensor, n):
    """The 32 random bits of each of a tensor's n values, as int64: the hash
    that the 8-bit states' rounding is defined with."""

    def mix(x):
        x = x ^ (x >> 16)
        x = (x * 0x6A09E667) & 0xFFFFFFFF
        x = x ^ (x >> 15)
        x = (x * 0xBB67AE85) & 0xFFFFFFFF
        return x ^ (x >> 16)

    i = torch.arange(n, device=DEVICE)
    key = mix((mix(seed) + tensor * 0x9E3779B9) & 0xFFFFFFFF)
    return mix(((i & 0xFFFFFFFF) * 0x9E3779B9 + key + (i >> 32) * 0xBB67AE85) & 0xFFFFFFFF)


def quantized(x, u, floor):
    """The codes (values in e4m3) and scales of a tensor's values, in blocks of
    QUANT: each magnitude over its block's scale is rounded down after adding
    the random u of a step.  ``floor``: nothing above zero becomes zero."""

    n = x.numel()
    pad = -n % QUANT
    x = torch.nn.functional.pad(x.reshape(-1), (0, pad)).view(-1, QUANT)
    u = torch.nn.functional.pad(u, (0, pad)).view(-1, QUANT)
    size = x.abs()
    scale = size.amax(1, keepdim=True) * (1.0 / 448)
    y = (size / torch.where(scale > 0, scale, 1.0)).clamp(max=448.0)
    step = torch.exp2(torch.frexp(y)[1].clamp(min=-5) - 4.0)
    code = torch.floor(y / step + u) * step
    if floor:
        code = torch.where(size > 0, code.clamp(min=2.0 ** -9), code)
    code = torch.copysign(code, x).reshape(-1)[:n]
    return code, scale.reshape(-1)


def valued(code, scale, dtype):
    """What codes stand for."""

    return code.reshape(-1).to(dtype) * scale.to(dtype).repeat_interleave(QUANT)[:code.numel()]


def update(case, p, g, m, v, hparams, clip, dtype):
    """The new parameter, and moments before they are rounded."""

    lr_mult, eps, decay = hparams
    g = g.to(dtype) * clip if clip is not None else g.to(dtype)
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    step = (m / (1 - BETA1 ** STEP)) / (torch.sqrt(v / (1 - BETA2 ** STEP)) + eps)
    return p - (LR * lr_mult) * (step + decay * p), m, v


def bits_as_steps(bits):
    """The random shares of a step for the two moments, from their 32 bits."""

    return ((bits & 0xFFFF).to(F32) + 0.5) / 65536, ((bits >> 16).to(F32) + 0.5) / 65536


def update_tensor(s, i):
    L, case = s["lists"], s["case"]
    p, g, m, v = L["p"][i], s["grads"][i], L["m"][i], L["v"][i]
    hp = s["hparams"][i]
    if case["bits"] == 32:
        new, m1, v1 = update(case, p, g, m, v, hp, s["clip"], F32)
        m.copy_(m1), v.copy_(v1)
    else:
        m0, v0 = valued(m, L["ms"][i], F32).view(p.shape), valued(v, L["vs"][i], F32).view(p.shape)
        new, m1, v1 = update(case, p, g, m0, v0, hp, s["clip"], F32)
        um, uv = bits_as_steps(random_bits(s["seed"], i, p.numel()))
        for_m, for_v = quantized(m1, um, False), quantized(v1, uv, True)
        m.copy_(for_m[0].view(p.shape)), L["ms"][i].copy_(for_m[1])
        v.copy_(for_v[0].view(p.shape)), L["vs"][i].copy_(for_v[1])
    p.copy_(new)
    if case["shadow"]:
        L["shadow"][i].copy_(new)


def run_adamw(s):
    L = s["lists"]
    if own:
        package()
        from gptrig.optim import adamw_tensors

        adamw_tensors(L["p"], s["grads"], L["m"], L["v"], s["hparams"], lr=LR, beta1=BETA1, beta2=BETA2, step=STEP,
                      exp_avg_scale=L.get("ms"), exp_avg_sq_scale=L.get("vs"), clip_scale=s["clip"],
                      shadow=L.get("shadow"), seed=s["seed"])
    else:
        _ = [update_tensor(s, i) for i in range(len(L["p"]))]
    return dict(s["flat"])


# -- what it cannot do without --------------------------------------------------------


def visible_pairs(case) -> float:
    """Visible (query, key) pairs of the whole batch, for documents and prefixes of one fixed draw."""

    B, S = case["batch"], case["seq"]
    r = np.random.RandomState(7)
    total = 0.0
    for _ in range(B):
        cuts = np.flatnonzero(r.rand(S) < 1.0 / case["documents"]) if case["documents"] else np.empty(0, np.int64)
        edges = np.unique(np.concatenate([[0], cuts, [S]]))
        n = np.diff(edges).astype(np.float64)
        total += float((n * (n + 1) / 2).sum())
        if case["prefix"]:
            inside = np.clip(r.randint(0, S + 1) - edges[:-1], 0, n)
            total += float((inside * (inside - 1) / 2).clip(min=0).sum())
    return total


def work(case) -> dict:
    if case["op"] == "norm":
        n, size, psize = case["rows"] * case["width"], TYPES[case["dtype"]].itemsize, TYPES[case["params"]].itemsize
        vectors = (2 if case["bias"] else 1) * case["width"] * psize
        return {"bytes": n * size * (4 if case["backward"] else 2) + vectors * (2 if case["backward"] else 1),
                "flops": n * (18 if case["backward"] else 7)}
    if case["op"] == "attention":
        B, H, Hk, S, D = (case[k] for k in ("batch", "heads", "kv_heads", "seq", "dim"))
        q, kv = 2 * B * H * S * D, 2 * B * Hk * S * D
        ids = (4 * B * S if case["documents"] else 0) + (4 * B if case["prefix"] else 0) + (4 * H if case["slopes"] else 0)
        return {"bytes": (4 * q + 4 * kv if case["backward"] else 2 * q + 2 * kv) + ids,
                "flops": visible_pairs(case) * H * D * (14 if case["backward"] else 4)}
    n = sum(math.prod(s) for s in shapes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / QUANT
    return {"bytes": n * (8 + TYPES[case["grads"]].itemsize + state + (2 if case["shadow"] else 0)), "flops": 20 * n}


# -- the same in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": exact_norm, "attention": exact_attention, "adamw": exact_adamw}[case["op"]](s)


def exact_norm(s):
    names = ("x", "scale", "bias") if s["bias"] is not None else ("x", "scale")
    leaves = [s[n].detach().to(F64).requires_grad_(s["dy"] is not None) for n in names]
    x = leaves[0]
    variance, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(variance + 1e-5) * leaves[1]
    if len(leaves) > 2:
        y = y + leaves[2]
    if s["dy"] is None:
        return {"y": y}
    return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, leaves, s["dy"].to(F64))))}


def exact_attention(s):
    """Head by head, the gradients by differentiating the formula."""

    c = s["case"]
    B, H, Hk, S, D = (c[k] for k in ("batch", "heads", "kv_heads", "seq", "dim"))
    back = s["do"] is not None
    leaf = {n: s[n].detach().to(F64) for n in "qkv"}
    out = {"o": torch.empty((B, H, S, D), dtype=F64, device=DEVICE)}
    if back:
        out.update({n: torch.zeros_like(leaf[n], memory_format=torch.contiguous_format) for n in "qkv"})
    i, j = torch.meshgrid(torch.arange(S, device=DEVICE), torch.arange(S, device=DEVICE), indexing="ij")
    for b in range(B):
        visible = j <= i
        if s["prefix"] is not None:
            visible = visible | (j < s["prefix"][b])
        if s["segments"] is not None:
            visible = visible & (s["segments"][b][i] == s["segments"][b][j])
        for h in range(H):
            kh = h // (H // Hk)
            q, k, v = (leaf[n][b, x].clone().requires_grad_(back) for n, x in (("q", h), ("k", kh), ("v", kh)))
            u = q @ k.T / math.sqrt(D)
            if c["cap"]:
                u = c["cap"] * torch.tanh(u / c["cap"])
            if s["slopes"] is not None:
                u = u - s["slopes"][h].to(F64) * (i - j).abs()
            o = torch.softmax(u.masked_fill(~visible, -math.inf), dim=1) @ v
            out["o"][b, h] = o.detach()
            if back:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"][b, h].to(F64))
                out["q"][b, h] = dq
                out["k"][b, kh] += dk
                out["v"][b, kh] += dv
    return out


def exact_adamw(s):
    case, L = s["case"], s["lists"]
    out = {k: t.to(F64) for k, t in s["flat"].items()}
    new = {k: views(t, shapes(case), QUANT if k in ("ms", "vs") else 1) for k, t in out.items()}
    for i, p in enumerate(L["p"]):
        g = s["grads"][i].to(F64).reshape(-1)
        if s["clip"] is not None:
            g = g * s["clip"].to(F64)
        if case["bits"] == 8:
            m0, v0 = (valued(L[a][i], L[b][i], F64) for a, b in (("m", "ms"), ("v", "vs")))
        else:
            m0, v0 = L["m"][i].to(F64).reshape(-1), L["v"][i].to(F64).reshape(-1)
        m = m0 + (1 - BETA1) * (g - m0)
        v = v0 + (1 - BETA2) * (g * g - v0)
        lr_mult, eps, decay = s["hparams"][i].to(F64)
        p1 = p.to(F64).reshape(-1)
        p1 = p1 * (1 - LR * lr_mult * decay) - LR * lr_mult * m / (1 - BETA1 ** STEP) / (
            (v / (1 - BETA2 ** STEP)).sqrt() + eps)
        new["p"][i].copy_(p1.view(p.shape))
        if case["shadow"]:
            new["shadow"][i].copy_(p1.view(p.shape))
        if case["bits"] == 8:
            um, uv = bits_as_steps(random_bits(s["seed"], i, p.numel()))
            m, new["ms"][i][:] = quantized(m, um.to(F64), False)
            v, new["vs"][i][:] = quantized(v, uv.to(F64), True)
        new["m"][i].copy_(m.view(p.shape))
        new["v"][i].copy_(v.view(p.shape))
    return out
