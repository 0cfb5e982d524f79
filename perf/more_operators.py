"""Token embedding with scaling, a gated feed-forward block, and the
orthogonalisation of updates by Newton-Schulz products, as cases that can be
timed and compared.

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

import torch

own = False

DEVICE = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": BF16, "f32": F32}
VOCAB = 50304  # storage rows of the embedding, as in the benchmark's model
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


def listed() -> list[dict]:
    return [
        # Looking up one prompt: the smallest call, where its launch counts.
        embedding("embedding-prompt", tokens=129, width=768, backward=False),
        # The embedding of the 125M model in training, at the tokens of a micro-batch.
        embedding("embedding-train", tokens=65536, width=768),
        # A byte-level model: few rows, each the sum of hundreds of tokens, a table held in bf16.
        embedding("embedding-bytes", tokens=131072, width=512, vocab=260, table="bf16"),
        # Padded batches, float32 activations scaled by the width's root, a width that is no multiple of a vector.
        embedding("embedding-odd", tokens=8191, width=1001, vocab=20011, out="f32", scale=True, padding=True),
        # One generated token through the block.
        gated("gated-token", tokens=1, width=768, hidden=2048, backward=False),
        # One prompt through the block.
        gated("gated-prompt", tokens=129, width=768, hidden=2048, backward=False),
        # The block in training at the 125M model's width and the tokens of a micro-batch.
        gated("gated-train", tokens=65536, width=768, hidden=2048),
        # GELU for the gate, sizes that are no multiples of any tile.
        gated("gated-odd", tokens=5001, width=1000, hidden=2664, activation="gelu"),
        # The updates of a small model, where the launches count.
        model("orthogonal-small", width=256, hidden=680, layers=2),
        # The updates of the 125M model's width, all layers.
        model("orthogonal-768", width=768, hidden=2048, layers=12),
        # The same at 960, bf16 momenta.
        model("orthogonal-960", width=960, hidden=2560, layers=12, dtype="bf16"),
        # One routed layer's expert matrices, of odd sizes.
        matrices("orthogonal-experts", count=7, rows=509, columns=1201),
    ]


def embedding(name, tokens, width, vocab=VOCAB, table="f32", out="bf16", scale=False, padding=False,
              backward=True) -> dict:
    return dict(name=name, op="embedding", tokens=tokens, width=width, vocab=vocab, table=table, out=out, scale=scale,
                padding=padding, backward=backward)


def gated(name, tokens, width, hidden, activation="silu", backward=True) -> dict:
    return dict(name=name, op="gated", tokens=tokens, width=width, hidden=hidden, activation=activation,
                backward=backward)


def model(name, width, hidden, layers, dtype="f32") -> dict:
    """The matrices of a model's blocks, a tensor each."""

    return dict(name=name, op="model", width=width, hidden=hidden, layers=layers, dtype=dtype)


def matrices(name, count, rows, columns, dtype="f32") -> dict:
    """One tensor of several matrices, as a routed layer holds its experts."""

    return dict(name=name, op="matrices", count=count, rows=rows, columns=columns, dtype=dtype)


def spread(rng, low, high) -> int:
    """A whole number between low and high, even over their logarithm."""

    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    op = rng.choice(("embedding", "gated", "gated", "model", "matrices"))
    if op == "embedding":
        width = rng.choice((256, 512, 768, 1024, spread(rng, 32, 2048)))
        tokens = spread(rng, 1, min(131072, 2 ** 26 // width))
        vocab = spread(rng, 100, min(VOCAB, 2 ** 26 // width))
        case = embedding("", tokens, width, vocab, rng.choice(("f32", "f32", "bf16")),
                         rng.choice(("bf16", "bf16", "f32")), rng.random() < 0.5, rng.random() < 0.4,
                         rng.random() < 0.7)
    elif op == "gated":
        width = 8 * spread(rng, 16, 192)
        hidden = 8 * spread(rng, 16, 512)
        tokens = spread(rng, 1, min(65536, 10 ** 11 // (width * hidden)))
        case = gated("", tokens, width, hidden, rng.choice(("silu", "silu", "gelu")), rng.random() < 0.7)
    elif op == "model":
        width = spread(rng, 64, 960)
        hidden = min(2560, round(width * rng.uniform(1.5, 4.0)))
        case = model("", width, hidden, rng.randint(1, 12), rng.choice(("f32", "f32", "bf16")))
    else:
        rows, columns = spread(rng, 1, 2048), spread(rng, 1, 2048)
        case = matrices("", spread(rng, 1, 32), rows, columns, rng.choice(("f32", "bf16")))
    del case["name"]
    return case


# -- what a program has in hand ---------------------------------------------------


def generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def prepare(case, seed):
    return {"embedding": prepare_embedding, "gated": prepare_gated, "model": prepare_updates,
            "matrices": prepare_updates}[case["op"]](case, seed)


def prepare_embedding(case, seed):
    g = generator(seed)
    n, d, vocab, back = case["tokens"], case["width"], case["vocab"], case["backward"]
    # Token k comes up about as often as 1 / (k + 1): a few rows take a large share of the gradient.
    u = torch.rand(n, generator=g, device=DEVICE, dtype=F64)
    tokens = torch.floor(torch.exp(u * math.log(vocab + 1)) - 1).clamp(0, vocab - 1).to(torch.int32)
    if case["padding"]:  # the last tenth of the batch is padding, and belongs to no row
        tokens[n - n // 10:] = -1
    table = 0.02 * torch.randn((vocab, d), generator=g, device=DEVICE)
    dy = torch.randn((n, d), generator=g, device=DEVICE).to(TYPES[case["out"]]) if back else None
    return dict(case=case, tokens=tokens, table=table.to(TYPES[case["table"]]).requires_grad_(back), dy=dy,
                scale=math.sqrt(d) if case["scale"] else 1.0)


def prepare_gated(case, seed):
    g = generator(seed)
    n, d, f, back = case["tokens"], case["width"], case["hidden"], case["backward"]

    def normal(rows, columns, scale):
        return (torch.randn((rows, columns), generator=g, device=DEVICE) * scale).to(BF16)

    return dict(case=case, x=normal(n, d, 1.0).requires_grad_(back),
                gate_up_w=normal(d, 2 * f, d ** -0.5).requires_grad_(back),
                down_w=normal(f, d, f ** -0.5).requires_grad_(back), dy=normal(n, d, 1.0) if back else None)


def shapes(case) -> list[tuple[int, ...]]:
    if case["op"] == "matrices":
        return [(case["count"], case["rows"], case["columns"])]
    d, f = case["width"], case["hidden"]
    return [(d, 3 * d), (d, d), (d, 2 * f), (f, d)] * case["layers"]


def prepare_updates(case, seed):
    """Momenta: a few strong directions that fall off, over a floor of noise."""

    g = generator(seed)
    updates = []
    for *lead, rows, columns in shapes(case):
        rank = max(1, min(rows, columns) // 8)
        fall = 1.0 / torch.arange(1, rank + 1, device=DEVICE, dtype=F32)
        a = torch.randn((*lead, rows, rank), generator=g, device=DEVICE) * fall
        b = torch.randn((*lead, rank, columns), generator=g, device=DEVICE)
        noise = torch.randn((*lead, rows, columns), generator=g, device=DEVICE)
        updates.append((1e-3 * (torch.matmul(a, b) + 0.1 * noise)).to(TYPES[case["dtype"]]))
    return dict(case=case, updates=updates)


# -- one pass ----------------------------------------------------------------------


def run(state):
    return {"embedding": run_embedding, "gated": run_gated, "model": run_updates,
            "matrices": run_updates}[state["case"]["op"]](state)


def package():
    path = os.path.join(os.getcwd(), "gpt-speedrun-tpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)


def run_embedding(s):
    out = TYPES[s["case"]["out"]]
    if own:
        package()
        from gptrig.nn import embedding as lookup

        y = lookup(s["tokens"], s["table"], scale=s["scale"], dtype=out)
        if s["dy"] is None:
            return {"y": y}
        return {"y": y.detach(), "table": torch.autograd.grad(y, s["table"], s["dy"])[0]}
    tokens, table = s["tokens"].long(), s["table"].detach()
    inside = (tokens >= 0) & (tokens < table.shape[0])
    at = torch.where(inside, tokens, 0)
    y = table[at].to(F32) * s["scale"] * inside[:, None]
    result = {"y": y.to(out)}
    if s["dy"] is not None:  # (long sums, in 64 bits)
        grad = torch.zeros(table.shape, dtype=F64, device=DEVICE)
        grad.index_add_(0, at, s["dy"].to(F64) * inside[:, None])
        result["table"] = (grad * s["scale"]).to(table.dtype)
    return result


def activated(g, kind):
    """The activation and its derivative."""

    if kind == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p * (1 + g * (1 - p))
    k, c = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(k * (g + c * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * c * g * g)


def run_gated(s):
    names = ("x", "gate_up_w", "down_w")
    if own:
        package()
        from gptrig.nn import gated_mlp

        y = gated_mlp(s["x"], s["gate_up_w"], s["down_w"], activation=s["case"]["activation"])
        if s["dy"] is None:
            return {"y": y}
        return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, [s[n] for n in names], s["dy"])))}
    x, w, v = (s[n].detach().to(F32) for n in names)
    f = v.shape[0]
    p = torch.mm(x, w)
    g, u = p[:, :f], p[:, f:]
    a, slope = activated(g, s["case"]["activation"])
    h = a * u
    out = {"y": torch.mm(h, v).to(BF16)}
    if s["dy"] is None:
        return out
    dy = s["dy"].to(F32)
    dh = torch.mm(dy, v.t().contiguous())
    dp = torch.cat((dh * u * slope, dh * a), 1)
    out["x"] = torch.mm(dp, w.t().contiguous()).to(BF16)
    out["gate_up_w"] = torch.mm(x.t().contiguous(), dp).to(BF16)
    out["down_w"] = torch.mm(h.t().contiguous(), dy).to(BF16)
    return out


def run_updates(s):
    if own:
        package()
        from gptrig.optim import orthogonalize_tensors

        return orthogonalize_tensors(s["updates"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    a, b, c = COEFFICIENTS
    out = []
    for update in s["updates"]:
        x = update.to(F32).reshape(-1, *update.shape[-2:])
        x = x / (x.to(F64).square().sum((1, 2), keepdim=True).sqrt() + EPS).to(F32)
        tall = x.shape[1] > x.shape[2]
        if tall:
            x = x.transpose(1, 2).contiguous()
        for _ in range(STEPS):
            gram = torch.bmm(x, x.transpose(1, 2).contiguous())
            x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
        out.append((x.transpose(1, 2) if tall else x).to(BF16).reshape(update.shape))
    return out


# -- what it cannot do without --------------------------------------------------------


def work(case) -> dict:
    if case["op"] == "embedding":
        n, d, vocab = case["tokens"], case["width"], case["vocab"]
        out, table = TYPES[case["out"]].itemsize, TYPES[case["table"]].itemsize
        share = torch.log1p(1 / torch.arange(1, vocab + 1, dtype=F64)) / math.log(vocab + 1)
        rows = -torch.expm1(-n * share).sum().item()  # (different rows that are read, as they are drawn)
        if case["backward"]:
            return {"bytes": 8 * n + n * d * out * 2 + rows * d * table + vocab * d * table, "flops": 2 * n * d}
        return {"bytes": 4 * n + n * d * out + rows * d * table, "flops": n * d}
    if case["op"] == "gated":
        n, d, f = case["tokens"], case["width"], case["hidden"]
        weights = 2 * 3 * d * f
        if case["backward"]:
            return {"bytes": 2 * 4 * n * d + 2 * weights, "flops": 18 * n * d * f}
        return {"bytes": 2 * 2 * n * d + weights, "flops": 6 * n * d * f}
    # Of the three products of a step two are symmetric, and half of each is enough.
    moved = flops = 0.0
    for shape in shapes(case):
        count, m, n = math.prod(shape[:-2]), min(shape[-2:]), max(shape[-2:])
        moved += count * m * n * (TYPES[case["dtype"]].itemsize + 2)
        flops += count * STEPS * (m * m * n * 3 + m * m * m)
    return {"bytes": moved, "flops": flops}


# -- the same in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"embedding": exact_embedding, "gated": exact_gated, "model": exact_updates,
            "matrices": exact_updates}[case["op"]](s)


def exact_embedding(s):
    """The rows of a one-hot product, token after token in sorted order."""

    case, table = s["case"], s["table"].detach().to(F64)
    tokens, d = s["tokens"].long(), case["width"]
    padded = torch.cat((table * s["scale"], torch.zeros((1, d), dtype=F64, device=DEVICE)))
    tokens = torch.where((tokens < 0) | (tokens >= case["vocab"]), case["vocab"], tokens)
    out = {"y": torch.index_select(padded, 0, tokens)}
    if s["dy"] is not None:
        order = torch.argsort(tokens, stable=True)
        counts = torch.bincount(tokens, minlength=case["vocab"] + 1)
        ends = torch.cumsum(counts, 0)
        grad = torch.empty((case["vocab"], d), dtype=F64, device=DEVICE)
        for at in range(0, d, 64):
            total = torch.cumsum(s["dy"][:, at:at + 64].to(F64)[order], 0)
            total = torch.cat((torch.zeros_like(total[:1]), total))
            grad[:, at:at + 64] = (total[ends] - total[ends - counts])[:-1]
        out["table"] = grad * s["scale"]
    return out


def exact_gated(s):
    names = ("x", "gate_up_w", "down_w")
    back = s["dy"] is not None
    leaves = [s[n].detach().to(F64).requires_grad_(back) for n in names]
    x, w, v = leaves
    gate, up = torch.matmul(x, w).split(v.shape[0], dim=1)
    if s["case"]["activation"] == "silu":
        a = gate * torch.sigmoid(gate)
    else:
        a = gate * torch.sigmoid(math.sqrt(8 / math.pi) * (gate + 0.044715 * gate ** 3))
    y = torch.matmul(a * up, v)
    if not back:
        return {"y": y}
    return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, leaves, s["dy"].to(F64))))}


def exact_updates(s):
    """Matrix by matrix, with the products on the longer side's right where the plain form has them on the left."""

    a, b, c = COEFFICIENTS
    out = []
    for update in s["updates"]:
        result = torch.empty(update.shape, dtype=F64, device=DEVICE)
        flat = update.reshape(-1, *update.shape[-2:])
        for i, u in enumerate(flat):
            x = u.to(F64)
            x = x / (torch.linalg.norm(x) + EPS)
            x = x if x.shape[0] >= x.shape[1] else x.T.contiguous()
            one = torch.eye(x.shape[1], dtype=F64, device=DEVICE)
            for _ in range(STEPS):
                k = torch.mm(x.T.contiguous(), x)
                x = torch.mm(x, a * one + torch.mm(k, b * one + c * k))
            result.view_as(flat)[i] = x if x.shape == u.shape else x.T
        out.append(result)
    return out
