"""Cases, inputs and plain forms of the training operators around the optimiser: the embedding lookup with its gradient,
the norm of many gradients, clipping by it, and SparseGaussianAdam's step with the clipping folded in.

`listed()` and `draw(rng)` name cases, `prepare(case, seed)` makes what a program holds before the call, `run(state)` is one
pass: through the plain torch form, or through dogs_amd where `own` is true.  `exact(case, seed)` is the same pass in 64 bits,
`work(case)` what it has to move and compute.

Formulas (t_i token i, E the table, s the scale, G the gradient of the lookup's result):
    lookup   Y[i] = s E[t_i]
    gradient dE[v] = s sum over i with t_i = v of G[i], in the order of i; 0 for the padding token
    norm     n = sqrt(sum over all tensors and elements of g^2)
    clip     g <- g min(1, max_norm / (n + 1e-6))
    step     m <- b1 m + (1 - b1) c g;  v <- b2 v + (1 - b2) (c g)^2;  p <- p - lr m / (sqrt(v) + eps) on the visible rows,
             c = min(1, max_norm / (n + 1e-6)), with b1, b2 the 32-bit numbers nearest to 0.9 and 0.999
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
B1, B2 = float(np.float32(0.9)), float(np.float32(0.999))
EPS = 1e-15
VIEWS = 4          # views whose gradients a clipped step averages; a power of two, so that the mean rounds nothing
# learning rates and widths of a scene's six tensors (position, colour, higher colour, opacity, scale, rotation)
GROUPS = (("xyz", 3, 0.00016), ("f_dc", 3, 0.0025), ("f_rest", 45, 0.000125), ("opacity", 1, 0.025),
          ("scaling", 3, 0.005), ("quaternion", 4, 0.001))
ROW = sum(w for _, w, _ in GROUPS)


def listed():
    return [
        # the appearance code of the one view that a training iteration renders
        {"name": "lookup_code", "op": "lookup", "vocab": 256, "dim": 64, "tokens": 1, "dtype": "float32", "index": "int64"},
        # one new token for each of a few requests
        {"name": "lookup_token", "op": "lookup", "vocab": 65536, "dim": 4096, "tokens": 8, "dtype": "bfloat16", "index": "int32"},
        # prompts
        {"name": "lookup_prompt", "op": "lookup", "vocab": 131072, "dim": 4096, "tokens": 16384, "dtype": "bfloat16", "index": "int64"},
        # a batch of views' appearance codes, trained
        {"name": "train_codes", "op": "train", "vocab": 2000, "dim": 64, "tokens": 256, "dtype": "float32", "index": "int64"},
        # ragged sizes: rows that start at no aligned place
        {"name": "train_odd", "op": "train", "vocab": 50021, "dim": 1023, "tokens": 8191, "dtype": "float16", "index": "int32"},
        # a training batch of text: few tokens make up most of it
        {"name": "train_batch", "op": "train", "vocab": 131072, "dim": 2048, "tokens": 65536, "dtype": "bfloat16", "index": "int64"},
        # the appearance network's 15 small tensors
        {"name": "norm_network", "op": "norm", "of": "network", "size": 500, "count": 1, "dtype": "float32"},
        # a scene of a million Gaussians
        {"name": "norm_scene", "op": "norm", "of": "scene", "size": 1000000, "count": 1, "dtype": "float32"},
        # the appearance network's step, clipped
        {"name": "clip_network", "op": "clip", "of": "network", "size": 500, "count": 1, "dtype": "float32", "max_norm": 0.5},
        # layers of a larger network
        {"name": "clip_layers", "op": "clip", "of": "layers", "size": 4096, "count": 2, "dtype": "bfloat16", "max_norm": 1.0},
        # the clipped step of a small scene, and of a large one
        {"name": "step_small", "op": "step", "rows": 20011, "visible": 0.7, "max_norm": 0.1},
        {"name": "step_scene", "op": "step", "rows": 1000000, "visible": 0.6, "max_norm": 0.1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("lookup", "train", "train", "norm", "clip", "step"))
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    if op in ("lookup", "train"):
        dim = _log(rng, 8, 4096)
        return {"op": op, "vocab": _log(rng, 64, 131072 * 2048 // max(dim, 2048)), "dim": dim,
                "tokens": _log(rng, 1, min(65536, 65536 * 2048 // dim)), "dtype": dtype, "index": rng.choice(("int64", "int32"))}
    if op == "step":
        return {"op": op, "rows": _log(rng, 1000, 1000000), "visible": round(rng.uniform(0.05, 1.0), 3),
                "max_norm": round(10 ** rng.uniform(-2, 1), 4)}
    of = rng.choice(("network", "scene", "layers"))
    case = {"op": op, "of": of, "dtype": "float32" if of != "layers" else dtype,
            "size": _log(rng, 20, 5000) if of == "network" else _log(rng, 1000, 1000000) if of == "scene" else _log(rng, 64, 2048),
            "count": rng.randint(1, 6) if of == "layers" else 1}
    if op == "clip":
        case["max_norm"] = round(10 ** rng.uniform(-2, 1), 4)
    return case


def _shapes(case):
    """The gradients' shapes: the appearance network over `size` views, a scene of `size` rows, or `count` layers of width `size`."""
    n = case["size"]
    if case["of"] == "scene":
        return [(n, w) for _, w, _ in GROUPS]
    if case["of"] == "layers":  # two vectors, four square matrices and two wide ones
        return [(n,), (n, n), (n, n), (n, n), (n, n), (n,), (2 * n, n), (n, 2 * n)] * case["count"]
    convs = ((67, 256), (64, 128), (32, 64), (16, 32), (8, 16), (16, 8), (8, 3))
    return [(n, 64)] + [s for cin, cout in convs for s in ((cout, cin, 3, 3), (cout,))]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tokens(case, gen):
    """Text-like: token v about as frequent as 1 / (v + 2.7), the ids shuffled; codes of views uniformly."""
    v, n = case["vocab"], case["tokens"]
    u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
    if case["dim"] <= 64:
        t = (u * v).long()
    else:
        t = (2.7 * ((v + 2.7) / 2.7) ** u - 2.7).long()
        t = torch.randperm(v, device="cuda", generator=gen)[t.clamp_(0, v - 1)]
    return t.clamp_(0, v - 1).to(torch.int64 if case["index"] == "int64" else torch.int32)


def prepare(case, seed):
    gen = _generator(seed)

    def normal(shape, dtype, std=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)

    state = dict(case)
    if case["op"] in ("lookup", "train"):
        dtype = DTYPES[case["dtype"]]
        state["scale"] = math.sqrt(case["dim"])
        state["tokens"] = _tokens(case, gen)
        state["table"] = normal((case["vocab"], case["dim"]), dtype, 0.02).requires_grad_(case["op"] == "train")
        if case["op"] == "train":
            # ragged sequences: some of the batch is padding, whose row learns nothing
            state["padding"] = case["vocab"] - 1
            state["tokens"][torch.rand(case["tokens"], device="cuda", generator=gen) < 0.05] = case["vocab"] - 1
            state["grad"] = normal((case["tokens"], case["dim"]), dtype, 1e-3)
    elif case["op"] in ("norm", "clip"):
        dtype = DTYPES[case["dtype"]]
        state["grads"] = [normal(s, dtype, 1e-2 / (1 + k % 5)) for k, s in enumerate(_shapes(case))]
        if case["op"] == "clip":
            state["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in state["grads"]]
    else:
        n = case["rows"]
        state["visible"] = torch.rand(n, device="cuda", generator=gen) < case["visible"]
        seen = state["visible"][:, None].float()
        state["params"] = [torch.nn.Parameter(normal((n, w), torch.float32)) for _, w, _ in GROUPS]
        state["grads"] = [normal((n, w), torch.float32, 1e-4) * seen for _, w, _ in GROUPS]
        state["m"] = [normal((n, w), torch.float32, 1e-5) for _, w, _ in GROUPS]
        state["v"] = [normal((n, w), torch.float32, 1e-5).square() + 1e-12 for _, w, _ in GROUPS]
        if own:  # the optimiser that a program holds; the plain form works on the same tensors
            state["optimizer"] = _optimizer(state)
    return state


def _optimizer(state):
    from dogs_amd.diff_gaussian_rasterization import SparseGaussianAdam
    opt = SparseGaussianAdam([{"params": [p], "lr": lr, "name": name} for p, (name, _, lr) in zip(state["params"], GROUPS)],
                             lr=0.0, eps=EPS)
    for p, g, m, v in zip(state["params"], state["grads"], state["m"], state["v"]):
        p.grad = g
        opt.state[p] = {"step": torch.tensor(0.0), "exp_avg": m, "exp_avg_sq": v}
    return opt


def run(state):
    return {"lookup": _lookup, "train": _train, "norm": _norm, "clip": _clip, "step": _step}[state["op"]](state)


def _lookup(state):
    table, tokens, scale = state["table"], state["tokens"], state["scale"]
    if own:
        from dogs_amd.embedding import embedding_lookup
        return embedding_lookup(table, tokens, scale=scale)
    return (table[tokens].float() * scale).to(table.dtype)


def _train(state):
    table, tokens, scale, grad, pad = (state[k] for k in ("table", "tokens", "scale", "grad", "padding"))
    if own:
        from dogs_amd.embedding import embedding_lookup
        out = embedding_lookup(table, tokens, scale=scale, padding_idx=pad)
        return [out.detach(), *torch.autograd.grad(out, table, grad)]
    with torch.no_grad():
        out = (table[tokens].float() * scale).to(table.dtype)
        total = torch.zeros(table.shape, dtype=torch.float32, device=table.device).index_add_(0, tokens, grad.float())
        total[pad] = 0.0
        return [out, (total * scale).to(table.dtype)]


def _total_norm(grads):
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def _coefficient(norm, max_norm):
    return (max_norm / (norm + 1e-6)).clamp(max=1.0)


def _norm(state):
    if own:
        from dogs_amd.gradclip import grad_norm
        return grad_norm(state["grads"])
    return _total_norm(state["grads"])


def _set_grad(param, grad):
    param.grad = grad


def _clip(state):
    # the gradients of VIEWS views, averaged: new ones each pass, as a backward pass would leave them
    grads = torch._foreach_mul(state["grads"], 1.0 / VIEWS)
    if own:
        from dogs_amd.gradclip import clip_grad_norm_
        list(map(_set_grad, state["params"], grads))
        return [clip_grad_norm_(state["params"], state["max_norm"]), *grads]
    norm = _total_norm(grads)
    c = _coefficient(norm, state["max_norm"])
    return [norm, *[g.copy_(g.float() * c) for g in grads]]


def _plain_adam(p, g, m, v, lr, c, seen):
    g = g * c
    new_m = m * B1 + g * (1.0 - B1)
    new_v = v * B2 + g * g * (1.0 - B2)
    p.copy_(torch.where(seen, p - lr * new_m / (new_v.sqrt() + EPS), p))
    m.copy_(torch.where(seen, new_m, m))
    v.copy_(torch.where(seen, new_v, v))


def _step(state):
    if own:
        norm = state["optimizer"].step(state["visible"], state["rows"], max_norm=state["max_norm"])
    else:
        with torch.no_grad():
            norm = _total_norm(state["grads"])
            c = _coefficient(norm, state["max_norm"])
            seen = state["visible"][:, None]
            [_plain_adam(p, g, m, v, lr, c, seen) for p, g, m, v, (_, _, lr) in
             zip(state["params"], state["grads"], state["m"], state["v"], GROUPS)]
    return [norm, *[p.detach() for p in state["params"]], *state["m"], *state["v"]]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("lookup", "train"):
        with torch.no_grad():
            table, tokens, scale = state["table"].double(), state["tokens"].long(), state["scale"]
            out = torch.index_select(table, 0, tokens).mul_(scale)
            if case["op"] == "lookup":
                return out
            del table
            kept = tokens != state["padding"]
            rows = state["grad"].double()[kept] * scale
            d = torch.zeros((case["vocab"], case["dim"]), dtype=torch.float64, device="cuda")
            return [out, d.index_put_((tokens[kept],), rows, accumulate=True)]
    squares = [float((g.double() ** 2).sum()) for g in state["grads"]]
    norm = math.sqrt(math.fsum(squares))
    if case["op"] == "norm":
        return torch.tensor(norm, dtype=torch.float64)
    if case["op"] == "clip":
        norm /= VIEWS
        c = min(1.0, case["max_norm"] / (norm + 1e-6))
        return [torch.tensor(norm, dtype=torch.float64), *[g.double() * (c / VIEWS) for g in state["grads"]]]
    c = min(1.0, case["max_norm"] / (norm + 1e-6))
    seen = state["visible"]
    params, moments, squares = [], [], []
    for p, g, m, v, (_, _, lr) in zip(state["params"], state["grads"], state["m"], state["v"], GROUPS):
        p, g, m, v = p.detach().double(), g.double()[seen] * c, m.double(), v.double()
        m[seen] = torch.lerp(g, m[seen], B1)
        v[seen] = torch.lerp(g ** 2, v[seen], B2)
        p[seen] -= lr * m[seen] / (torch.sqrt(v[seen]) + EPS)
        params.append(p)
        moments.append(m)
        squares.append(v)
    return [torch.tensor(norm, dtype=torch.float64), *params, *moments, *squares]


def work(case):
    if case["op"] in ("lookup", "train"):
        b, n, v, d = BYTES[case["dtype"]], case["tokens"], case["vocab"], case["dim"]
        forward = (min(n, v) + n) * d * b + n * (8 if case["index"] == "int64" else 4)
        if case["op"] == "lookup":
            return {"bytes": forward, "flops": n * d}
        return {"bytes": forward + (n + v) * d * b, "flops": 2 * n * d + v * d}
    if case["op"] == "step":
        n, seen = case["rows"] * ROW, case["rows"] * ROW * case["visible"]
        return {"bytes": 4 * n + 24 * seen + case["rows"], "flops": 2 * n + 12 * seen}
    n, b = sum(math.prod(s) for s in _shapes(case)), BYTES[case["dtype"]]
    return {"bytes": n * b * (1 if case["op"] == "norm" else 2), "flops": 2 * n + (n if case["op"] == "clip" else 0)}
