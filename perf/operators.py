"""Workloads of the dense training operators: the fused linear, the gated feed-forward block
and the global gradient norm with clipping.

Each case is one call as a user's program makes it.  ``run`` computes it from elementary torch
operations in 32 bits, or, with ``own`` set, through the package's entry points.

    linear       y = residual + act(x W^T + b), and its backward
    ffn          out = residual + down(act(gate(x)) * up(x)), and its backward
    clip         total norm of many gradients, which are scaled when it exceeds max_norm
"""
import math

import torch

own = False

ACTIVATIONS = ("none", "relu", "silu", "gelu_tanh", "era")
GAMMA = 0.1  # ERA's softplus weight, MoEConfig's default
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------ the cases
def _linear(name, tokens, k, n, act="none", dtype="bf16", bias=True, residual=False, train=False):
    return {"name": name, "op": "linear", "tokens": tokens, "in": k, "out": n, "act": act,
            "dtype": dtype, "bias": bias, "residual": residual, "train": train}


def _ffn(name, tokens, h, i, act="era", dtype="bf16", bias=True, residual=False, train=False):
    return {"name": name, "op": "ffn", "tokens": tokens, "hidden": h, "inter": i, "act": act,
            "dtype": dtype, "bias": bias, "residual": residual, "train": train}


def _clip(name, experts, h, i, rank, dtype, clipped, first=0):
    return {"name": name, "op": "clip", "experts": experts, "hidden": h, "inter": i, "rank": rank,
            "dtype": dtype, "clipped": clipped, "first": first}


def listed():
    return [
        # one generated token through a projection that adds to the residual stream
        _linear("linear_token", 1, 2048, 2048, residual=True),
        # a decode batch through a widening projection with its activation
        _linear("linear_decode", 64, 2048, 8192, act="gelu_tanh"),
        # a training micro-batch through a square projection with the residual
        _linear("linear_train", 16384, 2048, 2048, act="silu", residual=True, train=True),
        # a ragged packed batch; rows that no 16-byte load divides
        _linear("linear_train_odd", 1003, 1001, 777, act="era", residual=True, train=True),
        # the single-precision layer of the smallest configuration
        _linear("linear_train_f32", 512, 768, 1024, dtype="f32", train=True),
        # one generated token through the dense block
        _ffn("ffn_token", 1, 2048, 8192, residual=True),
        # a decode batch through the dense block
        _ffn("ffn_decode", 64, 2048, 8192, residual=True),
        # a short ragged training batch, widths off every tile
        _ffn("ffn_train_odd", 777, 520, 1304, residual=True, train=True),
        # the prefill configuration's sizes as one training micro-batch
        _ffn("ffn_train_large", 32768, 2048, 8192, train=True),
        # the gradients of one small dense block, clipped
        _clip("clip_ffn", 1, 768, 2048, 16, "bf16", True),
        # a mixture layer's gradients in two types from odd addresses, clipped
        _clip("clip_moe_mixed", 8, 1024, 2048, 16, "mixed", True, first=3),
        # a fine-grained mixture layer's gradients, below the limit
        _clip("clip_moe_fine", 64, 1024, 2048, 16, "f32", False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "ffn", "clip"))
    if op == "clip":
        experts = _log(rng, 1, 64)
        h = rng.randrange(64, 1025)
        i = rng.randrange(64, 2049)
        return {"op": op, "experts": experts, "hidden": h, "inter": i, "rank": rng.randrange(1, 33),
                "dtype": rng.choice(("f32", "bf16", "mixed")), "clipped": rng.random() < 0.5,
                "first": rng.randrange(0, 8)}
    train = rng.random() < 0.6
    dtype = "f32" if rng.random() < 0.2 else "bf16"
    tokens = _log(rng, 1, 2048 if dtype == "f32" else 16384)
    odd = rng.random() < 0.3
    step = 1 if odd else 8

    def width(lo, hi):
        return max(step, _log(rng, lo, hi) // step * step)

    c = {"op": op, "tokens": tokens, "dtype": dtype, "bias": rng.random() < 0.7,
         "residual": rng.random() < 0.5, "train": train}
    if op == "linear":
        c["in"], c["out"] = width(48, 4096), width(48, 8192)
        c["act"] = rng.choice(ACTIVATIONS)
    else:
        c["hidden"], c["inter"] = width(48, 2048), width(48, 8192)
        c["act"] = rng.choice(ACTIVATIONS[1:])
    return c


# ------------------------------------------------------------------------------ the inputs
def _clip_shapes(c):
    """The gradients of a mixture layer (a router and FlyLoRA experts), or of one dense block."""
    h, i, r, e = c["hidden"], c["inter"], c["rank"], c["experts"]
    one = 2 * [(i, h), (i,), (r, h), (r,), (i, r), (i,)] + [(h, i), (h,)]
    return ([(e, h), (e,)] if e > 1 else []) + e * one


def _clip_types(c, shapes):
    """Matrices in bf16 and vectors in f32 for the mixed case."""
    if c["dtype"] == "mixed":
        return ["bf16" if len(s) == 2 else "f32" for s in shapes]
    return [c["dtype"]] * len(shapes)


def _randn(gen, shape, std, dtype):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    c = dict(case)
    if c["op"] == "clip":
        shapes = _clip_shapes(c)
        types = _clip_types(c, shapes)
        s = {"case": c, "fresh": [], "flat": [], "params": []}
        parts = {}
        for kind in sorted(set(types)):  # one flat buffer of gradients per type, as buckets are
            n = c["first"] + sum(math.prod(sh) for sh, t in zip(shapes, types) if t == kind)
            s["fresh"].append(_randn(gen, (n,), 0.02, _TYPES[kind]))
            s["flat"].append(s["fresh"][-1].clone())
            parts[kind] = [s["flat"][-1], torch.zeros(n, device="cuda", dtype=_TYPES[kind]), c["first"]]
        for sh, t in zip(shapes, types):
            flat, weights, at = parts[t]
            p = torch.nn.Parameter(weights[at:at + math.prod(sh)].view(sh))
            p.grad = flat[at:at + math.prod(sh)].view(sh)
            parts[t][2] = at + math.prod(sh)
            s["params"].append(p)
        total = sum(math.prod(sh) for sh in shapes)
        s["max_norm"] = 0.02 * math.sqrt(total) * (0.25 if c["clipped"] else 2.0)
        return s
    dtype, t = _TYPES[c["dtype"]], c["tokens"]
    k = c["in"] if c["op"] == "linear" else c["hidden"]
    n = c["out"] if c["op"] == "linear" else c["hidden"]
    s = {"case": c, "x": _randn(gen, (t, k), 1.0, dtype)}
    if c["op"] == "linear":
        s["w"] = _randn(gen, (n, k), 0.02, dtype)
        s["b"] = _randn(gen, (n,), 0.02, dtype) if c["bias"] else None
    else:
        i = c["inter"]
        s["wg"], s["wu"] = (_randn(gen, (i, k), 0.02, dtype) for _ in range(2))
        s["wd"] = _randn(gen, (k, i), 0.02, dtype)
        s["bg"], s["bu"] = ((_randn(gen, (i,), 0.02, dtype) if c["bias"] else None) for _ in range(2))
        s["bd"] = _randn(gen, (k,), 0.02, dtype) if c["bias"] else None
    s["r"] = _randn(gen, (t, n), 1.0, dtype) if c["residual"] else None
    if c["train"]:
        s["dy"] = _randn(gen, (t, n), 1.0, dtype)
        for name in _leaves(c):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def _leaves(c):
    return ("x", "w", "b", "r") if c["op"] == "linear" else ("x", "wg", "bg", "wu", "bu", "wd", "bd", "r")


# ------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    if op == "clip":
        return _plain_clip(state)
    with torch.no_grad():
        return _plain_linear(state) if op == "linear" else _plain_ffn(state)


def _run_own(s, op):
    import velvetoptimizer_b200 as vb
    c = s["case"]
    if op == "clip":
        if c["clipped"]:  # the backward's part: new gradients in the buckets
            torch._foreach_copy_(s["flat"], s["fresh"])
        norm = vb.clip_grad_norm_(s["params"], s["max_norm"])
        return {"norm": norm, "grads": s["flat"]}
    if op == "linear":
        def call():
            return vb.linear(s["x"], s["w"], s["b"], residual=s["r"], activation=c["act"], gamma=GAMMA)
    else:
        def call():
            return vb.gated_ffn(s["x"], s["wg"], s["wu"], s["wd"], s["bg"], s["bu"], s["bd"],
                                residual=s["r"], activation=c["act"], gamma=GAMMA)
    if not c["train"]:
        with torch.no_grad():
            return {"y": call()}
    y = call()
    names = [n for n in _leaves(c) if s[n] is not None]
    got = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(names, got)}}


def _act(z, kind):
    """act(z) and its derivative."""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        d = (z > 0).to(z.dtype)
        return z * d, d
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    # gelu(z) = z sigmoid(2 q) with q = sqrt(2/pi) (z + 0.044715 z^3)
    q2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
    s = 1 / (1 + torch.exp(-q2))
    a = z * s
    d = s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if kind == "era":
        soft = torch.where(z > 20, z, torch.log1p(torch.exp(torch.clamp(z, max=20))))
        a = a + GAMMA * soft
        d = d + GAMMA * torch.where(z > 20, torch.ones_like(z), 1 / (1 + torch.exp(-z)))
    return a, d


def _f(t):
    return None if t is None else t.float()


def _affine(x, w, b):
    z = x @ w.t()
    return z if b is None else z + b


def _to(c, **outs):
    dtype = _TYPES[c["dtype"]]
    return {k: v.to(dtype) for k, v in outs.items() if v is not None}


def _plain_linear(s):
    c = s["case"]
    x, w, b, r = _f(s["x"]), _f(s["w"]), _f(s["b"]), _f(s["r"])
    z = _affine(x, w, b)
    a, d = _act(z, c["act"])
    y = a if r is None else r + a
    if not c["train"]:
        return _to(c, y=y)
    dy = _f(s["dy"])
    dz = dy * d
    return _to(c, y=y, dx=dz @ w, dw=dz.t() @ x, db=None if b is None else dz.sum(0),
               dr=None if r is None else dy)


def _plain_ffn(s):
    c = s["case"]
    x, r = _f(s["x"]), _f(s["r"])
    wg, wu, wd, bg, bu, bd = (_f(s[n]) for n in ("wg", "wu", "wd", "bg", "bu", "bd"))
    g, u = _affine(x, wg, bg), _affine(x, wu, bu)
    a, d = _act(g, c["act"])
    h = a * u
    y = _affine(h, wd, bd)
    y = y if r is None else r + y
    if not c["train"]:
        return _to(c, y=y)
    dy = _f(s["dy"])
    dh = dy @ wd
    du, dg = dh * a, dh * u * d
    return _to(c, y=y, dx=dg @ wg + du @ wu, dwg=dg.t() @ x, dwu=du.t() @ x, dwd=dy.t() @ h,
               dbg=None if bg is None else dg.sum(0), dbu=None if bu is None else du.sum(0),
               dbd=None if bd is None else dy.sum(0), dr=None if r is None else dy)


def _plain_clip(s):
    c = s["case"]
    if c["clipped"]:
        torch._foreach_copy_(s["flat"], s["fresh"])
    parts = [f[c["first"]:].float() for f in s["flat"]]
    total = torch.stack([p.square().sum(dtype=torch.float64) for p in parts]).sum().sqrt()
    coef = torch.clamp(s["max_norm"] / (total + 1e-6), max=1.0).float()
    torch._foreach_copy_([f[c["first"]:] for f in s["flat"]], [(p * coef) for p in parts])
    return {"norm": total.float(), "grads": s["flat"]}


# ------------------------------------------------------------------------------ work, exact
def work(case):
    c = case
    if c["op"] == "clip":
        sizes = {"bf16": 2, "f32": 4}
        shapes = _clip_shapes(c)
        n = sum(math.prod(sh) * sizes[t] for sh, t in zip(shapes, _clip_types(c, shapes)))
        elems = sum(math.prod(sh) for sh in shapes)
        # new gradients are read and written, then read for the norm, read and written scaled
        return {"bytes": n * (5 if c["clipped"] else 1), "flops": elems * (3 if c["clipped"] else 2)}
    e, t = (2 if c["dtype"] == "bf16" else 4), c["tokens"]
    if c["op"] == "linear":
        k, n = c["in"], c["out"]
        weights = n * k + (n if c["bias"] else 0)
        flops = 2 * t * k * n
    else:
        k = n = c["hidden"]
        weights = 3 * k * c["inter"] + (2 * c["inter"] + k if c["bias"] else 0)
        flops = 6 * t * k * c["inter"]
    elems = t * k + weights + t * n * (2 if c["residual"] else 1)
    if c["train"]:
        elems += t * n + t * k + weights  # dy; dx and the parameters' gradients
    return {"bytes": elems * e, "flops": flops * (3 if c["train"] else 1)}


def exact(case, seed):
    """The same outputs from the definition in 64 bits, gradients by differentiation."""
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "clip":
        squares = 0.0
        for p in s["params"]:
            squares += float((p.grad.double() ** 2).sum())
        norm = math.sqrt(squares)
        coef = min(1.0, s["max_norm"] / (norm + 1e-6))
        grads = []
        for f in s["fresh"]:
            f = f.double()
            f[c["first"]:] *= coef
            grads.append(f)
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": grads}
    F = torch.nn.functional
    acts = {"none": lambda z: z, "relu": F.relu, "silu": F.silu,
            "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"),
            "era": lambda z: F.gelu(z, approximate="tanh") + GAMMA * F.softplus(z)}
    act = acts[c["act"]]
    names = [n for n in _leaves(c) if s[n] is not None]
    v = {n: s[n].detach().double().requires_grad_(c["train"]) for n in names}
    with torch.set_grad_enabled(c["train"]):
        if c["op"] == "linear":
            y = act(F.linear(v["x"], v["w"], v.get("b")))
        else:
            h = act(F.linear(v["x"], v["wg"], v.get("bg"))) * F.linear(v["x"], v["wu"], v.get("bu"))
            y = F.linear(h, v["wd"], v.get("bd"))
        if "r" in v:
            y = v["r"] + y
    if not c["train"]:
        return {"y": y}
    got = torch.autograd.grad(y, [v[n] for n in names], s["dy"].double())
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(names, got)}}
