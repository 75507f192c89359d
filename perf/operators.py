"""Measured cases of the operators around a network block and behind its backward pass.

  residual   the join behind a block: the block's output is normalised, gated and scaled, added to the residual stream, and
             the sum is normalised for the next block; forward, and forward with every gradient
  norm       the norm before the first block (over rows), forward, and forward with its gradients
  gradnorm   one norm over all gradients of a model
  clip       that norm, and the gradients scaled by min(1, max_norm / (norm + 1e-6)) into the caller's buffers

`run` evaluates the plain form in elementary torch operations; with `own` set it calls disco_amd.ops.  `exact` evaluates the
definition in float64 from explicit gradient formulas, a slice of rows at a time.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5          # of the norms
CLIP_EPS = 1e-6     # in the clipping coefficient


# ---- cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one new row through a served block (the single-token form): nothing but latency
        _residual("join, one row", 1, 4096, "bf16", "bf16", "bf16", "rms", "rms", "none", "none", True, False),
        # full-graph evaluation of a residual network: the products-shaped node count at the usual hidden width
        _residual("join, evaluation", 2449029, 256, "f32", "f32", "f32", "layer", "layer", "channel", "sigmoid", True, False),
        # training at the arxiv-shaped node count, a gate per node and channel
        _residual("join, node gates", 169343, 256, "f32", "f32", "f32", "layer", "layer", "full", "sigmoid", True, True),
        # training on a condensed graph at the Reddit-shaped feature width (rows that are only 8-byte aligned)
        _residual("join, condensed graph", 25000, 602, "f32", "f32", "f32", "rms", "rms", "row", "tanh", False, True),
        # a wide block in mixed precision: float32 stream, bfloat16 block
        _residual("join, wide mixed", 16384, 4096, "f32", "bf16", "f32", "rms", "rms", "none", "none", True, True),
        # norm of one small row: latency
        _norm("norm, one row", 1, 128, "f32", "f32", "f32", "layer", False),
        # norm of the Reddit-shaped feature matrix, trained
        _norm("norm, feature matrix", 232965, 602, "f32", "f32", "f32", "layer", True),
        # half precision at an odd width: no row but the first starts on a vector boundary
        _norm("norm, odd width", 65537, 1433, "f16", "f16", "f16", "rms", True),
        # the link predictor's ten parameters: latency
        {"name": "gradient norm, scorer", "op": "gradnorm", "layout": "scorer", "width": 256, "hidden": 256, "grad": "f32",
         "p": "2"},
        # a deep stack of blocks in float32, largest entry
        {"name": "gradient norm, stack", "op": "gradnorm", "layout": "stack", "layers": 16, "hidden": 1024, "grad": "f32", "p": "inf"},
        # the link predictor at the Reddit-shaped feature width, clipped as its training loop would
        {"name": "clip, scorer", "op": "clip", "layout": "scorer", "width": 1204, "hidden": 256, "grad": "f32", "out": "f32", "p": "2",
         "max_norm": 1.0},
        # a deep wide stack: bfloat16 gradients into the float32 buffers an optimiser reads
        {"name": "clip, wide stack", "op": "clip", "layout": "stack", "layers": 24, "hidden": 2048, "grad": "bf16", "out": "f32", "p": "2",
         "max_norm": 1.0},
    ]


def _residual(name, rows, width, stream, block, param, post, pre, gate, act, scale, train):
    c = {"op": "residual", "rows": rows, "width": width, "stream": stream, "block": block, "param": param, "post": post, "pre": pre,
         "gate": gate, "act": act, "scale": scale, "train": train}
    return {"name": name, **c} if name else c


def _norm(name, rows, width, stream, block, param, pre, train):
    c = {"op": "norm", "rows": rows, "width": width, "stream": stream, "block": block, "param": param, "pre": pre, "train": train}
    return {"name": name, **c} if name else c


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["residual", "residual", "norm", "gradnorm", "clip"])
    if op in ("residual", "norm"):
        stream, block = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
        param = rng.choice(["f32", block])
        train = rng.random() < 0.6
        width = _spread(rng, 16, 8192)    # below that a standardised row keeps few free directions and its gradient cancels
        rows = _spread(rng, 1, min(3000000, max(2, (100000000 if train else 300000000) // width)))
        pre = rng.choice(["rms", "layer"])
        if op == "norm":
            return _norm(None, rows, width, stream, block, param, pre, train)
        gate = rng.choice(["none", "full", "row", "channel"])
        act = "none" if gate == "none" else rng.choice(["none", "sigmoid", "tanh"])
        return _residual(None, rows, width, stream, block, param, rng.choice(["none", "rms", "layer"]), rng.choice([pre, pre, "none"]),
                         gate, act, rng.random() < 0.5, train)
    c = {"op": op, "layout": "ragged", "tensors": _spread(rng, 1, 600), "total": _spread(rng, 1000, 600000000),
         "mix": rng.randrange(1 << 20), "grad": rng.choice(["f32", "bf16", "f16"]), "p": rng.choice(["2", "2", "1", "inf"])}
    if op == "clip":
        c["out"] = rng.choice([c["grad"], "f32"])
        c["max_norm"] = rng.choice([0.5, 1.0, 5.0, 1e9])
    return c


def _shapes(case):
    """Shapes of a model's parameters."""
    if case["layout"] == "scorer":      # three linear layers, two batch norms
        w, h = case["width"], case["hidden"]
        return [(h, 2 * w), (h,), (h, h), (h,), (1, h), (1,), (h,), (h,), (h,), (h,)]
    if case["layout"] == "stack":       # per block: four square products, a four times wider pair, two norms
        h = case["hidden"]
        return [s for _ in range(case["layers"]) for s in ((h,), (h, h), (h, h), (h, h), (h, h), (h,), (4 * h, h), (h, 4 * h))] + [(h,)]
    r = random.Random(case["mix"])
    share = [math.exp(r.uniform(0.0, 6.0)) for _ in range(case["tensors"])]
    return [(max(1, int(case["total"] * s / sum(share))),) for s in share]


# ---- inputs -----------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 2654435761 % (1 << 62) + 17)

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] in ("gradnorm", "clip"):
        # gradients of different layers differ by orders of magnitude
        size = torch.rand(len(_shapes(case)), generator=gen, device="cuda").mul_(4.6).exp_().mul_(1e-4)
        s["grads"] = [rand(*shape).mul_(m).to(TYPES[case["grad"]]) for shape, m in zip(_shapes(case), size)]
        if case["op"] == "clip":
            flat = torch.zeros(sum(g.numel() for g in s["grads"]), dtype=TYPES[case["out"]], device="cuda")
            s["flat"] = flat
            s["out"] = [v.view(g.shape) for v, g in zip(flat.split([g.numel() for g in s["grads"]]), s["grads"])]
        return s
    n, f, train = case["rows"], case["width"], case["train"]
    stream, block, param = (TYPES[case[k]] for k in ("stream", "block", "param"))

    def leaf(t, dtype):
        return t.to(dtype).requires_grad_(train)

    s["x"] = leaf(rand(n, f).mul_(1.5).add_(0.25), stream)
    if case["pre"] != "none":
        s["pre_weight"] = leaf(rand(f).mul_(0.2).add_(1.0), param)
        if case["pre"] == "layer":
            s["pre_bias"] = leaf(rand(f).mul_(0.2), param)
    if case["op"] == "residual":
        s["y"] = leaf(rand(n, f).mul_(torch.rand(f, generator=gen, device="cuda").add_(0.5)).add_(0.1), block)
        if case["post"] != "none":
            s["post_weight"] = leaf(rand(f).mul_(0.2).add_(1.0), param)
            if case["post"] == "layer":
                s["post_bias"] = leaf(rand(f).mul_(0.2), param)
        if case["gate"] != "none":
            shape = {"full": (n, f), "row": (n, 1), "channel": (f,)}[case["gate"]]
            s["gate"] = leaf(rand(*shape), param if case["gate"] == "channel" else block)
        if case["scale"]:
            s["scale"] = leaf(torch.rand(f, generator=gen, device="cuda").add_(0.1), param)
    if train:
        if case["op"] == "residual":
            s["grad_out"] = rand(n, f).to(stream)
        if case["pre"] != "none":
            s["grad_h"] = rand(n, f).to(block)
    return s


LEAVES = ("x", "y", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if case["op"] in ("gradnorm", "clip"):
        return _own_gradients(s) if own else _plain_gradients(s)
    with torch.set_grad_enabled(case["train"]):
        out, h = _own_block(s) if own else _plain_block(s)
    got = {}
    if case["op"] == "residual":
        got["out"] = out
    if h is not None:
        got["h"] = h
    if case["train"]:
        names = [k for k in LEAVES if k in s]
        ends = [(t, s["grad_" + k]) for k, t in got.items()]
        grads = torch.autograd.grad([t for t, _ in ends], [s[k] for k in names], [g for _, g in ends])
        got.update({"d_" + k: g for k, g in zip(names, grads)})
    return got


def _own_block(s):
    from disco_amd import ops
    case = s["case"]
    if case["op"] == "norm":
        return None, ops.row_norm(s["x"], s.get("pre_weight"), s.get("pre_bias"), kind=case["pre"], eps=EPS, dtype=TYPES[case["block"]])
    r = ops.residual_norm(s["x"], s["y"], gate=s.get("gate"), gate_act=None if case["act"] == "none" else case["act"],
                          scale=s.get("scale", 0.5), post=None if case["post"] == "none" else case["post"],
                          post_weight=s.get("post_weight"), post_bias=s.get("post_bias"),
                          pre=None if case["pre"] == "none" else case["pre"], pre_weight=s.get("pre_weight"),
                          pre_bias=s.get("pre_bias"), eps=EPS)
    return (r, None) if case["pre"] == "none" else r


def _own_gradients(s):
    from disco_amd import ops
    case = s["case"]
    if case["op"] == "gradnorm":
        return {"norm": ops.grad_norm(s["grads"], norm_type=float(case["p"]))}
    norm = ops.clip_grads(s["grads"], case["max_norm"], norm_type=float(case["p"]), out=s["out"])
    return {"norm": norm, "grads": s["flat"]}


def _plain_norm(v, kind, weight, bias):
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPS) * weight.float()
    return v + bias.float() if bias is not None else v


def _plain_block(s):
    case = s["case"]
    o = s["x"].float()
    if case["op"] == "residual":
        z = s["y"].float()
        if case["post"] != "none":
            z = _plain_norm(z, case["post"], s["post_weight"], s.get("post_bias"))
        if case["gate"] != "none":
            g = s["gate"].float()
            z = z * (1.0 / (1.0 + torch.exp(-g)) if case["act"] == "sigmoid" else torch.tanh(g) if case["act"] == "tanh" else g)
        o = o + z * (s["scale"].float() if case["scale"] else 0.5)
    h = None
    if case["pre"] != "none":
        h = _plain_norm(o, case["pre"], s["pre_weight"], s.get("pre_bias")).to(TYPES[case["block"]])
    return o.to(TYPES[case["stream"]]), h


def _plain_gradients(s):
    case = s["case"]
    if case["p"] == "inf":
        norm = torch.stack([g.float().abs().max() for g in s["grads"]]).max()
    elif case["p"] == "1":
        norm = torch.stack([g.float().abs().sum() for g in s["grads"]]).sum()
    else:
        norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    if case["op"] == "gradnorm":
        return {"norm": norm}
    factor = torch.clamp(case["max_norm"] / (norm + CLIP_EPS), max=1.0)
    [o.copy_(g.float() * factor) for g, o in zip(s["grads"], s["out"])]
    return {"norm": norm, "grads": s["flat"]}


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    if case["op"] in ("gradnorm", "clip"):
        total = sum(math.prod(s) for s in _shapes(case))
        if case["op"] == "gradnorm":
            return {"bytes": total * BYTES[case["grad"]], "flops": 2 * total}
        return {"bytes": total * (BYTES[case["grad"]] + BYTES[case["out"]]), "flops": 3 * total}
    e, sx, sy = case["rows"] * case["width"], BYTES[case["stream"]], BYTES[case["block"]]
    if case["op"] == "norm":
        return {"bytes": e * (sx + sy + (sy + sx if case["train"] else 0)), "flops": e * (8 + (14 if case["train"] else 0))}
    gate = {"none": 0.0, "channel": 0.0, "row": sy / case["width"], "full": sy}[case["gate"]]
    h = sy if case["pre"] != "none" else 0
    b = sx + sy + gate + sx + h                                   # x, y, gate -> out, h
    if case["train"]:
        b += sx + h + sx + sy + gate                              # the outputs' gradients -> those of x, y, gate
    return {"bytes": e * b, "flops": e * (18 + (40 if case["train"] else 0))}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("gradnorm", "clip"):
        return _exact_gradients(case, s)
    return _exact_block(case, s)


def _exact_gradients(case, s):
    p = case["p"]
    parts = []
    for g in s["grads"]:
        for piece in g.reshape(-1).split(1 << 26):
            a = piece.double().abs()
            parts.append(float(a.max() if p == "inf" else a.sum() if p == "1" else torch.dot(a, a)))
    norm = max(parts) if p == "inf" else math.fsum(parts)
    norm = math.sqrt(norm) if p == "2" else norm
    got = {"norm": torch.tensor(norm, dtype=torch.float64)}
    if case["op"] == "clip":
        factor = min(1.0, case["max_norm"] / (norm + CLIP_EPS))
        got["grads"] = torch.cat([g.reshape(-1).double() for g in s["grads"]]).mul_(factor)
    return got


def _standard(v, kind):
    """(standardised rows, 1 / deviation) of one slice."""
    c = v - v.sum(1, keepdim=True) / v.shape[1] if kind == "layer" else v
    r = 1.0 / torch.sqrt(c.pow(2).sum(1, keepdim=True) / v.shape[1] + EPS)
    return c * r, r


def _standard_back(q, u, r, kind):
    """Gradient of the rows from that of the standardised rows `u`."""
    m = q.shape[1]
    d = q - u * ((q * u).sum(1, keepdim=True) / m)
    if kind == "layer":
        d = d - q.sum(1, keepdim=True) / m
    return r * d


def _exact_block(case, s):
    n, f, train, residual = case["rows"], case["width"], case["train"], case["op"] == "residual"
    pre, post = case["pre"], case.get("post", "none")
    with torch.no_grad():
        d = {k: s[k].double() for k in ("scale", "post_weight", "post_bias", "pre_weight", "pre_bias") if k in s}
        zero = torch.zeros(f, dtype=torch.float64, device="cuda")
        lam = d.get("scale", zero + 0.5)
        w1, b1, w2, b2 = d.get("post_weight", zero + 1), d.get("post_bias", zero), d.get("pre_weight"), d.get("pre_bias", zero)
        sums = {}
        rows = {}

        def keep(name, v):
            rows.setdefault(name, []).append(v)

        def total(name, v):
            sums[name] = sums.get(name, 0) + v.sum(0)

        def act(g):
            if case["act"] == "sigmoid":
                a = torch.sigmoid(g)
                return a, a * (1 - a)
            if case["act"] == "tanh":
                a = torch.tanh(g)
                return a, 1 - a * a
            return g, torch.ones_like(g)

        step = max(1, (1 << 26) // f)
        for at in range(0, n, step):
            to = min(n, at + step)
            o = s["x"][at:to].double()
            if residual:
                y = s["y"][at:to].double()
                u1, r1 = _standard(y, post) if post != "none" else (y, None)
                z = u1 * w1 + b1
                if case["gate"] == "none":
                    a, da = torch.ones((), dtype=torch.float64, device="cuda"), None
                else:
                    a, da = act((s["gate"] if case["gate"] == "channel" else s["gate"][at:to]).double())
                o = o + lam * a * z
                keep("out", o)
            if pre != "none":
                u2, r2 = _standard(o, pre)
                keep("h", u2 * w2 + b2)
            if not train:
                continue
            do = s["grad_out"][at:to].double() if residual else torch.zeros_like(o)
            if pre != "none":
                dh = s["grad_h"][at:to].double()
                total("d_pre_weight", dh * u2)
                total("d_pre_bias", dh)
                do = do + _standard_back(dh * w2, u2, r2, pre)
            keep("d_x", do)
            if residual:
                dz = do * lam * a
                total("d_scale", do * a * z)
                total("d_post_weight", dz * u1)
                total("d_post_bias", dz)
                if case["gate"] == "channel":
                    total("d_gate", do * lam * z * da)
                elif case["gate"] == "row":
                    keep("d_gate", (do * lam * z * da).sum(1, keepdim=True))
                elif case["gate"] == "full":
                    keep("d_gate", do * lam * z * da)
                keep("d_y", _standard_back(dz * w1, u1, r1, post) if post != "none" else dz)
        got = {k: v[0] if len(v) == 1 else torch.cat(v) for k, v in rows.items()}
        got.update({k: v for k, v in sums.items() if k[2:] in s})
    return got
