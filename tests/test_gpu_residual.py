"""The residual join and the row norm against their formulas in float64, forward and every gradient.

Tolerances (u = 2^-24, the float32 half step).  A row's statistics are trees of at most 16 + 6 + 16 additions; each value
then passes a handful of roundings, so a standardised value u2 = (v - mean) * rstd is off by at most about
50 u * (|u2| + rstd * (mean |v| + |v's terms|)), and a gradient that passes one such norm by the same factor of its terms'
magnitudes, twice where it passes both.  C = 256 covers both norms; every bound below is C u times the magnitudes the
formula adds up (no cancellation is assumed), plus half a step of the output's own type."""
import itertools

import numpy as np
import pytest
import torch

from disco_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
C = 256 * U
EPS = 1e-5
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LEAVES = ("x", "y", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")


def make(n, F, stream="f32", block="f32", param="f32", post="layer", pre="layer", gate="full", act="sigmoid", scale="vector", bias=True,
         seed=0, mean=0.25):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + n * 31 + F)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    s = dict(post=post, pre=pre, gate_kind=gate, act=act if gate else None, const=0.5 if scale != "vector" else 1.0)
    t = {"x": (r(n, F) * 1.5 + mean).to(T[stream])}
    if block is not None:
        t["y"] = (r(n, F) * 0.8 + 0.1).to(T[block])
    if gate:
        t["gate"] = {"full": r(n, F), "row": r(n, 1), "channel": r(F)}[gate].to(T[param] if gate == "channel" else T[block])
    if scale == "vector":
        t["scale"] = (r(F) * 0.3 + 0.6).to(T[param])
    for k, kind in (("post", post), ("pre", pre)):
        if kind:
            t[k + "_weight"] = (r(F) * 0.2 + 1).to(T[param])
            if bias:
                t[k + "_bias"] = (r(F) * 0.2).to(T[param])
    s["t"] = t
    s["dout"], s["dh"] = r(n, F).to(T[stream]), (r(n, F).to(T[block]) if pre else None)
    return s


def call(s, t=None):
    t = s["t"] if t is None else t
    r = ops.residual_norm(t["x"], t["y"], gate=t.get("gate"), gate_act=s["act"], scale=t.get("scale", s["const"]), post=s["post"],
                          post_weight=t.get("post_weight"), post_bias=t.get("post_bias"), pre=s["pre"], pre_weight=t.get("pre_weight"),
                          pre_bias=t.get("pre_bias"), eps=EPS)
    return r if s["pre"] else (r, None)


def train(s, use=("out", "h")):
    t = {k: v.detach().clone(memory_format=torch.preserve_format).requires_grad_() for k, v in s["t"].items()}
    out, h = call(s, t)
    ends = [(o, g) for name, o, g in (("out", out, s["dout"]), ("h", h, s["dh"])) if o is not None and name in use]
    grads = torch.autograd.grad([o for o, _ in ends], list(t.values()), [g for _, g in ends], allow_unused=True)
    return out.detach(), None if h is None else h.detach(), dict(zip(t, grads))


def norm64(v, kind):
    c = v - v.mean(1, keepdim=True) if kind == "layer" else v
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    return c * r, r


def back64(q, u, r, kind):
    return r * (q - (q.mean(1, keepdim=True) if kind == "layer" else 0) - u * (q * u).mean(1, keepdim=True))


def act64(g, act):
    a = torch.sigmoid(g) if act == "sigmoid" else torch.tanh(g) if act == "tanh" else g
    return a, a * (1 - a) if act == "sigmoid" else 1 - a * a if act == "tanh" else torch.ones_like(a)


def formula(s, use=("out", "h")):
    """{name: (value, magnitude of what it is added up from)} in float64."""
    t = {k: v.double() for k, v in s["t"].items()}
    x, y = t["x"], t["y"]
    one, zero = torch.ones(x.shape[1], dtype=torch.float64, device=DEV), torch.zeros(x.shape[1], dtype=torch.float64, device=DEV)
    lam = t.get("scale", one * s["const"])
    w1, b1, w2, b2 = t.get("post_weight", one), t.get("post_bias", zero), t.get("pre_weight", one), t.get("pre_bias", zero)
    u1, r1 = norm64(y, s["post"]) if s["post"] else (y, torch.ones_like(y[:, :1]))
    S1 = u1.abs() + (r1 * (y.abs() + y.abs().mean(1, keepdim=True)) if s["post"] else 0)
    z = u1 * w1 + b1
    Z = S1 * w1.abs() + b1.abs()
    if "gate" in t:
        a, da = act64(t["gate"], s["act"])
    else:
        a, da = torch.ones((), dtype=torch.float64, device=DEV), None
    al = (a * lam).abs()
    out = x + a * lam * z
    M = x.abs() + al * Z                                  # magnitude of the sum's terms
    got = {"out": (out, M)}
    do = s["dout"].double() if "out" in use else torch.zeros_like(x)
    D = do.abs()
    if s["pre"]:
        u2, r2 = norm64(out, s["pre"])
        S2 = u2.abs() + r2 * (M + M.mean(1, keepdim=True))
        got["h"] = (u2 * w2 + b2, S2 * w2.abs() + b2.abs())
        if "h" in use:
            dh = s["dh"].double()
            q = dh * w2
            Q = q.abs()
            got["pre_weight"] = ((dh * u2).sum(0), (dh.abs() * S2).sum(0))
            got["pre_bias"] = (dh.sum(0), dh.abs().sum(0))
            do = do + back64(q, u2, r2, s["pre"])
            D = D + r2 * (Q + Q.mean(1, keepdim=True) + S2 * (Q * S2).mean(1, keepdim=True))
    got["x"] = (do, D)
    dz, DZ = do * a * lam, D * al
    got["scale"] = ((do * a * z).sum(0), (D * a.abs() * Z).sum(0))
    got["post_weight"] = ((dz * u1).sum(0), (DZ * S1).sum(0))
    got["post_bias"] = (dz.sum(0), DZ.sum(0))
    if "gate" in t:
        v, m = do * lam * z * da, D * lam.abs() * Z
        got["gate"] = (v, m) if s["gate_kind"] == "full" else (v.sum(1, keepdim=True), m.sum(1, keepdim=True)) if s["gate_kind"] == "row" else \
            (v.sum(0), m.sum(0))
    if s["post"]:
        p, P = dz * w1, DZ * w1.abs()
        got["y"] = (back64(p, u1, r1, s["post"]), r1 * (P + P.mean(1, keepdim=True) + S1 * (P * S1).mean(1, keepdim=True)))
    else:
        got["y"] = (dz, DZ)
    return got


def near(got, want, what):
    v, m = want
    assert got is not None and got.shape == v.shape, what
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    err, lim = (got.double() - v).abs(), C * m + half * v.abs() * (1 + C) + tiny
    bad = ~(err <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / lim).nan_to_num(nan=1e30).max()):.3g} x the bound"


def check(s, use=("out", "h"), what=""):
    want = formula(s, use)
    out, h = call(s)
    near(out, want["out"], what + " out")
    if s["pre"]:
        near(h, want["h"], what + " h")
    o2, h2, grads = train(s, use)
    assert torch.equal(out, o2) and (h is None or torch.equal(h, h2)), "the training forward differs from the plain one"
    assert out.dtype == s["t"]["x"].dtype and (h is None or h.dtype == s["t"]["y"].dtype)
    for k, g in grads.items():
        if k.startswith("pre") and "h" not in use:
            assert g is None
            continue
        assert g.dtype == s["t"][k].dtype, k
        near(g, want[k], f"{what} d_{k}")
    return grads


WIDTHS = [1, 2, 3, 4, 5, 7, 8, 15, 16, 17, 31, 32, 33, 41, 63, 64, 65, 100, 128, 129, 256, 257, 512, 513, 602, 768, 769, 1024, 1025, 1433, 2048, 2049, 4096, 4097, 8192,
          8193, 16383, 16384]


@pytest.mark.parametrize("F", WIDTHS)
def test_widths(F):
    check(make(7, F), what=f"F={F}")
    check(make(7, F, "f32", "bf16", "f32", "rms", "rms", "row", "tanh", "number"), what=f"F={F} mixed")


@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 17, 255, 257, 1000, 4097])
@pytest.mark.parametrize("F", [24, 602])
def test_rows(n, F):
    check(make(n, F), what=f"n={n} F={F}")


@pytest.mark.parametrize("post,pre,gate,act", [c for c in itertools.product((None, "rms", "layer"), (None, "rms", "layer"),
                                                                            (None, "full", "row", "channel"), (None, "sigmoid", "tanh"))
                                               if c[2] or not c[3]])
def test_norms_and_gates(post, pre, gate, act):
    check(make(33, 130, post=post, pre=pre, gate=gate, act=act, seed=3))
    check(make(9, 1300, post=post, pre=pre, gate=gate, act=act, scale="number", bias=False, seed=4))


@pytest.mark.parametrize("stream,block", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("param", ["f32", "block"])
@pytest.mark.parametrize("F", [96, 301, 1000, 2500, 5001])
def test_types(stream, block, param, F):
    check(make(21, F, stream, block, block if param == "block" else param, seed=5), what=f"{stream}/{block}")
    check(make(20, F, stream, block, "f32", "rms", "rms", None, None, seed=6), what=f"{stream}/{block} ungated")


@pytest.mark.parametrize("use", [("out",), ("h",)])
@pytest.mark.parametrize("post,gate", [("layer", "full"), (None, "row"), ("rms", "channel")])
def test_one_output_used(use, post, gate):
    check(make(40, 70, post=post, gate=gate, seed=8), use)
    check(make(40, 2100, post=post, gate=gate, seed=8), use)


def test_no_output_used_by_a_leaf_that_needs_none():
    s = make(12, 50)
    t = dict(s["t"])
    for needs in (("x",), ("y",), ("gate",), ("pre_weight",), ("scale", "post_bias"), ("y", "post_weight")):
        u = {k: v.clone().requires_grad_(k in needs) for k, v in t.items()}
        out, h = call(s, u)
        got = torch.autograd.grad([out, h], [u[k] for k in needs], [s["dout"], s["dh"]])
        want = formula(s)
        for k, g in zip(needs, got):
            near(g, want[k], f"{needs} d_{k}")


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("stream,block", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("n,F", [(1, 128), (5, 1), (300, 41), (17, 602), (3, 4099)])
def test_row_norm(kind, stream, block, n, F):
    s = make(n, F, stream, block, post=None, pre=kind, gate=None, scale="number", seed=11)
    s["t"]["y"] = torch.zeros_like(s["t"]["y"])
    want = formula(s, ("h",))
    x, w, b = (s["t"][k].clone().requires_grad_() for k in ("x", "pre_weight", "pre_bias"))
    h = ops.row_norm(x, w, b, kind=kind, eps=EPS, dtype=T[block])
    near(h, want["h"], "h")
    assert torch.equal(h, ops.row_norm(x.detach(), w.detach(), b.detach(), kind, EPS, T[block]))
    for k, g in zip(("x", "pre_weight", "pre_bias"), torch.autograd.grad(h, (x, w, b), s["dh"])):
        near(g, want[k], "d_" + k)
    del s["t"]["pre_weight"], s["t"]["pre_bias"]
    near(ops.row_norm(x.detach(), kind=kind, eps=EPS, dtype=T[block]), formula(s, ("h",))["h"], "without weights")


def test_gradients_against_differences():
    """The kernel's gradient against central differences of the formula itself, along random directions (float64: the
    difference is exact to about step^2 and 1e-16 / step of the values)."""
    for post, pre, gate, act in (("layer", "rms", "full", "sigmoid"), ("rms", "layer", "row", "tanh"), (None, "layer", "channel", None)):
        s = make(6, 37, post=post, pre=pre, gate=gate, act=act, seed=21)
        _, _, grads = train(s)
        g = torch.Generator(device=DEV).manual_seed(5)

        def loss(t):
            f = formula({**s, "t": t}, ())
            return float((f["out"][0] * s["dout"].double()).sum() + (f["h"][0] * s["dh"].double()).sum())

        for k, v in s["t"].items():
            d = torch.randn(v.shape, generator=g, device=DEV, dtype=torch.float64)
            step = 1e-5
            t = {**{q: w.double() for q, w in s["t"].items()}}
            plus, minus = loss({**t, k: t[k] + step * d}), loss({**t, k: t[k] - step * d})
            want, got = (plus - minus) / (2 * step), float((grads[k].double() * d).sum())
            size = float((grads[k].double().abs() * d.abs()).sum())
            assert abs(got - want) <= 1e-6 * size + 1e-8 * (1 + abs(plus)), (k, got, want)


def view_of(v, how):
    n, F = v.shape
    if how == "columns":          # a column slice: rows far apart, starting at any element
        buf = torch.full((n, 2 * F + 3), float("nan"), dtype=v.dtype, device=DEV)
        w = buf[:, 3:3 + F]
    elif how == "rows":           # every other row
        buf = torch.full((2 * n, F), float("nan"), dtype=v.dtype, device=DEV)
        w = buf[::2]
    elif how == "transposed":
        buf = torch.empty(F, n, dtype=v.dtype, device=DEV)
        w = buf.t()
    else:                         # a start that is aligned to the element only
        buf = torch.full((n * F + 1,), float("nan"), dtype=v.dtype, device=DEV)
        w = buf[1:].view(n, F)
    w.copy_(v)
    return w


@pytest.mark.parametrize("how", ["columns", "rows", "transposed", "shifted"])
@pytest.mark.parametrize("F,block", [(50, "f32"), (128, "bf16"), (602, "f16"), (1031, "f32")])
def test_layouts(how, F, block):
    s = make(19, F, "f32", block, block, seed=31)
    want = train(s)
    v = {**s, "t": {k: view_of(t, how) if t.dim() == 2 else view_of(t[None], "shifted")[0] for k, t in s["t"].items()}}
    v["dout"], v["dh"] = view_of(s["dout"], how), view_of(s["dh"], how)
    t = {k: w.detach().requires_grad_() for k, w in v["t"].items()}
    out, h = call(s, t)
    grads = torch.autograd.grad([out, h], list(t.values()), [v["dout"], v["dh"]])
    assert torch.equal(out, want[0]) and torch.equal(h, want[1])
    for k, g in zip(t, grads):
        assert torch.equal(g, want[2][k]), k


def test_broadcast_operands():
    """Expanded rows, gates and gradients: read as they are, their gradients summed by autograd over what was repeated."""
    s = make(30, 64, gate="row", seed=41)
    s["dout"], s["dh"] = torch.ones(1, device=DEV).expand(30, 64), torch.full((1, 64), 0.5, device=DEV).expand(30, 64)
    s["t"]["x"] = s["t"]["x"][:1].expand(30, 64)
    s["t"]["gate"] = s["t"]["gate"][:1].expand(30, 1)
    want = formula(s)
    x1, g1 = s["t"]["x"][:1].clone().requires_grad_(), s["t"]["gate"][:1].clone().requires_grad_()
    t = {k: v.clone().requires_grad_() for k, v in s["t"].items() if k not in ("x", "gate")}
    out, h = call(s, {**t, "x": x1.expand(30, 64), "gate": g1.expand(30, 1)})
    near(out, want["out"], "out")
    near(h, want["h"], "h")
    gx, gg, gy = torch.autograd.grad([out, h], [x1, g1, t["y"]], [s["dout"], s["dh"]])
    near(gx, tuple(v.sum(0, keepdim=True) for v in want["x"]), "d_x")
    near(gg, tuple(v.sum(0, keepdim=True) for v in want["gate"]), "d_gate")
    near(gy, want["y"], "d_y")
    # a gate that is one column of a wider matrix, and one row of gates for all rows
    wide = torch.randn(30, 7, device=DEV)
    s["t"]["gate"] = wide[:, 3:4]
    near(call(s)[0], formula(s)["out"], "gate column")
    got = train(s)[2]["gate"]
    near(got, formula(s)["gate"], "d_gate column")
    s["gate_kind"] = "full"
    s["t"]["gate"] = torch.randn(1, 64, device=DEV).expand(30, 64)
    check(s, what="repeated gates")
    # one scalar scale for all channels
    a = torch.full((), 0.7, device=DEV, requires_grad=True)
    out = ops.residual_norm(s["t"]["x"], s["t"]["y"], scale=a.expand(64))
    (ga,) = torch.autograd.grad(out, a, torch.ones_like(out))
    ref = s["t"]["y"].double()
    assert abs(float(ga) - float(ref.sum())) <= C * float(ref.abs().sum())


def test_a_gradient_with_one_repeated_row():
    """Without a pre norm the stream's gradient is the given one, which may be a single row for all (stride 0)."""
    for gate in (None, "row", "full"):
        s = make(21, 40, pre=None, gate=gate, act="tanh", seed=44)
        s["dout"] = torch.randn(1, 40, device=DEV).expand(21, 40)
        check(s, ("out",))
    x, y = (torch.randn(9, 24, device=DEV, requires_grad=True) for _ in range(2))
    ops.residual_norm(x, y, post="rms").sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x))
    ops.residual_norm(x.detach().requires_grad_(), y.detach()).sum().backward()      # nothing to compute


def test_mixed_parameter_types_meet_in_float32():
    s = make(11, 40, "f32", "bf16", "f32", seed=43)
    s["t"]["post_weight"], s["t"]["pre_bias"] = s["t"]["post_weight"].bfloat16(), s["t"]["pre_bias"].half()
    check(s)


def test_empty_and_constant_rows():
    x0, w0 = torch.empty(0, 5, device=DEV, requires_grad=True), torch.ones(5, device=DEV, requires_grad=True)
    gx, gw = torch.autograd.grad(ops.row_norm(x0, w0).sum(), (x0, w0))
    assert gx.shape == (0, 5) and torch.equal(gw, torch.zeros(5, device=DEV))
    s = make(0, 33)
    out, h, grads = train(s)
    assert out.shape == (0, 33) and h.shape == (0, 33) and grads["x"].shape == (0, 33) and grads["gate"].shape == (0, 33)
    for k in ("scale", "post_weight", "post_bias", "pre_weight", "pre_bias"):
        assert torch.equal(grads[k], torch.zeros(33, device=DEV)), k
    # rows of one value, of zeros, of large values: the variance is zero or its mean dominates
    s = make(6, 100, gate=None, act=None, seed=3)
    s["t"]["y"][0], s["t"]["y"][1], s["t"]["y"][2] = 0.0, 3.25, -1e4
    s["t"]["x"][3] = 0.0
    s["t"]["x"][4] += 1000.0
    check(s)
    # magnitudes whose squares stay inside float32
    s = make(5, 64, post="rms", pre="rms", gate=None, act=None)
    s["t"]["y"][0] *= 1e15
    s["t"]["x"][1] *= 1e15
    s["t"]["y"][2] *= 1e-15
    check(s)


@pytest.mark.parametrize("stream,block", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("F", [96, 3, 50, 1200])
def test_nan_and_inf_stay_in_their_rows(stream, block, F):
    s = make(40, F, stream, block, seed=51)
    clean = train(s)
    s["t"]["y"][3, F // 2], s["t"]["x"][7, F - 1], s["t"]["gate"][11, 0] = float("nan"), float("inf"), float("nan")
    out, h, grads = train(s)
    rest = [i for i in range(40) if i not in (3, 7, 11)]
    for a, b in ((out, clean[0]), (h, clean[1]), (grads["x"], clean[2]["x"]), (grads["y"], clean[2]["y"]), (grads["gate"], clean[2]["gate"])):
        assert torch.equal(a[rest], b[rest])
    assert out[3].isnan().all() and h[3].isnan().all() and out[7, F - 1] == float("inf") and h[7].isnan().any()
    assert out[11, 0].isnan() and torch.equal(out[11, 1:], clean[0][11, 1:]) and h[11].isnan().all()
    assert grads["pre_weight"].isnan().all()
    # a gate of plus / minus infinity is an open / closed gate
    s = make(4, 30, gate="full", act="sigmoid", pre=None)
    s["t"]["gate"][0], s["t"]["gate"][1] = float("inf"), float("-inf")
    out, _, grads = train(s)
    assert torch.equal(out[1], s["t"]["x"][1]) and out.isfinite().all() and all(g.isfinite().all() for g in grads.values())
    assert not grads["y"][1].any() and not grads["gate"][:2].any()


def test_rows_behind_the_result_and_columns_beside_it_are_left():
    """Outputs at a leading dimension: the C entry writes the rows and columns it is given and nothing else."""
    from disco_amd import _lib
    lib = _lib.load()
    for n, F, ld in ((5, 7, 11), (3, 602, 610), (2, 4097, 4100)):
        x, y = torch.randn(n, F, device=DEV), torch.randn(n, F, device=DEV)
        out, h = (torch.full((n + 2, ld), 7.0, device=DEV) for _ in range(2))
        d = _lib.ResidualNorm(rows=n, width=F, ldx=F, ldy=F, x=x.data_ptr(), y=y.data_ptr(), has_block=1, post_norm=1, pre_norm=2, scale=1.0, eps=EPS)
        _lib.check(lib.disco_residual_norm_forward(d, out.data_ptr(), ld, h.data_ptr(), ld, None, _lib.current_stream(x.device)), "forward")
        ref = ops.residual_norm(x, y, post="rms", pre="layer", eps=EPS)
        for got, want in zip((out, h), ref):
            assert torch.equal(got[:n, :F], want)
            assert (got[n:] == 7).all() and (got[:, F:] == 7).all()


def test_two_runs_and_two_streams_give_the_same_bits():
    s = make(5000, 200, seed=61)
    first = train(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = train(s)
    third = train(s)
    torch.cuda.current_stream().wait_stream(side)
    for other in (second, third):
        assert torch.equal(first[0], other[0]) and torch.equal(first[1], other[1])
        for k in first[2]:
            assert torch.equal(first[2][k], other[2][k]), k


def test_captured_training_step_replays():
    """Forward and backward captured into a graph, replayed on new inputs with eager work in between."""
    s = make(300, 90, seed=71)
    t = {k: v.clone().requires_grad_() for k, v in s["t"].items()}

    def step():
        out, h = call(s, t)
        return (out, h) + torch.autograd.grad([out, h], list(t.values()), [s["dout"], s["dh"]])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        with torch.no_grad():
            for k, v in t.items():
                v.copy_(torch.randn(v.shape, device=DEV) * 0.5 + 0.5)
        want = [w.clone() for w in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b), i


def test_backward_from_another_stream_and_thread():
    """A node runs on its forward's stream, whichever one its caller is on; calls from two threads do not disturb each other."""
    import threading
    s = make(3000, 120, seed=72)
    want = train(s)
    side = torch.cuda.Stream()
    t = {k: v.clone().requires_grad_() for k, v in s["t"].items()}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, h = call(s, t)
    torch.cuda.current_stream().wait_stream(side)
    for k, g in zip(t, torch.autograd.grad([out, h], list(t.values()), [s["dout"], s["dh"]])):
        assert torch.equal(g, want[2][k]), k
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            for _ in range(5):
                got[i] = train(s)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [w.start() for w in threads]
    [w.join() for w in threads]
    for r in got:
        assert torch.equal(r[0], want[0]) and torch.equal(r[1], want[1]) and all(torch.equal(r[2][k], want[2][k]) for k in want[2])


def test_what_autograd_keeps():
    """Operands changed in between are noticed, kept ones may move to the host and back, one tensor may be several operands."""
    s = make(20, 30)
    t = {k: v.clone().requires_grad_() for k, v in s["t"].items()}
    z = t["y"] * 1.0
    out, h = call(s, {**t, "y": z})
    z.detach().add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        out.sum().backward()
    want = train(s)
    with torch.autograd.graph.save_on_cpu():
        got = train(s)
    assert all(torch.equal(got[2][k], want[2][k]) for k in want[2])
    with torch.inference_mode():
        out, h = call(s)
    assert torch.equal(out, want[0]) and torch.equal(h, want[1])
    x, w = torch.randn(9, 16, device=DEV, requires_grad=True), torch.randn(16, device=DEV, requires_grad=True)
    out = ops.residual_norm(x, x, gate=x, post="rms", post_weight=w, scale=w)
    gx, gw = torch.autograd.grad(out.sum(), (x, w))
    X, W = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    u = X * torch.rsqrt((X * X).mean(1, keepdim=True) + EPS)
    for a, b in zip((gx, gw), torch.autograd.grad((X + W * X * u * W).sum(), (X, W))):
        assert ((a.double() - b).abs() <= C * (1 + b.abs().max())).all()


@pytest.mark.parametrize("gate", [None, "row", "full"])
def test_the_stream_may_change_where_no_norm_reads_it(gate):
    s = make(20, 30, pre=None, gate=gate, act=gate and "sigmoid")
    want = train(s, ("out",))
    t = {k: v.clone().requires_grad_() for k, v in s["t"].items()}
    x = t["x"] * 1.0
    out = call(s, {**t, "x": x})
    out = out[0] if isinstance(out, tuple) else out
    x.detach().add_(1.0)
    got = torch.autograd.grad((out * s["dout"]).sum(), list(t.values()))
    for k, g in zip(t, got):
        assert torch.equal(g, want[2][k]), k
    x = t["x"] * 1.0
    out, h = call(make(20, 30), {**make(20, 30)["t"], "x": x})
    x.detach().add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        (out.sum() + h.sum()).backward()


def test_second_derivatives_are_refused():
    s = make(4, 16, gate=None, act=None)
    t = {k: v.clone().requires_grad_() for k, v in s["t"].items()}
    out, h = call(s, t)
    (g,) = torch.autograd.grad(out.sum() + h.square().sum(), t["x"], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), t["x"])


def test_many_rows_pass_32_bit_offsets():
    """Rows behind 2^32 elements: offsets are 64 bits wide (fp16, one column more than four)."""
    n, F = 2 ** 30 + 5, 5
    x = torch.zeros(n, F, dtype=torch.float16, device=DEV)
    x[-3:] = torch.randn(3, F, device=DEV).half()
    h = ops.row_norm(x, kind="rms", eps=EPS)
    want = x[-3:].double() * torch.rsqrt(x[-3:].double().square().mean(1, keepdim=True) + EPS)
    assert ((h[-3:].double() - want).abs() <= 2.0 ** -11 * want.abs() * (1 + C) + C * want.abs() + 2.0 ** -24).all()
    assert not h[:1000].any() and not h[n // 2:n // 2 + 1000].any()
    del h
    x.requires_grad_()
    w = torch.ones(F, device=DEV, requires_grad=True)
    h = ops.row_norm(x, w, kind="rms", eps=EPS)
    g = torch.zeros(n, F, dtype=torch.float16, device=DEV)
    g[-2:] = 1.0
    dx, dw = torch.autograd.grad(h, (x, w), g)
    v = x.detach()[-2:].double().requires_grad_()
    u = v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS)
    (ref,) = torch.autograd.grad(u.sum(), v)
    size = torch.rsqrt(v.detach().square().mean(1, keepdim=True) + EPS)
    assert ((dx[-2:].double() - ref).abs() <= 2.0 ** -11 * ref.abs() * (1 + C) + C * F * size + 2.0 ** -24).all()
    assert not dx[:1000].any() and not dx[-1000:-2].any()
    assert ((dw.double() - u.detach().sum(0)).abs() <= C * u.detach().abs().sum(0)).all()


@pytest.mark.parametrize("case", range(40))
def test_drawn_cases(case):
    r = np.random.default_rng(1000 + case)
    stream, block = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")][r.integers(5)]
    F = int(np.exp(r.uniform(np.log(2), np.log(9000))))
    n = int(np.exp(r.uniform(0, np.log(max(2, 400000 // F)))))
    gate = [None, "full", "row", "channel"][r.integers(4)]
    s = make(n, F, stream, block, ["f32", block][r.integers(2)], [None, "rms", "layer"][r.integers(3)], [None, "rms", "layer"][r.integers(3)],
             gate, [None, "sigmoid", "tanh"][r.integers(3)], ["vector", "number"][r.integers(2)], bool(r.integers(2)), seed=case)
    check(s, what=f"{case}: n={n} F={F} {stream}/{block}")


@pytest.mark.parametrize("n,F,ld", [(1, 1, 1), (5, 7, 11), (300, 602, 610), (70000, 3, 4)])
@pytest.mark.parametrize("stream,block", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
def test_the_norm_without_a_gradient_has_zero_gradients(n, F, ld, stream, block):
    """C entry, norm alone, dh NULL ("NULL: zero"): x, the statistics and the workspace are not there, and nothing is read."""
    from disco_amd import _lib
    lib = _lib.load()
    dx = torch.full((n + 1, ld), 7.0, dtype=T[stream], device=DEV)
    w, dw, db = (torch.full((F,), 7.0, device=DEV) for _ in range(3))
    d = _lib.ResidualNorm(rows=n, width=F, ldx=F, has_block=0, pre_norm=2, pre_weight=w.data_ptr(), pre_bias=w.data_ptr(), scale=1.0, eps=EPS,
                          stream_type=_lib.DTYPES[T[stream]], block_type=_lib.DTYPES[T[block]])
    g = _lib.ResidualNormGrads(dx=dx.data_ptr(), ld_dx=ld, dpre_weight=dw.data_ptr(), dpre_bias=db.data_ptr())
    _lib.check(lib.disco_residual_norm_backward(d, None, g, None, 0, _lib.current_stream(dx.device)), "backward")
    assert not dx[:n, :F].any() and (dx[n:] == 7).all() and (dx[:, F:] == 7).all() and not dw.any() and not db.any()


def test_a_traced_call_runs_on_the_stream_of_its_caller():
    """Traced on one stream, called on another behind work that is still running there: it waits for that work."""
    x, w = torch.zeros(64, 48, device=DEV), torch.randn(48, device=DEV)
    new = torch.randn(64, 48, device=DEV)
    f = torch.jit.trace(lambda v: ops.row_norm(v, w) + ops.residual_norm(v, v, post="rms"), x)
    want = ops.row_norm(new, w) + ops.residual_norm(new, new, post="rms")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        x.copy_(new)
        got = f(x)
    side.synchronize()
    assert torch.equal(got, want)


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwad
    x, w = torch.randn(4, 8, device=DEV), torch.randn(8, device=DEV)
    with fwad.dual_level():
        d, dw = fwad.make_dual(x, torch.ones_like(x)), fwad.make_dual(w, torch.ones_like(w))
        for call in (lambda: ops.row_norm(d), lambda: ops.row_norm(x, dw), lambda: ops.residual_norm(x, d), lambda: ops.residual_norm(x, x, gate=dw),
                     lambda: ops.residual_norm(x, x, gate=d[:, :1]), lambda: ops.residual_norm(x, x, scale=dw.half()), lambda: ops.grad_norm([x, d]),
                     lambda: ops.grad_norm(d[:, ::2]), lambda: ops.clip_grads([x], 1.0, out=[d])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    ops.row_norm(d), ops.row_norm(x, dw)      # outside of the level they are ordinary tensors


@pytest.mark.parametrize("gate,pre", [("full", "layer"), ("row", "rms"), (None, None)])
def test_a_recorded_graph_computes_the_same(gate, pre):
    """make_fx records forward and backward; the graph gives the eager results, on other inputs too."""
    from torch.fx.experimental.proxy_tensor import make_fx
    s = make(20, 30, gate=gate, pre=pre, seed=81)
    names = list(s["t"])

    def step(*leaves):
        out, h = call(s, dict(zip(names, leaves)))
        return (out,) + (() if h is None else (h,)) + torch.autograd.grad([out] if h is None else [out, h], leaves,
                                                                          [s["dout"]] if h is None else [s["dout"], s["dh"]])

    leaves = [t.clone().requires_grad_() for t in s["t"].values()]
    graph = make_fx(step)(*leaves)
    targets = {n.target for n in graph.graph.nodes}
    assert {torch.ops.disco_amd.residual_norm_forward.default, torch.ops.disco_amd.residual_norm_backward.default} <= targets
    other = [torch.randn_like(t).requires_grad_() for t in leaves]
    for a, b in zip(graph(*other), step(*other)):
        assert torch.equal(a, b)


def test_the_operators_pass_the_dispatchers_checks():
    s = make(6, 20, "f32", "bf16", seed=82)
    t = s["t"]
    args = (t["x"], t["y"], t["gate"], t["scale"], t["post_weight"], t["post_bias"], t["pre_weight"], t["pre_bias"])
    plan = 2 | 2 << 2 | 1 << 4 | 1 << 6 | 2 << 8 | 1 << 12
    D = torch.ops.disco_amd
    forward = (*args, plan, 1.0, EPS, True)
    out, h, stats = D.residual_norm_forward(*forward)
    want = call(s)
    assert torch.equal(out, want[0]) and torch.equal(h, want[1]) and stats.shape == (24,)
    backward = (s["dout"], s["dh"], stats, *args, plan, 1.0, EPS, 255)
    for a, b in zip(D.residual_norm_backward(*backward), train(s)[2].values()):
        assert torch.equal(a, b)
    grads = [torch.randn(50, device=DEV), torch.randn(7, 3, device=DEV)]
    for op, a in ((D.residual_norm_forward, forward), (D.residual_norm_backward, backward), (D.grad_norm, (grads, 2)),
                  (D.grad_clip, (grads, [torch.empty_like(g) for g in grads], 2, 0.5))):
        torch.library.opcheck(op.default, a, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_a_compiled_function_computes_the_same(backend):
    s = make(20, 30, seed=83)
    names = list(s["t"])

    def f(*leaves):
        out, h = call(s, dict(zip(names, leaves)))
        return out * s["dout"], h * s["dh"]

    def step(g):
        leaves = [t.clone().requires_grad_() for t in s["t"].values()]
        return torch.autograd.grad([v.sum() for v in g(*leaves)], leaves)

    try:
        for a, b in zip(step(torch.compile(f, backend=backend)), step(f)):
            assert torch.equal(a, b)
        p, q = s["t"]["x"].clone(), s["t"]["x"].clone()
        assert torch.equal(torch.compile(lambda t: ops.clip_grads([t], 0.5), backend=backend)(p), ops.clip_grads([q], 0.5)) and torch.equal(p, q)
    finally:
        torch._dynamo.reset()


def test_lazily_negated_operands():
    """The imaginary part of a conjugate is negated when it is read: a row gate and a single column are passed as they lie."""
    z = torch.randn(30, 1, device=DEV, dtype=torch.complex64)
    v = z.conj().imag
    assert v.is_neg()
    s = make(30, 16, gate="row", seed=91)
    s["t"]["gate"] = v.clone()
    want = train(s)
    s["t"]["gate"] = v
    for a, b in zip(call(s), want):
        assert torch.equal(a, b)
    g = {k: t.requires_grad_() for k, t in s["t"].items() if k != "gate"}
    out, h = call(s, {**g, "gate": z.requires_grad_().conj().imag})
    got = torch.autograd.grad([out, h], list(g.values()) + [z], [s["dout"], s["dh"]])
    for k, d in zip(g, got):
        assert torch.equal(d, want[2][k]), k
    assert torch.equal(got[-1].imag, -want[2]["gate"]) and not got[-1].real.any()
    one = make(30, 1, gate=None, act=None, seed=92)
    one["t"]["x"] = v.clone()
    want = call(one)
    one["t"]["x"] = v.detach()
    for a, b in zip(call(one), want):
        assert torch.equal(a, b)
    n = torch._neg_view(torch.randn(7, 12, device=DEV))
    assert torch.equal(ops.row_norm(n), ops.row_norm(n.clone()))
    x = torch.randn(7, 12, device=DEV, requires_grad=True)
    up = torch.randn(7, 12, device=DEV)
    for a, b in zip(torch.autograd.grad(ops.row_norm(x), x, torch._neg_view(up)), torch.autograd.grad(ops.row_norm(x), x, -up)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("stream,block", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("n,F", [(1, 1), (20, 30), (3, 4099), (40, 3), (2, 16384)])
def test_the_blocks_output_may_change_where_no_gradient_reads_it(stream, block, n, F):
    """out = x + factor * y: neither x nor y is kept."""
    x, y = (torch.randn(n, F, device=DEV).to(T[k]).requires_grad_() for k in (stream, block))
    up = torch.randn(n, F, device=DEV).to(T[stream])
    a, b = x * 1.0, y * 1.0
    out = ops.residual_norm(a, b, scale=0.3)
    a.detach().fill_(float("nan"))
    b.detach().fill_(float("nan"))
    gx, gy = torch.autograd.grad(out, (x, y), up, retain_graph=True)
    assert torch.equal(gx, up) and gy.dtype == T[block] and torch.equal(gy, (up.float() * 0.3).to(T[block]))
    (gy,) = torch.autograd.grad(out, (y,), torch.full((1, 1), float("nan"), device=DEV, dtype=T[stream]).expand(n, F))
    assert gy.isnan().all()
    for kw in (dict(post="rms"), dict(gate=torch.ones(F, device=DEV)), dict(scale=torch.ones(F, device=DEV)), dict(pre="rms")):
        b = y * 1.0
        out = ops.residual_norm(x, b, **kw)
        b.detach().add_(1.0)
        with pytest.raises(RuntimeError, match="modified"):
            sum(o.sum() for o in (out if isinstance(out, tuple) else (out,))).backward()


@pytest.mark.parametrize("stream,block", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("gate", ["full", "row", "channel"])
@pytest.mark.parametrize("F", [13, 64, 700, 1200, 2100, 9000])
def test_the_slope_of_open_and_closed_gates(stream, block, gate, F, monkeypatch):
    """The slope a (1 - a) of a sigmoid keeps its relative accuracy where 1 - a is small: e = exp(-|g|) is off by 2 u, 1 + e by u,
    its reciprocal by 2 u and their product by u; the smaller of a and 1 - a then by 6 u, the larger by 7 u and their product by
    14 u.  The 256 u of a gradient's terms hold that, here with the slope among their factors.  (Float64's own a (1 - a) would
    cancel as well.)"""
    def exact(g, act):
        e = torch.exp(-g.abs())
        return torch.sigmoid(g), e / (1 + e) ** 2

    monkeypatch.setitem(globals(), "act64", exact)
    s = make(24, F, stream, block, gate=gate, seed=95)
    g = torch.tensor([0.0, 0.5, 4.0, 8.0, 10.0, 12.0, 14.0, 16.0, 18.0, 24.0, 40.0, 60.0], device=DEV)
    g, t = torch.cat([g, -g]), s["t"]["gate"]
    t.copy_(g.repeat(F)[:F] if gate == "channel" else g[:, None].expand(24, t.shape[1]))
    v, m = formula(s)["gate"]
    near(train(s)[2]["gate"], (v, m * exact(t.double(), None)[1]), "d_gate")


# rows, width: more than twice as many rows as a launch has workgroups for rows of two waves and more (by width 1536, 1024, 512,
# 512, 256, 256 and 256 in the backward), and no multiple of that
TURNS = [(3301, 1100), (2301, 1999), (1301, 2500), (1301, 4096), (701, 5001), (701, 8192), (701, 8193)]


@pytest.mark.parametrize("n,F", TURNS)
@pytest.mark.parametrize("stream,block", [("f32", "f32"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("gate", [None, "row", "full"])
def test_workgroups_that_take_several_rows(n, F, stream, block, gate):
    """One row after the other in a workgroup of several waves: column sums that go on, the two buffers of the row sums in turn,
    the next row's loads under way (half rows and rows of 4097 to 6144 without a gate for each element)."""
    check(make(n, F, stream, block, "f32", "layer", "rms", gate, gate and "sigmoid", seed=101))


@pytest.mark.parametrize("n,F", TURNS)
@pytest.mark.parametrize("stream,block", [("f32", "f32"), ("f16", "f16"), ("f32", "bf16")])
def test_workgroups_that_norm_several_rows(n, F, stream, block):
    s = make(n, F, stream, block, post=None, pre="layer", gate=None, scale="number", seed=102)
    s["t"]["y"] = torch.zeros_like(s["t"]["y"])
    want = formula(s, ("h",))
    x, w, b = (s["t"][k].clone().requires_grad_() for k in ("x", "pre_weight", "pre_bias"))
    h = ops.row_norm(x, w, b, kind="layer", eps=EPS, dtype=T[block])
    near(h, want["h"], "h")
    for k, g in zip(("x", "pre_weight", "pre_bias"), torch.autograd.grad(h, (x, w, b), s["dh"])):
        near(g, want[k], "d_" + k)


def test_a_recorded_graph_is_not_differentiated_again():
    """The operators that a trace holds have no derivative of their own: differentiating their results raises."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = torch.randn(9, 12, device=DEV), torch.randn(12, device=DEV, requires_grad=True)
    with torch.no_grad():
        graph = make_fx(lambda a, b: (ops.residual_norm(a, a, post="rms", post_weight=b), ops.grad_norm([a, b])))(x, w)
    for got, want in zip(graph(x, w), (ops.residual_norm(x, x, post="rms", post_weight=w), ops.grad_norm([x, w]))):
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="not implemented"):
            got.sum().backward()
