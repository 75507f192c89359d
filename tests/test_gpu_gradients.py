"""The norm over all gradients and clipping against float64.

Tolerances: the norm is summed in float64 (error about count * 2^-53, far below a float32 step), so the float32 result is
off by half a step, 2^-24 relative.  A clipped value is g * factor with the factor rounded to float32 and the product
rounded to float32: 2 half steps, and half a step of a narrower output type on top."""
import math

import numpy as np
import pytest
import torch

import disco_amd
from disco_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(sizes, dtypes, seed=0, size=0.05):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(s if isinstance(s, tuple) else (s,), generator=g, device=DEV) * size * (1 + i % 7)).to(dtypes[i % len(dtypes)])
            for i, s in enumerate(sizes)]


def norm64(grads, p):
    parts = [g.double().abs().reshape(-1) for g in grads]
    v = torch.cat(parts) if parts else torch.zeros(0, dtype=torch.float64, device=DEV)
    if p == math.inf:
        return float(v.max()) if v.numel() else 0.0
    return float(v.sum()) if p == 1 else math.sqrt(float((v * v).sum()))


def check_norm(got, want):
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - want) <= want * U * (1 + 1e-6), (float(got), want)


def check_clip(grads, out, max_norm, norm):
    factor = min(1.0, max_norm / (norm + 1e-6))
    for g, o in zip(grads, out):
        want = g.double() * factor
        half = 2 * U + (torch.finfo(o.dtype).eps / 2 if o.dtype != torch.float32 else 0.0)
        tiny = torch.finfo(o.dtype).smallest_normal * torch.finfo(o.dtype).eps
        assert ((o.double() - want).abs() <= half * want.abs() * (1 + 1e-6) + tiny).all()


SIZES = {"one": [1], "small": [1, 2, 3, 255, 256, 257, 1000], "edge": [4095, 4096, 4097, 8192, 8191, 12289], "shapes": [(3, 5), (1,), (), (64, 65), (2, 3, 4)],
         "empty ones": [0, 5, 0, (0, 4), 7], "many": [17 + 13 * i for i in range(450)], "uneven": [3, 3000000, 1, 70000, 5]}


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("sizes", SIZES, ids=list(SIZES))
@pytest.mark.parametrize("dtypes", [DTYPES[:1], DTYPES[1:2], DTYPES[2:], DTYPES], ids=["f32", "f16", "bf16", "mixed"])
def test_norm_and_clip(p, sizes, dtypes):
    grads = make(SIZES[sizes], dtypes, seed=len(sizes))
    want = norm64(grads, p)
    check_norm(ops.grad_norm(grads, p), want)
    for max_norm in (0.3 * want, 3.0 * want + 1.0, 0.0):
        to = [torch.full_like(g, 7, dtype=torch.float32 if i % 2 else g.dtype) for i, g in enumerate(grads)]
        before = [g.clone() for g in grads]
        check_norm(ops.clip_grads(grads, max_norm, p, out=to), want)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        check_clip(grads, to, max_norm, want)
        own = [g.clone() for g in grads]
        check_norm(ops.clip_grads(own, max_norm, p), want)
        check_clip(grads, own, max_norm, want)
        if max_norm > want:
            assert all(torch.equal(a, b) for a, b in zip(own, before))


@pytest.mark.parametrize("max_norm", [math.inf, 1e30])
def test_nothing_to_clip(max_norm):
    grads = make([100, 5000], DTYPES)
    own = [g.clone() for g in grads]
    ops.clip_grads(own, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(own, grads))


def test_no_tensors():
    for got in (ops.grad_norm([]), ops.clip_grads([], 1.0), ops.grad_norm(iter(())), ops.grad_norm([torch.zeros(0, device=DEV)]),
                ops.clip_grads([torch.zeros(0, device=DEV)], 1.0), disco_amd.clip_grad_norm_([torch.nn.Parameter(torch.ones(3, device=DEV))], 1.0)):
        assert got.dtype == torch.float32 and float(got) == 0.0


def test_one_tensor_and_generators():
    g = make([300], DTYPES[:1])[0]
    check_norm(ops.grad_norm(g), norm64([g], 2))
    check_norm(ops.grad_norm(t for t in (g, g)), math.sqrt(2) * norm64([g], 2))      # named twice, counted twice
    check_norm(ops.clip_grads(g, 0.1), norm64(make([300], DTYPES[:1]), 2))


def test_sums_that_leave_float32():
    g = [torch.full((1000,), 1e25, device=DEV), torch.full((1000,), 1e-30, device=DEV)]
    check_norm(ops.grad_norm(g), norm64(g, 2))
    check_norm(ops.grad_norm(g[1:]), norm64(g[1:], 2))
    big = [torch.full((4096,), 3e38, device=DEV)]
    assert float(ops.grad_norm(big)) == math.inf                    # 3e38 * 64 is no float32
    ops.clip_grads(big, 1.0)                                        # the factor comes from the float64 norm
    assert ((big[0] - 1 / 64).abs() <= 2 * U / 64).all()


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_nan_and_infinity(p):
    for bad, at in ((math.nan, 0), (math.nan, 9999), (math.inf, 4096), (-math.inf, 70)):
        grads = make([10000, 50], DTYPES[:1], seed=3)
        grads[0][at] = bad
        n = ops.grad_norm(grads, p)
        assert math.isnan(float(n)) if math.isnan(bad) else float(n) == math.inf
        own = [g.clone() for g in grads]
        with pytest.raises(RuntimeError, match="norm"):
            ops.clip_grads(own, 1.0, p, error_if_nonfinite=True)
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(own, grads))
        ops.clip_grads(own, 1.0, p)
        if math.isnan(bad):
            assert all(g.isnan().all() for g in own)
        else:
            assert own[0][at].isnan() and not own[1].any() and int(own[0].isnan().sum()) == 1
    finite = make([10, 20], DTYPES, seed=4)
    want = norm64(finite, p)
    check_norm(ops.clip_grads([g.clone() for g in finite], 0.01, p, error_if_nonfinite=True), want)


def test_layouts():
    base = make([(64, 48)], DTYPES[:1], seed=5)[0]
    dense_t = base.t()                                               # dense, in another order
    gaps = torch.randn(64, 100, device=DEV)[:, 10:58]                # rows with gaps
    step = torch.randn(1000, device=DEV)[1::3]
    shifted = torch.randn(5001, device=DEV)[1:]
    half = torch.randn(9001, device=DEV).half()[3:]
    grads = [dense_t, gaps, step, shifted, half]
    want = norm64(grads, 2)
    check_norm(ops.grad_norm(grads), want)
    keep = [g.clone() for g in grads]
    to = [torch.empty_like(g, memory_format=torch.contiguous_format) for g in grads]
    check_norm(ops.clip_grads(grads, 1.0, out=to), want)
    check_clip(keep, to, 1.0, want)
    hole = torch.full((64, 100), 5.0, device=DEV)
    hole[:, 10:58] = gaps
    grads[1] = hole[:, 10:58]
    check_norm(ops.clip_grads(grads, 1.0), want)
    check_clip(keep, grads, 1.0, want)
    assert (hole[:, :10] == 5).all() and (hole[:, 58:] == 5).all()


def test_views_of_one_buffer_and_shared_memory():
    flat = torch.randn(10007, device=DEV)
    views = [flat[:3], flat[3:4100], flat[4100:]]
    keep, want = flat.clone(), norm64([flat], 2)
    check_norm(ops.clip_grads(views, 1.0), want)
    check_clip([keep], [flat], 1.0, want)
    for bad in ([flat[:10], flat[:10]], [flat[:10], flat[9:20]], [flat[5:6].expand(4)], [flat[:100], flat[50:60], flat[200:]]):
        before = flat.clone()
        with pytest.raises(ValueError, match="share memory"):
            ops.clip_grads(bad, 1.0)
        assert torch.equal(flat, before)
    with pytest.raises(ValueError, match="share memory"):
        ops.clip_grads([flat[:10], flat[20:30]], 1.0, out=[flat[20:30], flat[:10]])
    with pytest.raises(ValueError, match="share memory"):
        ops.clip_grads([flat[:10]], 1.0, out=[flat[1:11]])


def test_views_with_gaps_that_share_memory_are_scaled_once():
    hole = torch.randn(64, 100, device=DEV)
    keep = hole.clone()
    for views in (lambda t: [t[:, 10:58], t[:, 10:58]], lambda t: [t[:, 10:58], t[:, 40:90]], lambda t: [t[:, ::2], t[:, 1::2]],
                  lambda t: [t[:, 10:58], t[20:30]]):
        hole.copy_(keep)
        before, after = views(keep), views(hole)
        want = norm64(before, 2)
        check_norm(ops.clip_grads(after, 1.0), want)
        check_clip(before, after, 1.0, want)


def test_parameters():
    m = torch.nn.Sequential(torch.nn.Linear(40, 30), torch.nn.BatchNorm1d(30), torch.nn.Linear(30, 1)).to(DEV)
    unused = torch.nn.Parameter(torch.ones(5, device=DEV))
    m(torch.randn(16, 40, device=DEV)).square().sum().backward()
    keep = [p.grad.clone() for p in m.parameters()]
    want = norm64(keep, 2)
    check_norm(ops.clip_grad_norm_(list(m.parameters()) + [unused], 0.25), want)
    check_clip(keep, [p.grad for p in m.parameters()], 0.25, want)
    assert unused.grad is None
    check_norm(ops.clip_grad_norm_(m[0].weight, 1.0), norm64([m[0].weight.grad], 2))


def test_captured_clip_replays_and_streams():
    """Two captured graphs of the same gradients, replayed in turn with eager calls in between: workspaces are not shared."""
    grads = make([5000, 33, 70001], DTYPES[:1], seed=9)
    to = [[torch.zeros_like(g) for g in grads] for _ in range(2)]
    for t in to:
        ops.clip_grads(grads, 1.0, out=t)
    torch.cuda.synchronize()
    graphs, norms = [], []
    for k, p in enumerate((2.0, math.inf)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(ops.clip_grads(grads, 1.0 if k == 0 else 0.02, p, out=to[k]))
        graphs.append(g)
    for i in range(4):
        for t in grads:
            t.copy_(torch.randn_like(t) * (i + 1))
        eager = [(ops.clip_grads(grads, 1.0, 2.0, out=(a := [torch.empty_like(g) for g in grads])), a),
                 (ops.clip_grads(grads, 0.02, math.inf, out=(b := [torch.empty_like(g) for g in grads])), b)]
        for g in (graphs if i % 2 else graphs[::-1]):
            g.replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(norms[k], eager[k][0]), i
            assert all(torch.equal(x, y) for x, y in zip(to[k], eager[k][1])), i
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n = ops.grad_norm(grads)
    side.synchronize()
    assert torch.equal(n, ops.grad_norm(grads))


def test_repeated_runs_give_the_same_bits():
    grads = make([123457, 99, 4096 * 50 + 1], DTYPES, seed=12)
    first = [float(ops.grad_norm(grads, p)) for p in (1, 2, math.inf)]
    for _ in range(5):
        assert [float(ops.grad_norm(grads, p)) for p in (1, 2, math.inf)] == first


def test_a_tensor_behind_2_to_the_32_elements():
    """Offsets inside a tensor are 64 bits wide: ones in front of and behind 2^32 elements."""
    n = 2 ** 32 + 12345
    g = torch.zeros(n, dtype=torch.float16, device=DEV)
    g[:7], g[-5:] = 1.0, 2.0
    assert float(ops.grad_norm([g], 1)) == 17.0 and float(ops.grad_norm([g], math.inf)) == 2.0
    check_norm(ops.grad_norm([g]), math.sqrt(27.0))
    ops.clip_grads([g], 1.7, 1)
    want = torch.tensor([1.7 / 17 * 2], device=DEV).half()
    assert (g[-5:] - want).abs().max() <= 2.0 ** -10 * 0.2 and (g[:7] - want / 2).abs().max() <= 2.0 ** -10 * 0.2
    assert not g[7:1000].any() and not g[-1000:-5].any()


@pytest.mark.parametrize("case", range(12))
def test_drawn_cases(case):
    r = np.random.default_rng(case)
    sizes = [int(np.exp(r.uniform(0, np.log(2e5)))) for _ in range(int(r.integers(1, 300)))]
    grads = make(sizes, [DTYPES[int(r.integers(3))], DTYPES[int(r.integers(3))]], seed=case)
    p = [1.0, 2.0, math.inf][int(r.integers(3))]
    want = norm64(grads, p)
    to = [torch.empty_like(g, dtype=[g.dtype, torch.float32][int(r.integers(2))]) for g in grads]
    check_norm(ops.clip_grads(grads, want * 0.5, p, out=to), want)
    check_clip(grads, to, want * 0.5, want)


def test_clipping_is_seen_by_autograd():
    """Gradients written in place count as modified: a graph that saved one of them refuses to use it."""
    x = torch.randn(50, device=DEV, requires_grad=True)
    g = torch.randn(50, device=DEV)
    y = x * g
    ops.clip_grads([g], 1e-3)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()
    with torch.inference_mode():
        h = torch.ones(10, device=DEV)
        check_norm(ops.clip_grads([h], 1.0), math.sqrt(10.0))
    want = norm64([h], 2)                        # max_norm * norm / (norm + 1e-6), not quite max_norm
    check_norm(ops.clip_grads([h, torch.zeros(3, device=DEV)], 5.0), want)


def test_a_recorded_graph_clips():
    from torch.fx.experimental.proxy_tensor import make_fx
    grads = make([100, 3000], DTYPES[:1], seed=21)
    graph = make_fx(lambda *g: (ops.grad_norm(g), ops.clip_grads(g, 0.5)))(*[g.clone() for g in grads])
    other = [g * 2 for g in grads]
    eager = [g.clone() for g in other]
    n1, n2 = graph(*other)
    want = ops.clip_grads(eager, 0.5)
    assert torch.equal(n1, want) and torch.equal(n2, want) and all(torch.equal(a, b) for a, b in zip(other, eager))


def test_the_norm_is_no_constant_of_a_graph():
    """Gradients of gradients: the norm has no derivative, and whoever differentiates it is told; without that it is a number like
    any other, and clipping leaves no trace in the graph."""
    x = torch.randn(50, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(x.pow(3).sum(), x, create_graph=True)
    norm = ops.grad_norm([g, torch.ones(3, device=DEV)])
    check_norm(norm.detach(), norm64([g.detach(), torch.ones(3, device=DEV)], 2))
    with pytest.raises(RuntimeError, match="no derivative"):
        (norm * 2.0).backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(g.sum() + norm, x, retain_graph=True)
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(ops.grad_norm(torch.stack([g, g], 1)[:, 0]), x, retain_graph=True)      # a view with gaps
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(ops.grad_norm([x]), x)
    with torch.no_grad():
        assert not ops.grad_norm([g]).requires_grad
    assert not ops.grad_norm([g.detach()]).requires_grad and not ops.clip_grads([g.detach().clone()], 1.0).requires_grad
    (h,) = torch.autograd.grad(g.sum(), x)
    assert torch.allclose(h, 6 * x.detach(), rtol=4 * U)


def test_lazily_negated_gradients():
    """Views that are negated when read (torch's negative bit): gradients and destinations, dense and with gaps."""
    z = torch.randn(40, 2, device=DEV)
    for view in (torch._neg_view, lambda t: torch._neg_view(t[:, :1])):
        store = z.clone()
        g = view(store)
        assert g.is_neg()
        keep = g.clone()
        want = norm64([keep], 2)
        check_norm(ops.grad_norm([g, torch.zeros(3, device=DEV)]), want)
        to = torch.empty_like(keep)
        check_norm(ops.clip_grads([g], 0.5, out=[to]), want)
        check_clip([keep], [to], 0.5, want)
        to = view(torch.zeros(40, 2, device=DEV))
        check_norm(ops.clip_grads([keep], 0.5, out=[to]), want)
        check_clip([keep], [to], 0.5, want)
        check_norm(ops.clip_grads([g], 0.5), want)
        check_clip([keep], [g], 0.5, want)


def test_two_gradients_into_one_view_with_gaps_are_refused():
    grads = make([(60, 48), (60, 48)], DTYPES[:1], seed=31)
    hole = torch.full((60, 100), 5.0, device=DEV)
    for out in ([hole[:, :48], hole[:, :48]], [hole[:, :48], hole[:, 47:95]], [hole[:, :48], hole.view(-1)[:60 * 49].view(60, 49)[:, :48]],
                [grads[1][:, :48], grads[1]]):
        before = [g.clone() for g in grads]
        with pytest.raises(ValueError, match="share memory"):
            ops.clip_grads(grads, 0.5, out=out)
        assert (hole == 5).all() and all(torch.equal(a, b) for a, b in zip(grads, before))
    out = [hole[:, :48], hole[:, 48:96]]                              # beside each other in one buffer
    want = norm64(grads, 2)
    check_norm(ops.clip_grads(grads, 0.5, out=out), want)
    check_clip(grads, out, 0.5, want)
    assert (hole[:, 96:] == 5).all()
    wide = torch.randn(60, 100, device=DEV)                           # in place beside a destination of its own
    keep = wide[:, :48].clone()
    pair = [wide[:, :48], grads[1]]
    want = norm64(pair, 2)
    check_norm(ops.clip_grads(pair, 0.5, out=[pair[0], wide[:, 50:98]]), want)
    check_clip([keep, grads[1]], [wide[:, :48], wide[:, 50:98]], 0.5, want)


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("top,most", [(0.05, 0.3), (3e38, 1e-3), (1e-30, 1e-33), (1e30, 1e-4)])
def test_the_factor_is_not_rounded(p, top, most):
    """Factor and product are float64 (the factor beside gradients near float32's end is no normal float32): a clipped value is
    rounded once, to float32, and once more to a narrower output: U, and half a step of that."""
    base = torch.rand(5000, generator=torch.Generator(device=DEV).manual_seed(41), device=DEV) * top
    grads = [base, base[:77].bfloat16()]
    norm = norm64(grads, p)
    factor = min(1.0, most / (norm + 1e-6))
    for dtypes in ((torch.float32, torch.float32), (torch.float32, torch.bfloat16)):
        to = [torch.empty_like(g, dtype=t) for g, t in zip(grads, dtypes)]
        ops.clip_grads(grads, most, p, out=to)
        for g, o in zip(grads, to):
            want = g.double() * factor
            half = U + (torch.finfo(o.dtype).eps / 2 if o.dtype != torch.float32 else 0.0)
            assert ((o.double() - want).abs() <= half * want.abs() * (1 + 1e-6) + torch.finfo(o.dtype).smallest_normal * torch.finfo(o.dtype).eps).all()


@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_clipping(dynamic):
    f = torch.compile(lambda g, o: (ops.clip_grads(g, 0.5, out=o), ops.grad_norm(o)), backend="aot_eager", dynamic=dynamic)
    try:
        for n in (100, 77, 3000):
            grads = make([(n, 3), n], DTYPES[:2], seed=n)
            got, want = ([torch.empty_like(g, dtype=torch.float32) for g in grads] for _ in range(2))
            a, b = f(grads, got)
            assert torch.equal(a, ops.clip_grads(grads, 0.5, out=want)) and torch.equal(b, ops.grad_norm(want))
            assert all(torch.equal(x, y) for x, y in zip(got, want))
    finally:
        torch._dynamo.reset()
