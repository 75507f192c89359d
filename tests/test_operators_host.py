"""Refusals of the residual join, the row norm and the gradient norm that need no GPU: arguments are checked before the
device is touched, in Python and again at the C entries."""
import ctypes as C
import math

import pytest
import torch

from disco_amd import _lib, ops

F, N = 12, 5


def _xy(dtype=torch.float32, block=None):
    return torch.zeros(N, F, dtype=dtype), torch.zeros(N, F, dtype=block or dtype)


@pytest.mark.parametrize("kwargs,error", [
    (dict(post="batch"), ValueError), (dict(pre="batch"), ValueError), (dict(gate=torch.zeros(F), gate_act="relu"), ValueError),
    (dict(gate_act="sigmoid"), ValueError), (dict(gate=torch.zeros(N)), ValueError), (dict(gate=torch.zeros(N, 2)), ValueError),
    (dict(gate=torch.zeros(1, F)), ValueError), (dict(gate=torch.zeros(N, F, dtype=torch.float16)), TypeError),
    (dict(gate=torch.zeros(N, 1, dtype=torch.bfloat16)), TypeError), (dict(gate=torch.zeros(F, dtype=torch.float64)), TypeError),
    (dict(scale=math.nan), ValueError), (dict(scale=math.inf), ValueError), (dict(scale=1e39), ValueError), (dict(eps=1e-46), ValueError), (dict(scale=torch.zeros(F + 1)), ValueError),
    (dict(scale=torch.zeros(())), ValueError), (dict(scale=torch.zeros(F, dtype=torch.int64)), TypeError),
    (dict(post_weight=torch.ones(F)), ValueError), (dict(post_bias=torch.ones(F)), ValueError),
    (dict(pre_weight=torch.ones(F)), ValueError), (dict(pre_bias=torch.ones(F)), ValueError),
    (dict(pre="rms", pre_weight=torch.ones(F, 1)), ValueError), (dict(post="rms", post_weight=torch.ones(F).double()), TypeError),
    (dict(eps=0.0), ValueError), (dict(eps=-1e-5), ValueError), (dict(eps=math.nan), ValueError), (dict(eps=math.inf), ValueError),
    (dict(), RuntimeError),                       # all in order, but on the CPU
    (dict(pre="layer", post="rms", gate=torch.zeros(N, 1), gate_act="tanh", scale=torch.ones(F)), RuntimeError)])
def test_residual_norm_refuses(kwargs, error):
    with pytest.raises(error):
        ops.residual_norm(*_xy(), **kwargs)


@pytest.mark.parametrize("x,y,error", [
    (torch.zeros(N, F), torch.zeros(N, F + 1), ValueError), (torch.zeros(N, F), torch.zeros(N + 1, F), ValueError),
    (torch.zeros(F), torch.zeros(F), ValueError), (torch.zeros(2, N, F), torch.zeros(2, N, F), ValueError),
    (torch.zeros(N, 0), torch.zeros(N, 0), ValueError), (torch.zeros(1, 16385), torch.zeros(1, 16385), ValueError),
    (torch.zeros(N, F).double(), torch.zeros(N, F).double(), TypeError), (torch.zeros(N, F).half(), torch.zeros(N, F), TypeError),
    (torch.zeros(N, F).half(), torch.zeros(N, F).bfloat16(), TypeError), (torch.zeros(N, F), torch.zeros(N, F).double(), TypeError),
    (torch.zeros(N, F), None, TypeError), (torch.zeros(N, F).to_sparse(), torch.zeros(N, F), TypeError)])
def test_residual_norm_refuses_operands(x, y, error):
    with pytest.raises(error):
        ops.residual_norm(x, y)


@pytest.mark.parametrize("args,kwargs,error", [
    ((), dict(kind="batch"), ValueError), ((), dict(kind=None), ValueError), ((torch.ones(F + 1),), {}, ValueError),
    ((torch.ones(F), torch.ones(2)), {}, ValueError), ((), dict(eps=0.0), ValueError), ((), dict(dtype=torch.float64), TypeError),
    ((), {}, RuntimeError), ((), dict(dtype=torch.bfloat16), RuntimeError)])
def test_row_norm_refuses(args, kwargs, error):
    with pytest.raises(error):
        ops.row_norm(torch.zeros(N, F), *args, **kwargs)
    with pytest.raises(TypeError):
        ops.row_norm(torch.zeros(N, F).half(), dtype=torch.float32)


def test_gradient_norm_refuses():
    g = [torch.zeros(3), torch.zeros(2, 2)]
    for p in (3, 0, -1, 0.5, math.nan):
        with pytest.raises(ValueError):
            ops.grad_norm(g, p)
    with pytest.raises(TypeError):
        ops.grad_norm([torch.zeros(3).double()])
    with pytest.raises(TypeError):
        ops.grad_norm([torch.zeros(3, 3).to_sparse()])
    with pytest.raises(TypeError):
        ops.grad_norm([None])
    with pytest.raises(ValueError):
        ops.grad_norm([torch.zeros(3), torch.zeros(3, device="meta")])
    for bad in (-1.0, math.nan, -math.inf):
        with pytest.raises(ValueError):
            ops.clip_grads(g, bad)
    for out in ([torch.zeros(3)], [torch.zeros(3), torch.zeros(4)], [torch.zeros(3), torch.zeros(2, 2).half()]):
        with pytest.raises(ValueError):
            ops.clip_grads(g, 1.0, out=out)
    for call in (lambda: ops.grad_norm(g), lambda: ops.clip_grads(g, 1.0), lambda: ops.clip_grads(g, 1.0, out=[t.clone() for t in g])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def _desc(**k):
    base = dict(rows=4, width=8, ldx=8, ldy=8, ld_gate=8, x=64, y=64, has_block=1, eps=1e-5, scale=1.0)
    return _lib.ResidualNorm(**{**base, **k})


@pytest.mark.parametrize("change", [
    dict(rows=-1), dict(width=0), dict(width=-3), dict(eps=0.0), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf),
    dict(scale=math.nan), dict(scale=math.inf), dict(stream_type=3), dict(block_type=3), dict(stream_type=1), dict(stream_type=1, block_type=2), dict(param_type=-1),
    dict(post_norm=3), dict(pre_norm=-1), dict(gate_kind=4), dict(gate_act=3), dict(x=None), dict(y=None), dict(gate_kind=1),
    dict(gate_kind=2), dict(gate_kind=3), dict(post_weight=64), dict(pre_bias=64), dict(ldx=-1), dict(ldy=-8),
    dict(has_block=0), dict(has_block=0, pre_norm=1, post_norm=1), dict(has_block=0, pre_norm=1, scale_vector=64),
    dict(has_block=0, pre_norm=1, gate_kind=1, gate=64)])
def test_residual_entries_refuse(change):
    lib = _lib.load()
    d = _desc(**change)
    assert lib.disco_residual_norm_forward(d, 64, 8, 64, 8, None, None) == -1
    g = _lib.ResidualNormGrads(dx=64, ld_dx=8, ld_dy=8, ld_dgate=8)
    if change.get("x", 64) is not None:           # the backward reads x only for the gradient of h
        assert lib.disco_residual_norm_backward(d, 64, g, 64, 1 << 20, None) == -1


def test_residual_entries_refuse_more():
    lib = _lib.load()
    assert lib.disco_residual_norm_forward(None, 64, 8, 64, 8, None, None) == -1
    assert lib.disco_residual_norm_forward(_desc(), None, 8, None, 8, None, None) == -1          # out is missing
    assert lib.disco_residual_norm_forward(_desc(pre_norm=1), 64, 8, None, 8, None, None) == -1  # h is missing
    assert lib.disco_residual_norm_forward(_desc(), 64, 7, None, 8, None, None) == -1            # rows of out overlap
    assert lib.disco_residual_norm_forward(_desc(width=16385), 64, 16385, None, 8, None, None) == -2
    assert lib.disco_residual_norm_forward(_desc(rows=0, x=None, y=None), None, 8, None, 8, None, None) == 0
    assert lib.disco_residual_norm_backward(_desc(), None, None, None, 0, None) == -1
    G = _lib.ResidualNormGrads
    ld = dict(ld_dx=8, ld_dy=8, ld_dgate=8)
    for d, g in ((_desc(), G(dpost_weight=64, **ld)), (_desc(), G(dpre_bias=64, **ld)), (_desc(), G(dscale=64, **ld)),
                 (_desc(), G(dgate=64, **ld)), (_desc(), G(dh=64, **ld)), (_desc(), G(dx=64, ld_dx=3, ld_dy=8, ld_dgate=8)),
                 (_desc(has_block=0, pre_norm=1), G(dy=64, **ld)), (_desc(has_block=0, pre_norm=1), G(dout=64, **ld)),
                 (_desc(gate_kind=2, gate=64, ld_gate=1), G(dgate=64, ld_dx=8, ld_dy=8, ld_dgate=0))):
        assert lib.disco_residual_norm_backward(d, 64, g, 64, 1 << 20, None) == -1
    d = _desc(pre_norm=1, pre_weight=64)
    assert lib.disco_residual_norm_backward(d, None, G(dh=64, dx=64, ld_dh=8, **ld), None, 0, None) == -1        # stats are missing
    assert lib.disco_residual_norm_backward(d, 64, G(dh=64, dpre_weight=64, ld_dh=8, **ld), None, 0, None) == -3
    need = lib.disco_residual_norm_workspace_bytes(4, 8)
    assert need > 0 and lib.disco_residual_norm_backward(d, 64, G(dh=64, dpre_weight=64, ld_dh=8, **ld), 64, need - 1, None) == -3
    for rows, width in ((-1, 8), (4, 0), (4, 16385)):
        assert lib.disco_residual_norm_workspace_bytes(rows, width) == 0


def test_gradient_entries_refuse():
    lib = _lib.load()
    ws = lib.disco_grad_norm_workspace_bytes(2)
    assert ws > 0 and lib.disco_grad_norm_workspace_bytes(-1) == 0

    def norm(ptrs=(4096, 8192), numel=(10, 10), types=(0, 0), n=2, p=2, out=64, work=64, nb=ws):
        return lib.disco_grad_norm((C.c_void_p * 2)(*ptrs), (C.c_int64 * 2)(*numel), (C.c_int * 2)(*types), n, p, out, work, nb, None)

    assert norm(ptrs=(None, 8192)) == -1 and norm(numel=(-1, 3)) == -1 and norm(types=(0, 3)) == -1 and norm(n=-1) == -1
    assert norm(p=3) == -1 and norm(p=-1) == -1 and norm(out=None) == -1 and norm(work=None) == -1 and norm(nb=8) == -3
    assert lib.disco_grad_norm(None, None, None, 2, 2, 64, 64, ws, None) == -1

    def clip(src=(4096, 8192), dst=(4096, 8192), numel=(10, 10), types=(0, 0), to=(0, 0), p=2, most=1.0, out=64, work=64, nb=8):
        return lib.disco_grad_clip((C.c_void_p * 2)(*src), (C.c_void_p * 2)(*dst), (C.c_int64 * 2)(*numel), (C.c_int * 2)(*types),
                                   (C.c_int * 2)(*to), 2, p, most, out, work, nb, None)

    assert clip() == -3                                                    # all in order, the workspace is too small
    assert clip(most=-1.0) == -1 and clip(most=math.nan) == -1 and clip(p=7) == -1 and clip(out=None) == -1 and clip(work=None) == -1
    assert clip(to=(1, 0)) == -1 and clip(types=(1, 1), to=(2, 2)) == -1   # neither the gradient's type nor float32
    assert clip(dst=(None, 8192)) == -1
    # shared memory: the same tensor twice, a part of another, an output over another gradient, over its own with an offset
    assert clip(src=(4096, 4096), dst=(4096, 4096)) == -1
    assert clip(src=(4096, 4132), dst=(4096, 4132)) == -1
    assert clip(src=(4096, 4136), dst=(4096, 4136)) == -3
    assert clip(dst=(8192, 4096)) == -1 and clip(dst=(4100, 8192)) == -1
    assert clip(types=(1, 1), to=(0, 1)) == -1                             # in place with a wider type
    assert clip(src=(4096, 4096), dst=(16384, 32768)) == -3                # read twice, written apart: allowed


def test_residual_models_refuse_and_leave_the_others_alone():
    from disco_amd.models import basicgnn_large as M
    from disco_amd.models.residual import ResidualNorm, RowNorm
    kw = dict(nfeat=6, nhid=8, nclass=3)
    for bad in (dict(nlayers=2), dict(nlayers=4, norm="BatchNorm"), dict(nlayers=4, jk="cat"), dict(nlayers=4, nclass=None)):
        with pytest.raises(ValueError):
            M.GCN(residual=True, **{**kw, **bad})
    with pytest.raises(ValueError):
        M.SGC(nlayers=3, sgc=True, residual=True, **kw)
    for bad in (dict(gate="edge"), dict(post="batch"), dict(pre="batch"), dict(pre=None)):
        with pytest.raises(ValueError):
            M.GCN(nlayers=4, residual=bad, **kw)
    with pytest.raises(ValueError):
        RowNorm(8, "batch")
    plain = M.GCN(nlayers=4, **kw)
    assert not any(k.startswith(("joins", "first_norm")) for k in plain.state_dict())
    keys = set(M.GCN(nlayers=4, residual=dict(gate="node", learn_scale=True, post="rms"), **kw).state_dict())
    assert keys - set(plain.state_dict()) == {"first_norm.weight", "first_norm.bias"} | {
        f"joins.{i}.{k}" for i in range(2) for k in ("post.weight", "pre.weight", "pre.bias", "scale", "gate.weight", "gate.bias")}
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ResidualNorm(8)(torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        RowNorm(8)(torch.zeros(4, 8))


def test_the_torch_operator_is_built_and_bound():
    op = _lib.torch_op("residual_norm")
    assert "libdisco_torch.so" in open("/proc/self/maps").read()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        op(torch.zeros(4, 8), None, None, None, None, None, None, None, 1 << 2, 1.0, 1e-5, 0)
    norm = _lib.torch_op("gradient_norm")
    assert norm([], None, 2, 0.0, 0) is None and norm([torch.zeros(3)], None, 2, 0.0, 0) is None


def test_the_torch_operators_take_no_stream():
    """A stream handle among the arguments would be a constant of a traced module: the operators read the current stream."""
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _lib.torch_op("residual_norm")(torch.zeros(4, 8), None, None, None, None, None, None, None, 1 << 2, 1.0, 1e-5)
    assert _lib.torch_op("gradient_norm")([torch.zeros(3)], None, 2, 0.0) is None


def test_forward_mode_derivatives_are_refused():
    """A tangent on a tensor that needs no gradient must not be dropped without a word."""
    import torch.autograd.forward_ad as fwad
    x, w = torch.zeros(4, 8), torch.ones(8)
    with fwad.dual_level():
        d, dw = fwad.make_dual(x, torch.ones_like(x)), fwad.make_dual(w, torch.ones_like(w))
        op, norm = _lib.torch_op("residual_norm"), _lib.torch_op("gradient_norm")
        for args in ((d, None, None, None, None, None, None, None), (x, d, None, None, None, None, None, None), (x, None, None, None, None, None, dw, None)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                op(*args, 1 << 2, 1.0, 1e-5)
        for grads, out in (([x, d], None), ([x, x], [d, x])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                norm(grads, out, 2, 1.0)


def test_a_trace_holds_the_operators():
    """Fake tensors pass through, and a recorded graph holds the calls (not the empty buffers that they fill)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    with FakeTensorMode():
        x, y, w = torch.empty(6, 8, device="cuda"), torch.empty(6, 8, device="cuda", dtype=torch.bfloat16), torch.empty(8, device="cuda")
        out, h = ops.residual_norm(x, y, post="rms", post_weight=w, pre="layer")
        assert out.dtype == torch.float32 and h.dtype == torch.bfloat16 and out.shape == h.shape == (6, 8)
        assert ops.grad_norm([x, y]).shape == ()
        block = make_fx(lambda x, y, w: ops.residual_norm(x, y, post="rms", post_weight=w, pre="layer"))(x, y, w)
        clip = make_fx(lambda x, w: (ops.grad_norm([x, w]), ops.clip_grads([x, w], 1.0), x))(x, w)
    calls = [[n.target for n in g.graph.nodes if n.op == "call_function"] for g in (block, clip)]
    assert torch.ops.disco_amd.residual_norm_forward.default in calls[0] and torch.ops.aten.empty.memory_format not in calls[0]
    assert calls[1] == [torch.ops.disco_amd.grad_norm.default, torch.ops.disco_amd.grad_clip.default]


class _Dense(torch.nn.Module):
    """Stands for a convolution where no graph is needed."""

    def __init__(self, nfeat, nclass):
        super().__init__()
        self.lin = torch.nn.Linear(nfeat, nclass)

    def reset_parameters(self):
        self.lin.reset_parameters()

    def forward(self, x, adj, edge_weight=None):
        return self.lin(x)


def test_models_from_before_residual_blocks_still_run():
    """A model pickled whole when BasicGNN had no residual blocks has no such attribute."""
    import copy
    from collections import namedtuple
    from disco_amd.models import basicgnn_large as M

    class Net(M.BasicGNN):
        def init_conv(self, nfeat, nclass, **kwargs):
            return _Dense(nfeat, nclass)

    new = Net(nfeat=6, nhid=8, nlayers=3, nclass=4).eval()
    old = copy.deepcopy(new)
    old.__dict__.pop("residual", None)
    x = torch.randn(5, 6)
    Batch = namedtuple("Batch", ["adj_t"])
    adj = torch.zeros(1)
    for call in (lambda m: m.forward(x, None), lambda m: m.forward_sampler(x, [(None, None, None)] * 3),
                 lambda m: m.inference(x, [(5, torch.arange(5), Batch(adj))], "cpu")):
        assert torch.equal(call(old), call(new))
    old.initialize()


@pytest.mark.parametrize("off", [False, None, 0])
def test_residual_blocks_can_be_switched_off(off):
    from disco_amd.models import basicgnn_large as M
    for kw in (dict(nlayers=4), dict(nlayers=2, norm="BatchNorm"), dict(nlayers=3, jk="cat")):
        m = M.GCN(nfeat=6, nhid=8, nclass=3, residual=off, **kw)
        assert m.residual is False and not hasattr(m, "joins")
    for on in (True, 1, {}, dict(pre="rms"), [("pre", "rms")]):
        m = M.GCN(nfeat=6, nhid=8, nclass=3, nlayers=4, residual=on)
        assert m.residual is True and len(m.joins) == 2


def test_the_c_library_is_built_without_torch(monkeypatch):
    """libdisco_hip.so needs hipcc alone; libdisco_torch.so is built beside it, after it."""
    from disco_amd import build
    called = []
    monkeypatch.setattr(build, "build_torch_lib", lambda *a, **k: called.append("torch") or "")
    monkeypatch.setattr(build, "_newest_source_mtime", lambda: 0.0)
    assert build.build_lib() == build.lib_path() and called == []
    monkeypatch.setattr(build, "build_lib", lambda *a, **k: called.append("hip") or "lib")
    assert build.build_all() == "lib" and called == ["hip", "torch"]


def _written_twice(dst, in_place):
    """Whether clipping refuses the destinations; those numbered in ``in_place`` are their gradients themselves."""
    try:
        _lib.torch_op("copied_pairs")([d if i in in_place else torch.empty(d.shape) for i, d in enumerate(dst)], dst)
    except ValueError as e:
        assert "share memory" in str(e)
        return True
    return False


def test_destinations_that_would_be_written_twice():
    t = torch.zeros(64, 100)
    half = t.view(torch.float16)
    same = t.as_strided((4, 4), (1, 1))
    apart = t.as_strided((3, 2), (2, 3))          # 0 3 2 5 4 7
    for dst, twice in (([t[:, :48], t[:, 48:]], False), ([t[:, :49], t[:, 48:]], True), ([t[:, ::2], t[:, 1::2]], False), ([t[:, ::2], t[:, ::4]], True),
                       ([t, t[:, ::2]], True), ([t[:32], t[32:, ::2]], False), ([t[:, 3], t[:, 4]], False), ([t[::2, 3], t[4, ::3]], True),
                       ([t[::2, 3], t[5, ::3]], False), ([same], True), ([apart], False), ([t.t()[:, ::2], t[1::2]], False), ([t[0:1].expand(5, 100)], True),
                       ([t[:, :50], half[:, 100:]], False), ([t[:, :51], half[:, 100::2]], True), ([t[:0], t[:0]], False), ([t[0, 0], t[:, 1::2]], False),
                       ([t[0, 1], t[:, 1::2]], True)):
        for order in (dst, dst[::-1]):
            assert _written_twice(order, ()) == twice, [(d.shape, d.stride(), d.storage_offset()) for d in order]
            assert not _written_twice(order, range(len(dst)))
            if len(dst) == 2:
                assert _written_twice(order, (0,)) == twice


def test_shared_memory_against_counting():
    """Random views of a small buffer against the places that each of them really has."""
    import random
    r, base, met = random.Random(5), torch.zeros(400), 0

    def view():
        dims = r.randint(0, 3)
        size, stride = [r.randint(1, 5) for _ in range(dims)], [r.choice([0, 1, 2, 3, 5, 7, 10, 20, 21]) for _ in range(dims)]
        return base.as_strided(size, stride, r.randint(0, 60))

    def places(v):
        return [int(i) for i in torch.arange(400).as_strided(v.size(), v.stride(), v.storage_offset()).reshape(-1)]

    for _ in range(3000):
        a, b = view(), view()
        p, q = places(a), places(b)
        want = len(set(p)) < len(p) or len(set(q)) < len(q) or bool(set(p) & set(q))
        assert _written_twice([a, b], ()) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        assert _written_twice([a, b], (0,)) == (len(set(q)) < len(q) or bool(set(p) & set(q)))
        met += want
    assert 500 < met < 2500


def test_the_backward_asks_for_y_where_it_reads_it():
    lib, G = _lib.load(), _lib.ResidualNormGrads
    g = dict(dout=64, ld_dout=8, ld_dx=8, ld_dy=8, ld_dgate=8)      # nothing is wanted: nothing is launched
    assert lib.disco_residual_norm_backward(_desc(y=None), None, G(**g), None, 0, None) == 0
    for d, more in ((dict(post_norm=1), {}), (dict(gate_kind=1, gate=64), {}), (dict(gate_kind=3, gate=64), {}), (dict(scale_vector=64), {}),
                    (dict(pre_norm=1), dict(dh=64, ld_dh=8)), ({}, dict(dout=None))):
        assert lib.disco_residual_norm_backward(_desc(y=None, **d), 64, G(**{**g, **more}), None, 0, None) == -1
        assert lib.disco_residual_norm_backward(_desc(**d), 64, G(**{**g, **more}), None, 0, None) == 0
