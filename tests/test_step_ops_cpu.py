"""The training-step operators without a GPU: their PyTorch forms, their checks
of arguments, and what the C ABI rejects before it touches a device."""

import ctypes
import math

import pytest
import torch
from torch.nn import functional as F

import step_oracle as O


@pytest.mark.parametrize("implementation", ["reference", "streaming", "kernel", "native"])
def test_norm_and_stabilize_on_the_cpu(implementation):
    import jakal_net as J

    g = torch.Generator().manual_seed(1)
    x, s = torch.randn(3, 7, 20, generator=g), torch.randn(3, 7, generator=g)
    norm = J.LayerNorm(20, implementation=implementation)
    with torch.no_grad():
        norm.weight.copy_(torch.rand(20, generator=g) + 0.5)
        norm.bias.copy_(torch.randn(20, generator=g))
    assert torch.equal(norm(x), F.layer_norm(x, (20,), norm.weight, norm.bias, norm.eps))
    t, y = J.stabilize(s, x, norm.weight, norm.bias, scale=0.3, implementation=implementation)
    assert torch.equal(t, torch.tanh(s * 0.3))
    want = O.norm(x.reshape(-1, 20), norm.weight.detach(), norm.bias.detach(), 1e-5, 0.3)["y"]
    O.close("cpu", y.reshape(-1, 20), want[0], want[1] + O.U * want[0].abs())
    layer = J.Layer(dim=20, num_nodes=7, state=s, val=x)
    kept = J.stabilize_layer(layer, norm)
    assert torch.equal(kept.state, torch.tanh(s)) and torch.equal(kept.val, norm(x))
    moved = J.stabilize_layer(layer, norm, J.LayerDelta(delta_state=s + 1, delta_val=x * 2), 0.3)
    assert torch.equal(moved.state, torch.tanh((s + 1) * 0.3)) and moved.val.shape == x.shape
    plain = torch.nn.LayerNorm(20)
    assert torch.equal(J.stabilize_layer(layer, plain).val, plain(x))


def test_layer_norm_is_a_layer_norm():
    import jakal_net as J

    torch.manual_seed(0)
    a, b = torch.nn.LayerNorm(12), J.LayerNorm(12)
    assert isinstance(b, torch.nn.LayerNorm) and list(a.state_dict()) == list(b.state_dict())
    b.load_state_dict(a.state_dict())
    bare = J.LayerNorm(12, elementwise_affine=False)
    x = torch.randn(4, 12)
    assert bare.weight is None and torch.equal(bare(x), F.layer_norm(x, (12,)))
    with pytest.raises(RuntimeError):
        b(torch.randn(4, 11))
    with pytest.raises(ValueError):
        J.LayerNorm(12, implementation="fast")
    with pytest.raises(ValueError):
        J.LayerNorm((3, 4))
    with pytest.raises(RuntimeError):
        J.stabilize_layer(J.Layer.zeros(11, 3), b)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_on_the_cpu(reduction):
    import jakal_net as J

    g = torch.Generator().manual_seed(2)
    z = torch.randn(4, 5, 11, generator=g)
    t = torch.randint(0, 11, (4, 5), generator=g)
    t[1, 2] = -100
    want = O.cross_entropy(z.reshape(-1, 11), t.reshape(-1), reduction=reduction)["loss"]
    got = J.cross_entropy(z, t, reduction=reduction)
    O.close("cpu loss", got.reshape(want[0].shape), want[0], want[1] + O.U * want[0].abs())
    assert J.cross_entropy(z.bfloat16(), t, reduction=reduction).dtype is torch.float32
    with pytest.raises(RuntimeError):
        J.cross_entropy(z, t[:3], reduction=reduction)


@pytest.mark.parametrize("kind", [2.0, float("inf")])
def test_clip_on_the_cpu(kind):
    import jakal_net as J

    p = [torch.nn.Parameter(torch.zeros(s)) for s in ((3, 4), (), (0,), (70,))]
    for i, q in enumerate(p[:3]):
        q.grad = torch.full_like(q, i + 1.0)
    before = [q.grad.clone() for q in p[:3]]
    want = O.grads_norm(before, kind)
    assert float(J.clip_grad_norm_(p + p, 0.5, kind)) == pytest.approx(want, rel=1e-6)
    for q, b in zip(p, before):
        assert torch.allclose(q.grad, b * (0.5 / (want + 1e-6)), rtol=1e-6)
    assert p[3].grad is None
    out = [torch.empty(b.shape, dtype=torch.bfloat16) for b in before]
    assert float(J.clip_grads(before, 100.0, kind, out=out)) == pytest.approx(want, rel=1e-6)
    assert all(torch.equal(o, b.bfloat16()) for o, b in zip(out, before))
    assert float(J.grad_norm(None for _ in range(3))) == 0.0
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            J.clip_grads(before, bad)
    with pytest.raises(ValueError):
        J.clip_grads(before, 1.0, out=out[:2])
    p[0].grad[0, 0] = math.nan
    with pytest.raises(RuntimeError, match="cannot be clipped"):
        J.clip_grad_norm_(p, 1.0, kind, error_if_nonfinite=True)


def test_step_of_the_model_with_clipping():
    from jakal_net.progressive import ProgressiveBConfig, ProgressiveBStep, train_step
    import jakal_net as J

    cfg = ProgressiveBConfig(vocab=97, dim=32, prefix=48, query=8, rank=8, topk=4, s_window=6, warmup=1, blocks=2,
                             expanded=24, compressed=8, refine=1, query_refine=2)
    g = torch.Generator().manual_seed(3)
    prefix, target = (torch.randint(0, 96, (2, n), generator=g) for n in (48, 8))
    models = []
    for limit in (None, 1e-3):
        torch.manual_seed(4)
        model = ProgressiveBStep(cfg, implementation="streaming")
        opt = torch.optim.SGD(model.parameters(), lr=1.0)
        before = [p.detach().clone() for p in model.parameters()]
        loss, norm = train_step(model, opt, prefix, target, max_norm=limit)
        assert (norm is None) == (limit is None) and bool(torch.isfinite(loss))
        models.append([p.detach() - b for p, b in zip(model.parameters(), before)])
    # SGD at rate 1 moves by the gradients: clipped ones to a norm of 1e-3
    assert float(norm) == pytest.approx(float(J.grad_norm(models[0])), rel=1e-3)
    assert float(J.grad_norm(models[1])) == pytest.approx(1e-3, rel=1e-3)


def test_native_module_refuses_host_tensors_and_types():
    import jakal_net_native as jn

    x = torch.randn(3, 4)
    for call in (lambda: jn.layer_norm(x), lambda: jn.stabilize(x[:, 0], x), lambda: jn.grad_norm([x]),
                 lambda: jn.cross_entropy(x, torch.zeros(3, dtype=torch.int64)), lambda: jn.clip_grads([x], 1.0)):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()
    for call in (lambda: jn.layer_norm(x.double()), lambda: jn.grad_norm([x.double()]),
                 lambda: jn.stabilize(x[:, 0].long(), x), lambda: jn.grad_norm([x], 3.0),
                 lambda: jn.cross_entropy(x.double(), torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(NotImplementedError):
            call()
    for op in ("layer_norm", "stabilize", "cross_entropy", "grad_norm", "clip_grads"):
        assert op in jn.supported_ops() and hasattr(torch.ops.jakal_net_hip, op)
    # tensors without memory of their own reach no kernel
    with pytest.raises(RuntimeError):
        jn.layer_norm(torch.empty(3, 4, device="meta"))


def test_dispatch_of_the_functional_operators(monkeypatch):
    from jakal_net import native_backend as nb

    with_op = nb.NativeStatus(True, "m", "b", ("layer_norm",), ("cuda",), None)
    without = nb.NativeStatus(True, "m", "b", ("propagation_topk",), ("cuda",), None)
    missing = nb.NativeStatus(False, "m", None, (), (), "no module")
    module = type("M", (), {"layer_norm": staticmethod(lambda *a: "here")})
    for status, implementation, device, want in (
            (with_op, "native", "cuda", "here"), (with_op, "kernel", "cuda", "here"), (with_op, "reference", "cuda", None),
            (with_op, "native", "cpu", None), (without, "native", "cuda", None), (missing, "kernel", "cuda", None),
            (missing, "native", "cpu", None)):
        monkeypatch.setattr(nb, "native_status", lambda s=status: s)
        monkeypatch.setattr(nb._LOADER, "module", module)
        op = nb.native_op("layer_norm", device, implementation)
        assert (op() if op else None) == want, (status, implementation, device)
    monkeypatch.setattr(nb, "native_status", lambda: missing)
    with pytest.raises(RuntimeError, match="unavailable"):
        nb.native_op("layer_norm", "cuda", "native")
    monkeypatch.setenv("JAKAL_NET_DISABLE_NATIVE", "1")
    assert nb.native_op("layer_norm", "cuda", "native") is None


def _lib():
    import jakal_net_native as jn

    return jn._LIB


def test_c_abi_norm_checks():
    lib = _lib()
    p = ctypes.c_void_p(4096)  # never read: every call below fails or has nothing to do

    def forward(rows=4, dim=8, eps=1e-5, kind=0, state_kind=0, param=0, x=p, y=p, state=None, out=None):
        return lib.jn_layer_norm_forward(state, x, None, None, rows, dim, 1.0, eps, kind, state_kind, param, out, y,
                                         None, None)

    assert forward(rows=0) == 0
    for bad in (dict(rows=-1), dict(dim=0), dict(dim=1 << 28), dict(eps=-1.0), dict(eps=float("nan")), dict(kind=3),
                dict(kind=-1), dict(state_kind=7), dict(kind=1, param=2), dict(x=None), dict(y=None), dict(state=p),
                dict(rows=1 << 40)):
        assert forward(**bad) == 1, bad

    def backward(rows=4, dim=8, x=p, stats=p, g=p, gx=None, gw=None, gs=None, gb=None, state=None, g_state=None, ws=None,
                 ws_bytes=0):
        return lib.jn_layer_norm_backward(state, x, None, stats, g_state, g, rows, dim, 1.0, 0, 0, 0, gs, gx, gw, gb, ws,
                                          ws_bytes, None)

    assert backward() == 0  # nothing wanted
    need = lib.jn_layer_norm_backward_workspace_bytes(4, 8)
    assert need >= 4 * 2 * 8 and lib.jn_layer_norm_backward_workspace_bytes(0, 8) == 0
    for bad in (dict(rows=0), dict(gx=p, g=None), dict(gx=p, stats=None), dict(gs=p), dict(gs=p, state=p)):
        assert backward(**bad) == 1, bad
    for bad in (dict(gw=p), dict(gb=p, ws=p, ws_bytes=need - 1)):
        assert backward(**bad) == 4, bad


def test_c_abi_loss_checks():
    lib = _lib()
    p = ctypes.c_void_p(4096)

    def forward(rows=4, classes=8, reduction=2, kind=0, z=p, t=p, loss=p, reduced=p, count=p):
        return lib.jn_cross_entropy_forward(z, t, rows, classes, -100, reduction, kind, loss, None, reduced, count, None)

    for bad in (dict(rows=0), dict(classes=0), dict(classes=1 << 31), dict(reduction=3), dict(reduction=-1),
                dict(kind=3), dict(z=None), dict(t=None), dict(loss=None), dict(reduced=None), dict(count=None),
                dict(rows=1 << 40)):
        assert forward(**bad) == 1, bad

    def backward(stats=p, count=p, g=p, dz=p, reduction=2):
        return lib.jn_cross_entropy_backward(p, p, stats, count, g, 4, 8, -100, reduction, 0, dz, None)

    for bad in (dict(stats=None), dict(count=None), dict(g=None), dict(dz=None), dict(reduction=5)):
        assert backward(**bad) == 1, bad


def test_c_abi_clip_checks():
    lib = _lib()
    ws = lib.jn_grads_workspace_bytes(3)
    assert ws > 0 and lib.jn_grads_workspace_bytes(-1) == 0 and lib.jn_grads_workspace_bytes(100000) > ws
    p = ctypes.c_void_p(4096)

    def clip(spans, max_norm=1.0, kind=0, norm=p, workspace=p, ws_bytes=ws):
        n = len(spans)
        arrays = ((ctypes.c_void_p * n)(*[s[0] for s in spans]), (ctypes.c_void_p * n)(*[s[1] for s in spans]),
                  (ctypes.c_int64 * n)(*[s[2] for s in spans]), (ctypes.c_int32 * n)(*[s[3] for s in spans]),
                  (ctypes.c_int32 * n)(*[s[4] for s in spans]))
        return lib.jn_grads_clip(*arrays, n, max_norm, kind, norm, workspace, ws_bytes, None)

    good = (4096, 8192, 16, 0, 0)
    for bad in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(kind=2), dict(norm=None), dict(workspace=None)):
        assert clip([good], **bad) == 1, bad
    assert clip([good], ws_bytes=0) == 4
    for spans in ([(4096, 8192, -1, 0, 0)], [(4096, 8192, 16, 3, 0)], [(4096, 8192, 16, 0, 3)], [(None, 8192, 16, 0, 0)],
                  [(4096, None, 16, 0, 0)], [(4096, 8192, 1 << 40, 0, 0)],
                  [(4096, 4096, 16, 0, 1)],                            # in place into another type
                  [(4096, 4100, 16, 0, 0)], [(4100, 4096, 16, 0, 0)],  # an output that overlaps its gradient
                  [good, (12288, 8192 + 60, 16, 0, 0)],                # two outputs that overlap
                  [good, (8192 + 32, 20000, 4, 1, 0)],                 # an output inside another gradient
                  [(4096, 4096, 16, 0, 0), (4096, 4096, 16, 0, 0)]):   # the same tensor twice
        assert clip(spans) == 1, spans
    assert lib.jn_grads_norm(None, None, None, 1, 0, p, p, ws, None) == 1
    assert lib.jn_grads_norm(None, None, None, -1, 0, p, p, ws, None) == 1
