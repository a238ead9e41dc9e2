"""Operators on microscaled numbers without a GPU: their PyTorch forms against
tests/mx_oracle.py, their checks of arguments, fake tensors, the modules and the
model, and what the C ABI rejects before it touches a device."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.nn import functional as F

import mx_oracle as M
import step_oracle as O

MODES = ["reference", "streaming", "kernel", "native"]


def _rand(seed, *shape, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


@pytest.mark.parametrize("form", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_quantize(form, dtype):
    import jakal_net as J

    for dim in (1, 7, 31, 32, 33, 100, 256):
        x = _rand(dim, 3, 5, dim) * torch.exp(3 * _rand(dim + 1, 3, 5, 1))
        x[0, 0], x[1, 0] = 0.0, -0.0
        x[2, 0, dim // 2], x[2, 1, 0] = float("inf"), float("nan")
        x = x.to(O.DTYPES[dtype])
        value, code, scale = M.quantize(x, form)
        for mode in MODES:
            q = J.mx_quantize(x, form, implementation=mode)
            assert torch.equal(q.codes, M.packed(code, form)) and torch.equal(q.scales.long(), scale.long())
            assert q.shape == x.shape and q.dtype is x.dtype and q.nbytes == q.codes.numel() + q.scales.numel()
            back = J.mx_dequantize(q, torch.float32, implementation=mode)
            want = value.float()
            assert bool(((back == want) | (back.isnan() & want.isnan())).all()) and J.mx_dequantize(q).dtype is x.dtype


def test_every_code_of_every_scale():
    import jakal_net as J

    for form, codes in (("e4m3", 256), ("e2m1", 16)):
        grid = M.magnitudes(form)
        width = 32 if form == "e4m3" else 16
        for s in (0, 1, 2, 127, 200, 254, 255):
            for code in range(codes):
                c = torch.zeros(1, width, dtype=torch.uint8)
                c[0, 0] = code
                t = J.MXTensor(c, torch.tensor([[s]], dtype=torch.uint8), form, 32)
                got = float(J.mx_dequantize(t)[0, 0])
                size, sign = code % (codes // 2), -1.0 if code >= codes // 2 else 1.0
                if s == 255 or size >= len(grid):
                    assert got != got
                else:
                    assert got == float((sign * grid[size] * 2.0 ** (s - 127)).float())


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("acts", [None, "e2m1"])
def test_mx_linear(mode, acts):
    import jakal_net as J

    x, g, b = _rand(1, 4, 6, 50), _rand(2, 4, 6, 9), _rand(3, 9)
    weight = J.mx_quantize(_rand(4, 9, 50), "e2m1")
    w = M.quantize(_rand(4, 9, 50), "e2m1")[0]
    x.requires_grad_(), b.requires_grad_()
    y = J.mx_linear(x, weight, b, activations=acts, implementation=mode)
    a = x.detach().reshape(-1, 50) if acts is None else M.quantize(x.reshape(-1, 50), acts)[0]
    value, bound = M.product(a, w.t(), b.detach())
    O.close("y", y.reshape(-1, 9), value, bound + O.U * value.abs())
    gx, gb = torch.autograd.grad(y, (x, b), g)
    value, bound = M.product(g.reshape(-1, 9), w)
    O.close("grad_x", gx.reshape(-1, 50), value, bound + O.U * value.abs())
    value, bound = M.sums(g.reshape(-1, 9))
    O.close("grad_bias", gb, value, bound + O.U * value.abs())


@pytest.mark.parametrize("mode", MODES)
def test_layers_that_keep_their_input(mode):
    import jakal_net as J

    x, w, b, g = _rand(1, 3, 7, 40), _rand(2, 6, 40, scale=0.2), _rand(3, 6), _rand(4, 3, 7, 6)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = J.linear(*leaves, saved="e4m3", implementation=mode)
    assert torch.equal(y, F.linear(*leaves)) and torch.equal(J.linear(*leaves, implementation=mode), y)
    gx, gw, gb = torch.autograd.grad(y, leaves, g)
    flat = g.reshape(-1, 6)
    for name, got, (value, bound) in (("grad_x", gx.reshape(-1, 40), M.product(flat, w.detach())),
                                      ("grad_weight", gw, M.product(flat.t(), M.quantize(x.reshape(-1, 40), "e4m3")[0])),
                                      ("grad_bias", gb, M.sums(flat))):
        O.close(name, got, value, bound + O.U * value.abs())
    y, g = J.gelu(x, saved="e4m3", implementation=mode), _rand(5, 3, 7, 40)
    assert torch.equal(y, F.gelu(x)) and torch.equal(J.gelu(x, implementation=mode), y)
    value, bound = M.gelu_slope(M.quantize(x, "e4m3")[0], g)
    O.close("gelu", torch.autograd.grad(y, x, g)[0], value, bound + O.U * value.abs())
    state, weight, bias = _rand(6, 3, 7), 1 + 0.1 * _rand(7, 40), _rand(8, 40)
    leaves = [t.requires_grad_() for t in (state, x, weight, bias)]
    t, y = J.stabilize(*leaves, scale=0.4, saved="e4m3", implementation=mode)
    plain = J.stabilize(*leaves, scale=0.4, implementation=mode)
    assert torch.equal(t, plain[0]) and torch.equal(y, plain[1])
    grads = torch.autograd.grad((t, y), leaves, (torch.ones_like(t), g))
    assert torch.equal(grads[0], torch.autograd.grad(plain[0].sum(), state)[0])
    want = M.kept_norm(x.detach().reshape(-1, 40), weight.detach(), 1e-5, 0.4, g.reshape(-1, 40))
    for name, got in (("grad_x", grads[1].reshape(-1, 40)), ("grad_weight", grads[2]), ("grad_bias", grads[3])):
        value, bound = want[name]
        O.close(name, got, value, bound + O.U * value.abs())
    y = J.layer_norm(x, saved="e4m3", implementation=mode)
    assert torch.equal(y, F.layer_norm(x, (40,))) and torch.autograd.grad(y.sum(), x)[0].shape == x.shape


def test_gradients_against_differences():
    """Each gradient is the derivative of the layer's formula at what was kept, taken by differences of it in 64 bits."""
    import jakal_net as J

    x = _rand(1, 5, 64).requires_grad_()
    k = M.quantize(x, "e4m3")[0]
    got, = torch.autograd.grad(J.gelu(x, saved="e4m3").sum(), x)
    h = 1e-5
    gelu = lambda t: t * torch.special.ndtr(t)
    # the third derivative of x Phi(x) is below 2; h^2 / 6 of it, and the fp32 gradient's own error
    assert float((got.double() - (gelu(k + h) - gelu(k - h)) / (2 * h)).abs().max()) < 2 * h * h / 6 + 1e-9 + 40 * O.U
    # the loss of a norm that keeps its input is linear in h's part: differences of the plain norm where nothing rounds
    v = torch.zeros(2, 32)
    v[0, ::2], v[0, 1::2] = 1.5, -1.5  # centred, and whole numbers of the format
    v[1, ::2], v[1, 1::2] = 0.75, -0.75
    v.requires_grad_()
    g = _rand(2, 2, 32)
    kept, = torch.autograd.grad(J.layer_norm(v, saved="e4m3"), v, g)
    plain, = torch.autograd.grad(F.layer_norm(v.double(), (32,)), v, g.double())
    assert float((kept - plain).abs().max()) < 64 * O.U * float(g.abs().max())


def test_modules_and_the_model():
    import jakal_net as J
    from jakal_net.progressive import ProgressiveBConfig, ProgressiveBStep, train_step

    torch.manual_seed(0)
    a, b = torch.nn.Linear(12, 5), J.Linear(12, 5)
    assert isinstance(b, torch.nn.Linear) and list(a.state_dict()) == list(b.state_dict())
    b.load_state_dict(a.state_dict())
    x = torch.randn(3, 12)
    assert torch.equal(a(x), b(x)) and torch.equal(J.GELU()(x), F.gelu(x))
    mx = J.MXLinear.from_linear(a)
    assert list(mx.state_dict()) == ["codes", "scales", "bias"] and not list(mx.parameters())
    assert torch.equal(mx(x), J.mx_linear(x, J.mx_quantize(a.weight.detach(), "e2m1"), a.bias.detach()))
    assert J.MXLinear.from_linear(torch.nn.Linear(12, 5, bias=False))(x.bfloat16()).dtype is torch.bfloat16
    assert J.LayerNorm(12, saved="e4m3").saved == "e4m3" and J.LayerNorm(12).saved is None

    cfg = ProgressiveBConfig(vocab=97, dim=32, prefix=48, query=8, rank=8, topk=4, s_window=6, warmup=1, blocks=2,
                             expanded=24, compressed=8, refine=1, query_refine=2)
    g = torch.Generator().manual_seed(3)
    prefix, target = (torch.randint(0, 96, (2, n), generator=g) for n in (48, 8))
    models, grads = [], []
    for saved in (None, "e4m3"):
        torch.manual_seed(4)
        model = ProgressiveBStep(cfg, implementation="streaming", activations=saved)
        loss = model(prefix, target)
        loss.backward()
        models.append((model, loss.detach()))
        grads.append([p.grad.clone() if p.grad is not None else None for p in model.parameters()])
    assert list(models[0][0].state_dict()) == list(models[1][0].state_dict())
    assert torch.equal(models[0][1], models[1][1])  # the forward is the same
    kept = torch.cat([p.reshape(-1) for p in grads[1] if p is not None])
    plain = torch.cat([p.reshape(-1) for p in grads[0] if p is not None])
    assert kept.shape == plain.shape and not torch.equal(kept, plain) and bool(torch.isfinite(kept).all())
    assert float(F.cosine_similarity(kept, plain, dim=0)) > 0.9  # rounding to three bits turns no gradient round
    opt = torch.optim.SGD(models[1][0].parameters(), lr=0.1)
    train_step(models[1][0], opt, prefix, target, max_norm=1.0)
    model = models[0][0].quantize_head(activations="e2m1").quantize_head()
    assert [type(m).__name__ for m in model.head] == ["MXLinear", "GELU", "MXLinear"]
    assert model.head[0].activations == "e2m1"
    plain = models[1][0].quantize_head()
    with pytest.raises(RuntimeError, match="quantized already"):
        plain.quantize_head(activations="e2m1")
    s = model.encode_prefix(prefix)
    assert model.query_logits(s, target).shape == (2, 8, 97)
    with pytest.raises(ValueError):
        ProgressiveBStep(cfg, activations="e5m2")


def test_refusals():
    import jakal_net as J

    x, w = torch.randn(3, 64), J.mx_quantize(torch.randn(5, 64), "e2m1")
    for call in (lambda: J.mx_quantize(x, "int8"), lambda: J.mx_linear(x, J.mx_quantize(torch.randn(5, 64))),
                 lambda: J.mx_linear(x, w, activations="e4m3"), lambda: J.linear(x, torch.randn(5, 64), saved="e2m1"),
                 lambda: J.gelu(x, saved="fp8"), lambda: J.layer_norm(x, saved="e5m2"), lambda: J.GELU(saved="x"),
                 lambda: J.stabilize(x[:, 0], x, saved=""), lambda: J.Linear(3, 4, saved="e2m1"),
                 lambda: J.Linear(3, 4, implementation="fast"), lambda: J.LayerNorm(4, saved="e2m1"),
                 lambda: J.MXTensor(w.codes, w.scales, "e2m1", 65), lambda: J.MXTensor(w.codes, w.scales, "e4m3", 64),
                 lambda: J.MXTensor(w.codes.int(), w.scales, "e2m1", 64), lambda: J.MXTensor(w.codes[1:], w.scales, "e2m1", 64),
                 lambda: J.MXLinear(J.mx_quantize(torch.randn(5, 64)))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: J.mx_linear(torch.randn(3, 65), w), lambda: J.mx_linear(x, w, torch.randn(4)),
                 lambda: J.mx_quantize(torch.randn(3, 0))):
        with pytest.raises(RuntimeError):
            call()


def test_native_module_refuses_host_tensors_and_types():
    import jakal_net_native as jn

    x, u8 = torch.randn(3, 64), torch.uint8
    codes, scales = torch.zeros(3, 32, dtype=u8), torch.zeros(3, 2, dtype=u8)
    for call in (lambda: jn.mx_quantize(x, "e4m3"), lambda: jn.gelu_saved(x), lambda: jn.linear_saved(x, x),
                 lambda: jn.mx_dequantize(codes, scales, "e2m1", 64), lambda: jn.mx_linear(x, codes, scales),
                 lambda: jn.layer_norm_saved(x), lambda: jn.stabilize_saved(x[:, 0], x)):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()
    for call in (lambda: jn.mx_quantize(x.double(), "e4m3"), lambda: jn.gelu_saved(x.double()),
                 lambda: jn.layer_norm_saved(x.long())):
        with pytest.raises(NotImplementedError):
            call()
    for call in (lambda: jn.mx_quantize(x, "e5m2"), lambda: jn.mx_linear(x, codes, scales, None, "e4m3")):
        with pytest.raises(ValueError):
            call()
    for op in ("mx_quantize", "mx_dequantize", "mx_linear", "linear_saved", "gelu_saved", "layer_norm_saved",
               "stabilize_saved"):
        assert op in jn.supported_ops() and hasattr(torch.ops.jakal_net_hip, op)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fake_tensors(dtype):
    import jakal_net as J

    with FakeTensorMode():
        x = torch.empty(4, 7, 50, device="cuda", dtype=dtype, requires_grad=True)
        q = J.mx_quantize(x, "e4m3")
        assert q.codes.shape == (4, 7, 64) and q.scales.shape == (4, 7, 2) and q.codes.dtype is torch.uint8
        assert J.mx_dequantize(q).shape == x.shape and J.mx_dequantize(q).dtype is dtype
        w = J.mx_quantize(torch.empty(9, 50, device="cuda"), "e2m1")
        assert w.codes.shape == (9, 32)
        y = J.mx_linear(x, w)
        assert y.shape == (4, 7, 9) and y.dtype is dtype and y.requires_grad
        weight = torch.empty(9, 50, device="cuda", dtype=dtype, requires_grad=True)
        assert J.linear(x, weight, saved="e4m3").shape == (4, 7, 9) and J.gelu(x, saved="e4m3").shape == x.shape
        t, y = J.stabilize(torch.empty(4, 7, device="cuda"), x, saved="e4m3")
        assert t.shape == (4, 7) and y.shape == x.shape and y.requires_grad and not t.requires_grad
        for call in (lambda: J.linear(x, weight[:, 1:], saved="e4m3"), lambda: J.linear(x, weight.double(), saved="e4m3"),
                     lambda: J.linear(x, weight, weight[1], saved="e4m3"), lambda: J.gelu(x.double(), saved="e4m3"),
                     lambda: J.gelu(torch.empty(3, 0, device="cuda"), saved="e4m3"),
                     lambda: J.mx_linear(x, w, torch.empty(9, device="cuda", dtype=torch.float64))):
            with pytest.raises(RuntimeError):
                call()


def _lib():
    import jakal_net_native as jn

    return jn._LIB


def test_c_abi_checks():
    """Every call below fails before it reads a pointer."""
    lib, p, odd = _lib(), ctypes.c_void_p(4096), ctypes.c_void_p(4104)

    def quantize(x=p, rows=4, dim=64, kind=0, form=0, codes=p, scales=p):
        return lib.jn_mx_quantize(x, rows, dim, kind, form, codes, scales, None)

    for bad in (dict(x=None), dict(rows=0), dict(dim=0), dict(dim=1 << 31), dict(rows=1 << 40), dict(kind=3),
                dict(form=2), dict(form=-1), dict(codes=None), dict(scales=None), dict(codes=odd)):
        assert quantize(**bad) == 1, bad
    assert lib.jn_mx_dequantize(p, p, 4, 64, 5, 0, p, None) == 1 and lib.jn_mx_dequantize(None, p, 4, 64, 0, 0, p, None) == 1

    sizes = lib.jn_mx_linear_forward_workspace_bytes
    assert sizes(0, 64, 8, 0, -1) == 0 and sizes(16, 64, 8, 0, 1) == 0  # few rows need none
    assert sizes(65, 64, 8, 1, 1) >= 65 * 32 + 65 * 2

    def forward(x=p, w=p, ws=p, rows=80, dim=256, out=64, kind=1, acts=1, y=p, work=p, count=1 << 30):
        return lib.jn_mx_linear_forward(x, w, ws, None, rows, dim, out, kind, acts, y, work, count, None)

    for bad in (dict(x=None), dict(w=None), dict(ws=None), dict(y=None), dict(rows=0), dict(rows=1 << 31), dict(dim=0),
                dict(dim=1 << 24), dict(out=0), dict(out=1 << 24), dict(kind=9), dict(acts=0), dict(acts=2),
                dict(w=odd), dict(y=odd), dict(ws=ctypes.c_void_p(4097))):
        assert forward(**bad) == 1, bad
    for bad in (dict(work=None), dict(work=odd), dict(count=sizes(80, 256, 64, 1, 1) - 1)):
        assert forward(**bad) == 4, bad

    def backward(g=p, w=p, s=p, rows=300, dim=256, out=16384, kind=0, gx=p, work=p, count=1 << 40):
        return lib.jn_mx_linear_backward(g, w, s, rows, dim, out, kind, gx, work, count, None)

    need = lib.jn_mx_linear_backward_workspace_bytes(300, 256, 16384, 0)
    assert need > 0
    for bad in (dict(g=None), dict(w=None), dict(s=None), dict(gx=None), dict(rows=0), dict(kind=3), dict(w=odd), dict(gx=odd)):
        assert backward(**bad) == 1, bad
    for bad in (dict(work=None), dict(work=odd), dict(count=need - 1)):
        assert backward(**bad) == 4, bad

    def weight(g=p, c=p, s=p, rows=4096, dim=256, out=64, kind=1, gw=p, gb=p, work=p, count=1 << 40):
        return lib.jn_mx_weight_grad(g, c, s, rows, dim, out, kind, gw, gb, work, count, None)

    need = lib.jn_mx_weight_grad_workspace_bytes(4096, 256, 64, 1, 1)
    assert need > lib.jn_mx_weight_grad_workspace_bytes(4096, 256, 64, 1, 0) > 0
    for bad in (dict(g=None), dict(c=None), dict(s=None), dict(gw=None), dict(dim=0), dict(kind=-1), dict(c=odd), dict(gw=odd)):
        assert weight(**bad) == 1, bad
    for bad in (dict(work=None), dict(count=need - 1)):
        assert weight(**bad) == 4, bad

    fits = lib.jn_linear_input_grad_fits
    assert fits(1024, 2048, 16384, 1) == 1 and fits(1024, 2048, 16384, 0) == 0 and fits(1, 8, 8, 1) == 0
    assert fits(1024, 2048, 16380, 1) == 0 and fits(-1, 2048, 16384, 1) == 0
    assert lib.jn_linear_input_grad(p, p, 4, 64, 64, 1, p, p, 1 << 30, None) == 2  # left to the library
    assert lib.jn_linear_input_grad(None, p, 1024, 2048, 16384, 1, p, p, 1 << 40, None) == 1
    assert lib.jn_linear_input_grad(p, p, 1024, 2048, 16384, 1, p, None, 0, None) == 4
    assert lib.jn_column_sums(None, 4, 8, 0, p, p, 1 << 20, None) == 1
    assert lib.jn_column_sums(p, 4, 8, 0, p, p, lib.jn_column_sums_workspace_bytes(4, 8) - 1, None) == 4

    for bad in (dict(x=None), dict(y=None), dict(codes=None), dict(scales=None), dict(codes=odd), dict(dim=0)):
        a = dict(x=p, y=p, codes=p, scales=p, dim=64) | bad
        assert lib.jn_gelu_forward(a["x"], 4, a["dim"], 0, a["y"], a["codes"], a["scales"], None) == 1, bad
    for at in range(4):
        a = [p, p, p, p]
        a[at] = None
        assert lib.jn_gelu_backward(a[0], a[1], a[2], 4, 64, 0, a[3], None) == 1

    def norm(x=p, codes=p, scales=p, rows=4, dim=64, kind=0):
        return lib.jn_layer_norm_forward_kept(None, x, None, None, rows, dim, 1.0, 1e-5, kind, 0, kind, None, p, p, codes,
                                              scales, None)

    assert norm(rows=0) == 0
    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(codes=odd), dict(dim=0), dict(kind=4)):
        assert norm(**bad) == 1, bad
    for codes, scales in ((None, p), (p, None), (odd, p)):
        assert lib.jn_layer_norm_backward_kept(None, codes, scales, None, p, None, p, 4, 64, 1.0, 0, 0, 0, None, p, None,
                                               None, None, 0, None) == 1
