"""Microscaled tensors, products by 4-bit weights and layers that keep their inputs
in 8 bits on the HIP library, against tests/mx_oracle.py in float64: every format
and type, lengths from one element, runs and tiles that end inside, rows off 16
bytes, infinities and NaN, each gradient alone."""

import ctypes

import pytest
import torch

import mx_oracle as M
import step_oracle as O

pytestmark = pytest.mark.gpu

TYPES = list(O.DTYPES)
FORMS = ["e4m3", "e2m1"]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


def _rand(seed, *shape, scale=1.0, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * scale
    return x * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g)) if spread else x


def _rounded(what, got, want, dtype):
    value, bound = want
    assert got.dtype is dtype, f"{what}: {got.dtype}"
    O.close(what, got, value, bound + O.half(dtype) * value.abs() + O.floor(dtype))


def _quantized(what, x, form):
    import jakal_net as J

    q = J.mx_quantize(x, form)
    value, code, scale = M.quantize(x, form)
    assert torch.equal(q.scales.cpu().long(), scale.long()), f"{what}: scales"
    assert torch.equal(q.codes.cpu(), M.packed(code, form)), f"{what}: codes"
    for dtype in (torch.float32, x.dtype):
        back = J.mx_dequantize(q, dtype)
        assert back.dtype is dtype and back.shape == x.shape
        same = (back.cpu() == value.to(dtype)) | (torch.isnan(back.cpu()) & torch.isnan(value))
        assert bool(same.all()), f"{what}: values"
    return q


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 7, 8, 31, 32, 33, 64, 100, 383, 512, 1000, 2048])
def test_quantize_widths(dev, dim, dtype, form):
    for rows in (1, 3, 67):
        x = _rand(dim * 7 + rows, rows, dim, spread=3.0).to(O.DTYPES[dtype]).to(dev)
        _quantized(f"{form} {dtype} {rows}x{dim}", x, form)


@pytest.mark.parametrize("form", FORMS)
def test_quantize_every_border(dev, form):
    """Every magnitude, the middles between two and their neighbours, at several scales, as the
    second of two whose first fixes the scale."""
    grid = M.magnitudes(form).float()
    middle = (grid[1:] + grid[:-1]) / 2
    points = torch.cat([grid, middle, torch.nextafter(middle, torch.tensor(0.0)),
                        torch.nextafter(middle, torch.tensor(1e9))])
    points = torch.cat([points, -points])
    x = torch.zeros(len(points), 32)
    x[:, 0], x[:, 1] = grid[-1], points
    _quantized("borders", torch.cat([x * 2.0 ** k for k in (-100, -3, 0, 60)]).to(dev), form)


@pytest.mark.parametrize("form", FORMS)
def test_quantize_extremes(dev, form):
    inf, nan = float("inf"), float("nan")
    x = _rand(5, 12, 70)
    x[0] = 0.0
    x[1, 3] = inf
    x[2, 40], x[2, 41] = nan, -inf
    x[3] = 3.4e38
    x[4] = 1e-40
    x[5] = 1.4e-45
    x[6, 0], x[6, 33] = 448.0, 449.0
    x[7, 0], x[7, 33] = 6.0, 6.0000005
    x[8] = -0.0
    x[9, ::2] = 1e30
    x[10] *= 2.0 ** -120
    _quantized("extremes fp32", x.to(dev), form)
    _quantized("extremes bf16", x.bfloat16().to(dev), form)
    _quantized("extremes fp16", x.half().to(dev), form)


@pytest.mark.parametrize("form", FORMS)
def test_quantize_views_and_empties(dev, form):
    import jakal_net as J

    x = _rand(9, 6, 5, 64).to(dev)
    for view in (x[:, :, 1:50], x.transpose(0, 1), x[::2], x.reshape(-1)[1:1 + 320].view(5, 64), x[0, 0]):
        _quantized("view", view, form)
    q = J.mx_quantize(x[:0], form)
    assert q.shape == (0, 5, 64) and J.mx_dequantize(q).shape == (0, 5, 64)


def _weight(dev, out, dim, seed):
    import jakal_net as J

    w = _rand(seed, out, dim, scale=dim ** -0.5)
    return J.mx_quantize(w.to(dev), "e2m1"), M.quantize(w, "e2m1")[0]


def _mx_case(dev, rows, dim, out, dtype, acts, bias=True, train=True, seed=1):
    import jakal_net as J

    kind = O.DTYPES[dtype]
    weight, w = _weight(dev, out, dim, seed)
    x = _rand(seed + 1, rows, dim).to(kind)
    g = _rand(seed + 2, rows, out, spread=0.0).to(kind)
    b = _rand(seed + 3, out, spread=0.0).to(kind) if bias else None
    xd = x.to(dev).requires_grad_(train)
    bd = None if b is None else b.to(dev).requires_grad_(train)
    y = J.mx_linear(xd, weight, bd, activations=acts)
    what = f"mx_linear {dtype} {acts} {rows}x{dim}x{out}"
    _rounded(what, y, M.product(x if acts is None else M.quantize(x, acts)[0], w.t(), b), kind)
    if train:
        grads = torch.autograd.grad(y, [xd] if b is None else [xd, bd], g.to(dev))
        _rounded(what + " grad_x", grads[0], M.product(g, w), kind)
        if b is not None:
            _rounded(what + " grad_bias", grads[1], M.sums(g), kind)


@pytest.mark.parametrize("acts", [None, "e2m1"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,out", [(1, 32, 16), (1, 1, 1), (2, 33, 5), (3, 64, 128), (17, 96, 130), (64, 512, 256),
                                          (127, 100, 129), (128, 256, 128), (129, 383, 257), (300, 288, 514)])
def test_mx_linear(dev, rows, dim, out, dtype, acts):
    _mx_case(dev, rows, dim, out, dtype, acts, bias=rows % 2 == 1)


@pytest.mark.parametrize("rows,dim,out", [(1, 2048, 4100), (5, 4099, 1000), (16, 8192, 512), (40, 1024, 3001), (700, 2048, 90),
                                          (2050, 64, 700)])
def test_mx_linear_long(dev, rows, dim, out):
    _mx_case(dev, rows, dim, out, "bf16", "e2m1")
    _mx_case(dev, rows, dim, out, "fp32", None, bias=False)
    _mx_case(dev, rows, dim, out, "fp16", None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("rows,dim,out", [(1, 1, 1), (1, 32, 8), (2, 33, 65), (31, 64, 128), (65, 96, 130), (130, 383, 257),
                                          (1000, 40, 24), (64, 512, 1000), (257, 128, 384)])
def test_linear_saved(dev, rows, dim, out, bias, dtype):
    import jakal_net as J

    kind = O.DTYPES[dtype]
    x, w = _rand(1, rows, dim).to(kind), _rand(2, out, dim, scale=dim ** -0.5, spread=0.0).to(kind)
    b = _rand(3, out, spread=0.0).to(kind) if bias else None
    g = _rand(4, rows, out, spread=0.0).to(kind)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, *((b,) if bias else ()))]
    y = J.linear(*leaves, saved="e4m3")
    plain = torch.nn.functional.linear(*leaves)
    assert torch.equal(y, plain)  # the forward is the plain layer's
    grads = torch.autograd.grad(y, leaves, g.to(dev))
    what = f"linear {dtype} {rows}x{dim}x{out}"
    _rounded(what + " grad_x", grads[0], M.product(g, w), kind)
    _rounded(what + " grad_weight", grads[1], M.product(g.t(), M.quantize(x, "e4m3")[0]), kind)
    if bias:
        _rounded(what + " grad_bias", grads[2], M.sums(g), kind)


@pytest.mark.parametrize("rows,dim,out", [(256, 256, 16384), (300, 520, 16392), (1024, 256, 4104), (8, 2048, 131072)])
def test_linear_saved_wide_tiles(dev, rows, dim, out):
    """bf16 sums over many outputs, split over workgroups: the input gradient's wide tiles, whole and ragged."""
    import jakal_net as J

    x, w = _rand(1, rows, dim).bfloat16(), _rand(2, out, dim, scale=dim ** -0.5, spread=0.0).bfloat16()
    g = _rand(4, rows, out, spread=0.0).bfloat16()
    xd = x.to(dev).requires_grad_()
    gx, = torch.autograd.grad(J.linear(xd, w.to(dev).requires_grad_(), saved="e4m3"), xd, g.to(dev))
    _rounded(f"linear {rows}x{dim}x{out} grad_x", gx, M.product(g, w), torch.bfloat16)


@pytest.mark.parametrize("rows,dim,out", [(512, 4096, 4096), (520, 4104, 4360), (2048, 1000, 16384)])
def test_products_of_wide_tiles(dev, rows, dim, out):
    """bf16 outputs of many wide tiles, whole and ragged: forward, input gradient and weight gradient."""
    import jakal_net as J

    weight, w = _weight(dev, out, dim, 3)
    x, g = _rand(1, rows, dim).bfloat16(), _rand(2, rows, out, spread=0.0).bfloat16()
    b = _rand(3, out, spread=0.0).bfloat16()
    xd, gd = x.to(dev).requires_grad_(), g.to(dev)
    w, gs, xs = w.to(dev), gd.double(), x.to(dev).double()
    for acts in (None, "e2m1"):
        y = J.mx_linear(xd, weight, b.to(dev), activations=acts)
        a = xs if acts is None else M.quantize(x, acts)[0].to(dev)
        _rounded(f"{acts} y", y, M.product(a, w.t(), b.to(dev)), torch.bfloat16)
    gx, = torch.autograd.grad(y, xd, gd)
    _rounded("grad_x", gx, M.product(gs, w), torch.bfloat16)
    codes, scales = torch.ops.jakal_net_hip.mx_codes(x.to(dev), 0)
    gw, gb = torch.ops.jakal_net_hip.mx_weight_grad(gd, codes, scales, dim, True)
    _rounded("grad_weight", gw, M.product(gs.t(), M.quantize(x, "e4m3")[0].to(dev)), torch.bfloat16)
    _rounded("grad_bias", gb, M.sums(gs), torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,out", [(100, 300, 700), (300, 100, 9000), (600, 72, 20000)])
def test_mx_linear_every_tile(dev, rows, dim, out, dtype):
    """Both operands e2m1: tiles of 64, 128 and 256."""
    _mx_case(dev, rows, dim, out, dtype, "e2m1")


# (tiles of 64 x 64, 128 x 64, 128 x 128 and 256 x 256, each with a whole sum and with a split one)
@pytest.mark.parametrize("m,n,r", [(72, 72, 72), (72, 72, 520), (200, 16392, 72), (72, 520, 16392), (1544, 2056, 72),
                                   (72, 1000, 8200), (1000, 8200, 72), (152, 4104, 8200), (72, 72, 128), (136, 520, 8192),
                                   (200, 16390, 256), (1536, 2056, 384)])
def test_products_of_every_tile(dev, m, n, r):
    """bf16 outputs [m, n] of sums over r: forward, input gradient and weight gradient with its bias."""
    import jakal_net as J

    ops = torch.ops.jakal_net_hip
    x, g, a = _rand(1, m, r).bfloat16().to(dev), _rand(2, m, r, spread=0.0).bfloat16().to(dev), _rand(4, r, m).bfloat16().to(dev)
    weight, w = _weight(dev, n, r, 3)
    b = _rand(3, n, spread=0.0).bfloat16().to(dev)
    _rounded("y", J.mx_linear(x, weight, b), M.product(x, w.to(dev).t(), b), torch.bfloat16)
    weight, w = _weight(dev, r, n, 5)
    _rounded("grad_x", ops.mx_input_grad(g, weight.codes, weight.scales, n), M.product(g, w.to(dev)), torch.bfloat16)
    kept = _rand(6, r, n).bfloat16()
    gw, gb = ops.mx_weight_grad(a, *ops.mx_codes(kept.to(dev), 0), n, True)
    _rounded("grad_weight", gw, M.product(a.t(), M.quantize(kept, "e4m3")[0].to(dev)), torch.bfloat16)
    _rounded("grad_bias", gb, M.sums(a), torch.bfloat16)


@pytest.mark.parametrize("rows,dim,out", [(16, 8, 8), (33, 1000, 256), (72, 72, 512), (72, 520, 16392), (200, 16392, 72),
                                          (1544, 2056, 72), (64, 1000, 8200), (1, 520, 16384), (2000, 4104, 136)])
def test_linear_saved_input_grads(dev, rows, dim, out):
    """The input gradient's own products of bf16: short sums and long ones, every tile, whole and split."""
    import jakal_net_native as jn

    i64 = ctypes.c_int64
    assert ctypes.CDLL(str(jn.library_path())).jn_linear_input_grad_fits(i64(rows), i64(dim), i64(out), 1) == 1
    g, w = _rand(1, rows, out, spread=0.0).bfloat16().to(dev), _rand(2, out, dim, spread=0.0).bfloat16().to(dev)
    got = torch.ops.jakal_net_hip.linear_input_grad(g, w)
    _rounded(f"{rows}x{dim}x{out}", got, M.product(g, w), torch.bfloat16)
    loose = torch.empty(out, dim + 1, dtype=torch.bfloat16, device=dev)[:, 1:]
    loose.copy_(w)
    assert torch.equal(torch.ops.jakal_net_hip.linear_input_grad(g, loose), got)


@pytest.mark.parametrize("rows", [4096, 10007])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_saved_many_rows(dev, rows, dtype):
    """Sums over rows that are split over workgroups."""
    import jakal_net as J

    kind = O.DTYPES[dtype]
    x, g = _rand(1, rows, 72).to(kind), _rand(4, rows, 136, spread=0.0).to(kind)
    w, b = torch.zeros(136, 72, dtype=kind, device=dev).requires_grad_(), torch.zeros(136, dtype=kind, device=dev).requires_grad_()
    gw, gb = torch.autograd.grad(J.linear(x.to(dev), w, b, saved="e4m3"), [w, b], g.to(dev))
    _rounded("grad_weight", gw, M.product(g.t(), M.quantize(x, "e4m3")[0]), kind)
    _rounded("grad_bias", gb, M.sums(g), kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 7, 32, 33, 100, 512, 2048])
def test_gelu_saved(dev, dim, dtype):
    import jakal_net as J

    kind = O.DTYPES[dtype]
    for rows in (1, 5, 130):
        x, g = _rand(dim + rows, rows, dim, scale=2.0).to(kind), _rand(3, rows, dim, spread=0.0).to(kind)
        xd = x.to(dev).requires_grad_()
        y = J.gelu(xd, saved="e4m3")
        _rounded(f"gelu {dtype} {rows}x{dim}", y, M.gelu(x), kind)
        assert torch.equal(y.detach(), J.gelu(xd.detach(), saved="e4m3"))
        got, = torch.autograd.grad(y, xd, g.to(dev))
        _rounded(f"gelu {dtype} {rows}x{dim} grad", got, M.gelu_slope(M.quantize(x, "e4m3")[0], g), kind)


NORM_DIMS = [1, 2, 7, 8, 32, 33, 64, 65, 100, 200, 383, 512, 520, 1000, 1536, 2050, 4096, 4100, 8192, 16384, 20011]


def _norm_case(dev, rows, dim, kind, params, affine=2, scale=0.3, state=True, offset=0):
    import jakal_net as J

    def put(t, k):
        flat = torch.zeros(offset + t.numel(), dtype=k, device=dev)
        flat[offset:] = t.reshape(-1).to(dev)
        return flat[offset:].view(t.shape)

    x, g = (_rand(dim + rows, rows, dim, scale=1.3, spread=0.3) + 0.3).to(kind), _rand(2, rows, dim, spread=0.0).to(kind)
    w = (1 + 0.2 * _rand(3, dim, spread=0.0)).to(params) if affine else None
    b = _rand(4, dim, spread=0.0).to(params) if affine > 1 else None
    s, gs = _rand(5, rows, spread=0.0).to(kind), _rand(6, rows, spread=0.0).to(kind)
    xd, sd = put(x, kind).requires_grad_(), s.to(dev).requires_grad_()
    ps = [put(p, params).requires_grad_() for p in (w, b) if p is not None]
    args = ps + [None] * (2 - len(ps))
    t, y = J.stabilize(sd, xd, *args, scale=scale, saved="e4m3")
    want = J.stabilize(sd, xd, *args, scale=scale)
    assert torch.equal(t, want[0]) and torch.equal(y, want[1])
    grads = torch.autograd.grad([t, y], [sd, xd, *ps], [gs.to(dev), g.to(dev)])
    plain = torch.autograd.grad(want[0], sd, gs.to(dev))[0]
    assert torch.equal(grads[0], plain)
    bounds = M.kept_norm(x, w, 1e-5, scale, g)
    what = f"norm {rows}x{dim} {kind}"
    for name, got, k in zip(("grad_x", "grad_weight", "grad_bias"), grads[1:], (kind, params, params)):
        _rounded(f"{what} {name}", got, bounds[name], k)
    if scale == 1.0:
        assert torch.equal(J.layer_norm(xd, *args, saved="e4m3"), y)


@pytest.mark.parametrize("dim", NORM_DIMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_saved(dev, dim, dtype):
    kind = O.DTYPES[dtype]
    _norm_case(dev, 37 if dim < 5000 else 5, dim, kind, kind)
    _norm_case(dev, 3, dim, kind, torch.float32, affine=dim % 3, scale=1.0)
    _norm_case(dev, 5, dim, kind, kind, offset=1)


@pytest.mark.parametrize("rows", [1, 2, 63, 257, 2047, 9001])
@pytest.mark.parametrize("dim", [48, 130, 512])
def test_norm_saved_rows(dev, rows, dim):
    _norm_case(dev, rows, dim, torch.float32, torch.float32)
    _norm_case(dev, rows, dim, torch.bfloat16, torch.float32)


def test_norm_keeps_what_quantize_gives(dev):
    """The norm's own kernels and mx_quantize agree on every run, non-finite ones among them."""
    for dim in NORM_DIMS:
        for kind in O.DTYPES.values():
            x = _rand(dim, 9, dim, spread=2.0)
            x[2, dim // 2], x[5, 0] = float("inf"), float("nan")
            x = x.to(kind).to(dev)
            y, *rest = torch.ops.jakal_net_hip.kept_norm_forward(None, x, None, None, 1e-5, 1.0)[1:]
            codes, scales = torch.ops.jakal_net_hip.mx_codes(M.centred(x), 0)
            assert torch.equal(rest[1], codes) and torch.equal(rest[2], scales), f"{dim} {kind}"
