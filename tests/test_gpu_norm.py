"""Layer norm and the layer update's stabilisation on the HIP library against
their definitions in float64 (tests/step_oracle.py): widths from one element to
several workgroup strides, odd widths, rows that start off 16 bytes, every
type, each gradient alone, rows that hold infinities, captured steps."""

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu

DIMS = [1, 2, 7, 8, 32, 64, 65, 200, 256, 383, 512, 520, 1000, 1024, 1536, 2048, 2050, 4096, 4100, 5003, 8192, 16384,
        20011, 33000]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


def _made(dev, rows, dim, dtype, params, affine="both", seed=0, offset=0):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 101 + dim)

    def rand(*shape, scale=1.0, mean=0.0, kind=dtype):
        flat = torch.randn(offset + int(torch.tensor(shape).prod()), generator=g) * scale + mean
        return flat.to(kind).to(dev)[offset:].view(shape)

    x, gy = rand(rows, dim, scale=1.3, mean=0.4), rand(rows, dim)
    weight = rand(dim, scale=0.2, mean=1.0, kind=params) if affine in ("both", "weight") else None
    bias = rand(dim, scale=0.3, kind=params) if affine in ("both", "bias") else None
    return x, gy, weight, bias


def _check(what, names, got, want, dtypes):
    for name, tensor, dtype in zip(names, got, dtypes):
        value, bound = want[name]
        assert tensor.dtype is dtype, f"{what} {name}: {tensor.dtype}"
        O.close(f"{what} {name}", tensor, value, bound + O.half(dtype) * value.abs() + O.floor(dtype))


def _norm_case(dev, rows, dim, dtype, params, affine="both", offset=0, eps=1e-5):
    import jakal_net as J

    x, gy, weight, bias = _made(dev, rows, dim, dtype, params, affine, offset=offset)
    leaves = [t.requires_grad_() for t in (x.detach(), *(p.detach() for p in (weight, bias) if p is not None))]
    ws = {n: t for n, t in zip([n for n, p in (("w", weight), ("b", bias)) if p is not None], leaves[1:])}
    y = J.layer_norm(leaves[0], ws.get("w"), ws.get("b"), eps=eps)
    grads = torch.autograd.grad(y, leaves, gy)
    names = ["y", "grad_x"] + [n for n, p in (("grad_weight", weight), ("grad_bias", bias)) if p is not None]
    want = O.norm(x, weight, bias, eps, 1.0, gy)
    _check(f"norm {rows}x{dim} {dtype}", names, [y, *grads], want, [dtype, dtype] + [params] * (len(names) - 2))


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_widths(dev, dim, dtype):
    _norm_case(dev, 37 if dim < 5000 else 5, dim, O.DTYPES[dtype], O.DTYPES[dtype])


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 257, 1031, 4099])
@pytest.mark.parametrize("dim", [48, 512, 1536])
def test_row_counts(dev, rows, dim):
    _norm_case(dev, rows, dim, torch.float32, torch.float32)
    _norm_case(dev, rows, dim, torch.bfloat16, torch.float32)


@pytest.mark.parametrize("rows", [3, 15, 33, 255, 2047, 2049, 9001])
@pytest.mark.parametrize("dim", [8, 60, 64, 128, 130, 200, 1000, 3000, 8000])
def test_groups_that_end_inside_a_workgroup(dev, rows, dim):
    """Rows that do not fill the last workgroup's groups, few and many, for each number of threads a row."""
    if rows * dim <= 1 << 24:
        _norm_case(dev, rows, dim, torch.float32, torch.float32)
        _norm_case(dev, rows, dim + 1, torch.bfloat16, torch.bfloat16)
        _norm_case(dev, rows, dim, torch.float16, torch.float32)


@pytest.mark.parametrize("affine", ["both", "weight", "bias", "none"])
@pytest.mark.parametrize("dim", [100, 512, 4096, 9000])
def test_parameters_left_out(dev, dim, affine):
    _norm_case(dev, 19, dim, torch.float16, torch.float32, affine)


@pytest.mark.parametrize("dtype", list(O.DTYPES))
@pytest.mark.parametrize("dim", [64, 512, 2048, 8192])
def test_rows_that_start_off_16_bytes(dev, dim, dtype):
    _norm_case(dev, 33, dim, O.DTYPES[dtype], O.DTYPES[dtype], offset=1)


def test_offset_far_above_the_spread(dev):
    """A mean a thousand times the deviation: the centred pass keeps the digits that x has."""
    import jakal_net as J

    g = torch.Generator().manual_seed(3)
    x = (torch.randn(11, 512, generator=g) + 1000.0).to(dev)
    want = O.norm(x, None, None, 1e-5)
    _check("far mean", ["y"], [J.layer_norm(x)], want, [torch.float32])


def test_constant_rows_and_one_column(dev):
    import jakal_net as J

    x = torch.full((4, 96), 3.0, device=dev)
    b = torch.arange(96.0, device=dev)
    assert torch.equal(J.layer_norm(x, None, b), b.expand(4, 96))
    one = torch.randn(5, 1, device=dev)
    assert torch.equal(J.layer_norm(one), torch.zeros_like(one))


@pytest.mark.parametrize("shape", [(0, 16), (3, 0, 16), (2, 3, 1, 24), (8,)])
def test_batch_shapes(dev, shape):
    import jakal_net as J

    x = torch.randn(shape, device=dev, requires_grad=True)
    w = torch.randn(shape[-1], device=dev, requires_grad=True)
    y = J.layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert y.shape == gx.shape == x.shape and gw.shape == w.shape
    if not x.numel():
        assert not gw.any()
        return
    flat = x.detach().reshape(-1, shape[-1])
    want = O.norm(flat, w.detach(), None, 1e-5, 1.0, torch.ones_like(flat))
    _check("shape", ["y", "grad_x"], [y.reshape(flat.shape), gx.reshape(flat.shape)], want, [torch.float32] * 2)


def test_stabilize_without_rows(dev):
    import jakal_net as J

    s = torch.randn(2, 0, device=dev, requires_grad=True)
    x = torch.randn(2, 0, 12, device=dev, requires_grad=True)
    w, b = (torch.ones(12, device=dev, requires_grad=True) for _ in range(2))
    t, y = J.stabilize(s, x, w, b, scale=0.5)
    gs, gx, gw, gb = torch.autograd.grad([t, y], [s, x, w, b], [torch.ones_like(t), torch.ones_like(y)])
    assert t.shape == gs.shape == (2, 0) and y.shape == gx.shape == (2, 0, 12)
    assert not gw.any() and not gb.any()


@pytest.mark.parametrize("kinds", [("bf16", "fp32", "bf16"), ("fp32", "bf16", "fp32"), ("fp16", "bf16", "fp32")])
def test_parameters_of_other_types(dev, kinds):
    """Weight and bias of types of their own are taken in fp32, their gradients come back in their types."""
    import jakal_net as J

    kx, kw, kb = (O.DTYPES[k] for k in kinds)
    x, gy, weight, bias = _made(dev, 21, 72, kx, torch.float32)
    leaves = [t.to(k).requires_grad_() for t, k in ((x, kx), (weight, kw), (bias, kb))]
    y = J.layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, gy)
    want = O.norm(*(t.detach() for t in leaves), 1e-5, 1.0, gy)
    _check(f"types {kinds}", ["y", "grad_x", "grad_weight", "grad_bias"], [y, *grads], want, [kx, kx, kw, kb])


def test_strided_inputs_and_expanded_gradients(dev):
    import jakal_net as J

    base = torch.randn(40, 6, 30, device=dev)
    x = base.transpose(0, 1)[:, ::2].requires_grad_()
    y = J.layer_norm(x)
    (gx,) = torch.autograd.grad(y, x, torch.ones(1, 1, 30, device=dev).mul(0.5).expand(y.shape))
    flat = x.detach().reshape(-1, 30)
    want = O.norm(flat, None, None, 1e-5, 1.0, torch.full_like(flat, 0.5))
    _check("strided", ["y", "grad_x"], [y.reshape(-1, 30), gx.reshape(-1, 30)], want, [torch.float32] * 2)


@pytest.mark.parametrize("dim", [64, 200, 1024, 6000])
@pytest.mark.parametrize("which", ["state", "val", "weight", "bias", "state,weight", "val,bias"])
def test_each_gradient_alone(dev, which, dim):
    import jakal_net as J

    x, gy, weight, bias = _made(dev, 29, dim, torch.float32, torch.float32)
    s, gs = torch.randn(29, device=dev), torch.randn(29, device=dev)
    t = dict(state=s, val=x, weight=weight, bias=bias)
    full = {n: v.clone().requires_grad_() for n, v in t.items()}
    part = {n: v.clone().requires_grad_(n in which.split(",")) for n, v in t.items()}
    want = dict(zip(full, torch.autograd.grad(J.stabilize(**full, scale=0.3), list(full.values()), [gs, gy])))
    names = which.split(",")
    ends, seeds = zip(*[(e, g) for e, g in zip(J.stabilize(**part, scale=0.3), (gs, gy)) if e.requires_grad])
    got = torch.autograd.grad(ends, [part[n] for n in names], seeds, allow_unused=True)
    for n, v in zip(names, got):
        assert torch.equal(v, want[n]), n


def test_an_output_that_nothing_uses(dev):
    import jakal_net as J

    s = torch.randn(3, 9, device=dev, requires_grad=True)
    x = torch.randn(3, 9, 40, device=dev, requires_grad=True)
    w = torch.ones(40, device=dev, requires_grad=True)
    t, y = J.stabilize(s, x, w)
    gs, gx, gw = torch.autograd.grad(t.sum(), [s, x, w], allow_unused=True, retain_graph=True)
    assert gx is None and gw is None and bool(gs.abs().sum() > 0)
    gs, gx = torch.autograd.grad(y.sum(), [s, x], allow_unused=True)
    assert gs is None and bool(torch.isfinite(gx).all())


@pytest.mark.parametrize("scale", [1.0, 0.0625, 0.3, -2.0, 0.0])
@pytest.mark.parametrize("dtype", list(O.DTYPES))
@pytest.mark.parametrize("dim", [96, 512, 1028])
def test_stabilize(dev, dim, dtype, scale):
    import jakal_net as J

    kind = O.DTYPES[dtype]
    x, gy, weight, bias = _made(dev, 3 * 41, dim, kind, torch.float32, seed=2)
    g = torch.Generator().manual_seed(dim)
    s = (torch.randn(3 * 41, generator=g) * 4).to(dev)
    s[:2] = torch.tensor([40.0, -90.0])
    gs = torch.randn(3 * 41, generator=g).to(dev)
    leaves = [t.view(3, 41, *t.shape[1:]).detach().requires_grad_() for t in (s, x)]
    leaves += [p.detach().requires_grad_() for p in (weight, bias)]
    t, y = J.stabilize(*leaves, scale=scale)
    grads = torch.autograd.grad([t, y], leaves, [gs.view(3, 41), gy.view(3, 41, dim)])
    scale32 = float(torch.tensor(scale))
    want = {**O.norm(x, weight, bias, 1e-5, scale32, gy), **O.state(s, scale32, gs)}
    flat = [v.reshape(-1, *v.shape[2:]) if v.dim() > 1 else v for v in (t, y, *grads)]
    _check(f"stabilize {dim} {dtype} {scale}", ["state", "y", "grad_state", "grad_x", "grad_weight", "grad_bias"], flat,
           want, [torch.float32, kind, torch.float32, kind, torch.float32, torch.float32])


@pytest.mark.parametrize("state_dtype", list(O.DTYPES))
def test_states_of_their_own_type(dev, state_dtype):
    import jakal_net as J

    kind = O.DTYPES[state_dtype]
    s = torch.randn(50, device=dev).mul(2).to(kind).requires_grad_()
    x = torch.randn(50, 64, device=dev).bfloat16()
    t, y = J.stabilize(s, x, scale=0.5)
    gs = torch.randn(50, device=dev).to(kind)
    (grad,) = torch.autograd.grad(t, s, gs)
    want = O.state(s.detach(), 0.5, gs)
    _check("state", ["state", "grad_state"], [t, grad], want, [kind, kind])
    assert torch.equal(y, J.stabilize(s.detach().float(), x, scale=0.5)[1])


@pytest.mark.parametrize("dim", [64, 383, 2048, 7000])
def test_rows_that_are_not_finite_stay_alone(dev, dim):
    import jakal_net as J

    x, gy, weight, bias = _made(dev, 12, dim, torch.float32, torch.float32)
    clean_y = J.layer_norm(x, weight, bias)
    bad = x.clone()
    bad[3, dim // 2], bad[7, 0], bad[9, -1] = float("inf"), float("nan"), float("-inf")
    leaf = bad.requires_grad_()
    y = J.layer_norm(leaf, weight, bias)
    (gx,) = torch.autograd.grad(y, leaf, gy)
    clean = x.clone().requires_grad_()
    (want,) = torch.autograd.grad(J.layer_norm(clean, weight, bias), clean, gy)
    rows = torch.tensor([r not in (3, 7, 9) for r in range(12)], device=dev)
    assert torch.equal(y[rows], clean_y[rows]) and torch.equal(gx[rows], want[rows])
    assert bool(torch.isnan(y[~rows]).any(-1).all()) and bool(torch.isnan(gx[~rows]).any(-1).all())


@pytest.mark.parametrize("dim", [96, 512])
def test_gradient_against_differences(dev, dim):
    """<grad, d> against (f(x + t d) - f(x - t d)) / 2 t of the operator itself, f the
    output times fixed weights: the difference's own error is that of the same
    quotient in float64, and the outputs' bounds over 2 t."""
    import jakal_net as J

    x, c, weight, bias = _made(dev, 7, dim, torch.float32, torch.float32)
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(9)).to(dev)
    t = 2.0 ** -6
    leaf = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(J.layer_norm(leaf, weight, bias), leaf, c)
    up, down = x + t * d, x - t * d
    got = ((J.layer_norm(up, weight, bias).double() - J.layer_norm(down, weight, bias).double()) * c).sum() / (2 * t)
    a, b = O.norm(up, weight, bias, 1e-5)["y"], O.norm(down, weight, bias, 1e-5)["y"]
    exact = ((a[0] - b[0]) * c).sum() / (2 * t)
    value, bound = O.norm(x, weight, bias, 1e-5, 1.0, c)["grad_x"]
    # up and down are rounded: their distance is 2 t d to within a rounding of x each
    slope = (value.abs() * O.U * (up.abs() + down.abs())).sum() / (2 * t)
    noise = ((a[1] + b[1] + O.U * (a[0].abs() + b[0].abs())) * c.abs()).sum() / (2 * t)
    limit = (exact - (value * d).sum()).abs() + slope + noise + ((bound + O.U * value.abs()) * d.abs()).sum()
    assert (got - (gx.double() * d).sum()).abs() <= limit
    # and the quotient is near enough the slope for this to say something
    assert limit <= 0.05 * (value * d).abs().sum()


def test_two_captured_steps_replay_as_eager(dev):
    """Two training steps in two graphs, replayed in turn with eager work between."""
    import jakal_net as J

    sizes = [(700, 512), (123, 1000)]
    made = [_made(dev, r, d, torch.float32, torch.float32, seed=4) for r, d in sizes]
    states = [torch.randn(r, device=dev) for r, _ in sizes]

    def step(x, gy, weight, bias, s):
        leaves = [t.detach().requires_grad_() for t in (s, x, weight, bias)]
        t, y = J.stabilize(*leaves, scale=0.25)
        return [t.detach(), y.detach(), *torch.autograd.grad([t, y], leaves, [torch.ones_like(t), gy])]

    want = [step(*m, s) for m, s in zip(made, states)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for m, s in zip(made, states):
            step(*m, s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for m, s in zip(made, states):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*m, s))
    for rep in range(3):
        for out in outs:
            for t in out:
                t.fill_(float("nan"))
        for graph in graphs:
            graph.replay()
        torch.randn(1 << 20, device=dev).sum()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for a, b in zip(out, w):
                assert torch.equal(a, b), f"replay {rep}"


def test_repeats_bit_for_bit_and_on_another_stream(dev):
    import jakal_net as J

    x, gy, weight, bias = _made(dev, 5000, 512, torch.bfloat16, torch.float32)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, weight, bias)]
        return torch.autograd.grad(J.layer_norm(*leaves), leaves, gy)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(want, again, step()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_more_than_2_31_elements(dev):
    """Rows beyond 2^31 elements: the last rows and the parameter gradients."""
    import jakal_net as J

    dim, rows = 1024, (1 << 21) + 3
    x = torch.empty(rows, dim, device=dev, dtype=torch.bfloat16).normal_()
    gy = torch.empty_like(x).normal_()
    w = torch.ones(dim, device=dev).requires_grad_()
    b = torch.zeros(dim, device=dev).requires_grad_()
    leaf = x.requires_grad_()
    y = J.layer_norm(leaf, w, b)
    gx, gw, gb = torch.autograd.grad(y, [leaf, w, b], gy)
    x = x.detach()
    for at in (slice(0, 5), slice(rows - 5, rows)):
        want = O.norm(x[at], w.detach(), b.detach(), 1e-5, 1.0, gy[at])
        _check("far rows", ["y", "grad_x"], [y[at], gx[at]], want, [torch.bfloat16] * 2)
    # each chunk's bounds, and the roundings of the sums over all rows (one each 64 rows and 16 of a tree)
    sums = {n: [torch.zeros(dim, device=dev, dtype=torch.float64) for _ in range(3)] for n in ("w", "b")}
    for x0, g0 in zip(x.split(1 << 17), gy.split(1 << 17)):
        part = O.norm(x0, None, None, 1e-5, 1.0, g0)
        h = part["y"][0]
        for n, key, terms in (("w", "grad_weight", g0.double() * h), ("b", "grad_bias", g0.double())):
            for total, t in zip(sums[n], (*part[key], terms.abs().sum(0))):
                total += t
    for n, got in (("w", gw), ("b", gb)):
        value, bound, size = sums[n]
        O.close("far grad " + n, got, value, bound + O.depth(rows) * O.U * size + O.U * value.abs())


def test_inputs_changed_before_the_backward_raise(dev):
    import jakal_net as J

    for which in ("val", "weight", "state"):
        t = dict(state=torch.randn(4, device=dev), val=torch.randn(4, 16, device=dev), weight=torch.ones(16, device=dev))
        leaves = {n: v.requires_grad_() for n, v in t.items()}
        used = {n: v * 1.0 for n, v in leaves.items()}
        a, b = J.stabilize(**used)
        with torch.no_grad():
            used[which].mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            (a.sum() + b.sum()).backward()
    x = torch.randn(4, 16, device=dev, requires_grad=True)
    y = J.layer_norm(x)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()


def test_pending_negations(dev):
    """Tensors whose negation torch has put off (the imaginary parts of conjugates), inputs and gradients."""
    import jakal_net as J

    _, _, weight, bias = _made(dev, 6, 40, torch.float32, torch.float32)
    x, gy = torch.randn(6, 40, device=dev), torch.randn(6, 40, device=dev)
    state, gs = torch.randn(6, device=dev), torch.randn(6, device=dev)
    results = []
    for lazy in (False, True):
        neg = torch._neg_view if lazy else torch.neg
        leaves = [t.detach().requires_grad_() for t in (state, x, weight, bias)]
        out, y = J.stabilize(*(neg(t) for t in leaves), scale=0.5)
        results.append((out, y, *torch.autograd.grad((out, y), leaves, (neg(gs), neg(gy)))))
    assert torch._neg_view(gy).is_neg() and torch._neg_view(gy).is_contiguous()
    for eager, late in zip(*results):
        assert torch.equal(eager, late)


def test_transforms(dev):
    """vmap runs it slice by slice; torch.func's gradients and forward mode raise."""
    import jakal_net as J
    from torch.autograd import forward_ad

    x = torch.randn(3, 4, 8, device=dev)
    assert torch.equal(torch.func.vmap(J.layer_norm)(x), J.layer_norm(x))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: J.layer_norm(t).pow(3).sum())(x)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(J.layer_norm, (x,), (x,))
    with pytest.raises((RuntimeError, NotImplementedError)), forward_ad.dual_level():
        J.layer_norm(forward_ad.make_dual(x, x))
    with pytest.raises((RuntimeError, NotImplementedError)):
        J.layer_norm(x[0].to_sparse())


def test_autocast_returns_fp32_rows(dev):
    import jakal_net as J

    norm = J.LayerNorm(64).to(dev)
    x = torch.randn(5, 64, device=dev).bfloat16()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert norm(x).dtype is torch.float32
        t, y = J.stabilize(torch.zeros(5, device=dev).bfloat16(), x)
        assert t.dtype is torch.bfloat16 and y.dtype is torch.float32
    assert norm(x).dtype is torch.bfloat16


def test_refusals(dev):
    import jakal_net as J
    import jakal_net_native as jn

    x = torch.randn(3, 8, device=dev)
    with pytest.raises(NotImplementedError):
        J.layer_norm(x.double())
    assert J.layer_norm(x.double(), implementation="kernel").dtype is torch.float64
    for call in (lambda: J.layer_norm(x, torch.ones(7, device=dev)), lambda: J.layer_norm(x, torch.ones(8)),
                 lambda: J.layer_norm(x, eps=-1.0), lambda: J.layer_norm(x, eps=float("nan")),
                 lambda: J.layer_norm(torch.randn(3, 0, device=dev)), lambda: J.layer_norm(torch.tensor(1.0, device=dev)),
                 lambda: J.stabilize(torch.randn(4, device=dev), x), lambda: J.stabilize(torch.randn(3), x),
                 lambda: J.LayerNorm(9).to(dev)(x), lambda: jn.layer_norm(torch.randn(3, 8))):
        with pytest.raises(RuntimeError):
            call()
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(J.layer_norm(leaf).pow(2).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
