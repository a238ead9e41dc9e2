"""The vocabulary loss on the HIP library against its definition in float64
(tests/step_oracle.py): class counts from one to a large odd vocabulary, every
type and reduction, ignored and out-of-range targets, masked (-inf), infinite
and NaN logits, rows that start off 16 bytes, captured steps."""

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu

CLASSES = [1, 2, 3, 31, 64, 65, 97, 200, 512, 1000, 1024, 1031, 2048, 4099, 8192, 16384, 16381, 40000, 65537, 131071]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


def _made(dev, rows, classes, dtype, seed=0, offset=0, scale=2.5):
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + classes)
    z = (torch.randn(offset + rows * classes, generator=g) * scale).to(dtype).to(dev)[offset:].view(rows, classes)
    return z, torch.randint(0, classes, (rows,), generator=g).to(dev)


def _case(dev, z, target, reduction="mean", g=None, ignore=-100, what=""):
    import jakal_net as J

    leaf = z.detach().requires_grad_()
    loss = J.cross_entropy(leaf, target, ignore_index=ignore, reduction=reduction)
    (grad,) = torch.autograd.grad(loss, leaf, g)
    want = O.cross_entropy(z.detach(), target, ignore, reduction, g)
    assert loss.dtype is torch.float32 and grad.dtype is z.dtype
    value, bound = want["loss"]
    O.close(f"{what} loss", loss, value, bound + O.U * value.abs())
    value, bound = want["grad"]
    O.close(f"{what} grad", grad, value, bound + O.half(z.dtype) * value.abs() + O.floor(z.dtype))
    return loss.detach(), grad


@pytest.mark.parametrize("classes", CLASSES)
@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_class_counts(dev, classes, dtype):
    z, t = _made(dev, 37 if classes < 20000 else 5, classes, O.DTYPES[dtype])
    _case(dev, z, t, what=f"{classes} {dtype}")


@pytest.mark.parametrize("rows", [1, 2, 15, 17, 63, 64, 65, 257, 1031, 5000])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_and_reductions(dev, rows, reduction):
    z, t = _made(dev, rows, 130, torch.float32)
    t[rows // 3:rows // 2] = -100
    g = torch.randn(rows, device=dev) if reduction == "none" else torch.tensor(1.7, device=dev)
    _case(dev, z, t, reduction, g, what=f"{rows} {reduction}")


@pytest.mark.parametrize("dtype", list(O.DTYPES))
@pytest.mark.parametrize("classes", [64, 1024, 16384])
def test_rows_that_start_off_16_bytes(dev, classes, dtype):
    z, t = _made(dev, 9, classes, O.DTYPES[dtype], offset=1)
    _case(dev, z, t, what=f"offset {classes}")


@pytest.mark.parametrize("classes", [50, 4099, 16384])
def test_ignored_rows_hold_anything(dev, classes):
    """Ignored rows of NaN and infinity reach neither the loss nor the gradient."""
    z, t = _made(dev, 12, classes, torch.float32)
    t[2], t[5], t[11] = -100, -100, -100
    clean = _case(dev, z, t)
    z[2], z[5], z[11, 0] = float("nan"), float("inf"), float("-inf")
    import jakal_net as J

    leaf = z.requires_grad_()
    loss = J.cross_entropy(leaf, t)
    (grad,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(loss, clean[0]) and torch.equal(grad, clean[1])
    assert not grad[[2, 5, 11]].any()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_nothing_counts(dev, reduction):
    import jakal_net as J

    z = torch.randn(4, 33, device=dev, requires_grad=True)
    loss = J.cross_entropy(z, torch.full((4,), 7, device=dev), ignore_index=7, reduction=reduction)
    assert bool(torch.isnan(loss)) if reduction == "mean" else not loss.any()
    (grad,) = torch.autograd.grad(loss.sum(), z)
    assert not grad.any()
    none = torch.randn(0, 33, device=dev, requires_grad=True)
    loss = J.cross_entropy(none, torch.zeros(0, dtype=torch.int64, device=dev), reduction=reduction)
    assert loss.shape == ((0,) if reduction == "none" else ())
    assert torch.autograd.grad(loss.sum(), none)[0].shape == (0, 33)


@pytest.mark.parametrize("classes", [96, 1024, 4099, 16384])
def test_targets_outside_the_classes(dev, classes):
    z, t = _made(dev, 8, classes, torch.float32)
    t[1], t[4], t[6] = classes, -1, 1 << 40
    loss, grad = _case(dev, z, t, "none", torch.ones(8, device=dev), what="outside")
    assert bool(torch.isnan(loss[[1, 4, 6]]).all()) and bool(torch.isnan(grad[[1, 4, 6]]).all())


@pytest.mark.parametrize("classes", [70, 1024, 4099, 16384])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_masked_logits(dev, classes, dtype):
    """-inf and the type's lowest value in masked classes; all but one class masked."""
    z, t = _made(dev, 6, classes, O.DTYPES[dtype])
    z[0, ::2], t[0] = float("-inf"), 1
    z[1, 1:] = float("-inf")
    t[1] = 0
    z[2, : classes // 2], t[2] = torch.finfo(z.dtype).min, classes - 1
    z[3, 1::3], t[3] = float("-inf"), 1  # the target is masked: the loss is infinite
    import jakal_net as J

    leaf = z.requires_grad_()
    loss = J.cross_entropy(leaf, t, reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    want = O.cross_entropy(z.detach()[[0, 1, 2, 4, 5]], t[[0, 1, 2, 4, 5]], reduction="none")
    keep = [0, 1, 2, 4, 5]
    O.close("masked loss", loss[keep], want["loss"][0], want["loss"][1])
    O.close("masked grad", grad[keep], want["grad"][0],
            want["grad"][1] + O.half(z.dtype) * want["grad"][0].abs() + O.floor(z.dtype))
    loss = loss.detach()
    assert float(loss[3]) == float("inf") and bool(torch.isfinite(grad[3]).all()) and float(grad[3, 1]) == -1.0
    assert float(loss[1]) == 0.0 and not grad[1].any()


@pytest.mark.parametrize("classes", [70, 4099])
def test_rows_that_are_not_finite_stay_alone(dev, classes):
    import jakal_net as J

    z, t = _made(dev, 9, classes, torch.float32)
    clean = J.cross_entropy(z, t, reduction="none")
    z[2, classes // 2], z[4], z[7, 0] = float("nan"), float("-inf"), float("inf")
    loss = J.cross_entropy(z, t, reduction="none")
    rows = torch.tensor([0, 1, 3, 5, 6, 8], device=dev)
    assert torch.equal(loss[rows], clean[rows])
    assert bool(torch.isnan(loss[[2, 4, 7]]).all())


def test_large_logits_keep_their_differences(dev):
    """Logits around 1e4: the loss keeps the digits that their differences have."""
    z, t = _made(dev, 20, 300, torch.float32)
    _case(dev, (z + 1.0e4), t, "none", torch.ones(20, device=dev), what="large")
    _case(dev, z * 1.0e4, t, "none", torch.ones(20, device=dev), what="wide")


@pytest.mark.parametrize("kind", ["int32", "strided", "batch", "transposed"])
def test_layouts(dev, kind):
    import jakal_net as J

    z, t = _made(dev, 24, 60, torch.float32)
    want = J.cross_entropy(z, t, reduction="none")
    if kind == "int32":
        got = J.cross_entropy(z, t.int(), reduction="none")
    elif kind == "batch":
        got = J.cross_entropy(z.view(2, 3, 4, 60), t.view(2, 3, 4), reduction="none").reshape(24)
    elif kind == "strided":
        wide = torch.stack([t, t + 5], dim=1)[:, 0]
        got = J.cross_entropy(torch.cat([z, z], dim=1)[:, :60], wide, reduction="none")
    else:
        got = J.cross_entropy(z.t().contiguous().t(), t, reduction="none")
    assert torch.equal(got, want)


def test_one_row_without_axes(dev):
    import jakal_net as J

    z, t = _made(dev, 3, 40, torch.float32)
    loss = J.cross_entropy(z[1], t[1], reduction="none")
    assert loss.shape == () and torch.equal(loss, J.cross_entropy(z, t, reduction="none")[1])
    assert torch.equal(J.cross_entropy(z[1], t[1]), loss)


def test_backward_twice_and_scaled(dev):
    import jakal_net as J

    z, t = _made(dev, 10, 5000, torch.float32)
    leaf = z.requires_grad_()
    loss = J.cross_entropy(leaf, t)
    (one,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (two,) = torch.autograd.grad(loss, leaf, torch.tensor(2.0, device=dev), retain_graph=True)
    (again,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(one, again) and torch.equal(two, 2 * one)


def test_pending_negations(dev):
    """Logits whose negation torch has put off, and a loss's gradient that comes through a conjugate."""
    import jakal_net as J

    z, t = _made(dev, 9, 70, torch.float32)
    results = []
    for lazy in (False, True):
        leaf = z.detach().requires_grad_()
        loss = J.cross_entropy(torch._neg_view(leaf) if lazy else -leaf, t)
        whole = torch.complex(torch.zeros_like(loss), loss)
        part = whole.conj().imag if lazy else -whole.imag
        results.append((loss, *torch.autograd.grad(part, leaf)))
    for eager, late in zip(*results):
        assert torch.equal(eager, late)
    want = O.cross_entropy(-z, t, -100, "mean", None)["grad"]  # (of the logits; minus for the leaf, minus for the part)
    O.close("grad", results[1][1], want[0], want[1] + O.U * want[0].abs() + O.floor(torch.float32))


def test_gradient_against_differences(dev):
    """<grad, d> against the loss's own quotient of differences over 2 t."""
    import jakal_net as J

    z, t = _made(dev, 6, 203, torch.float32)
    d = torch.randn(z.shape, generator=torch.Generator().manual_seed(8)).to(dev)
    step = 2.0 ** -6
    leaf = z.clone().requires_grad_()
    (grad,) = torch.autograd.grad(J.cross_entropy(leaf, t, reduction="sum"), leaf)
    up, down = z + step * d, z - step * d
    sums = [J.cross_entropy(v, t, reduction="none").double() for v in (up, down)]
    got = (sums[0] - sums[1]).sum() / (2 * step)
    a, b = (O.cross_entropy(v, t, reduction="none")["loss"] for v in (up, down))
    value, bound = O.cross_entropy(z, t, reduction="sum")["grad"]
    exact = (a[0] - b[0]).sum() / (2 * step)
    noise = (a[1] + b[1]).sum() / (2 * step) + (value.abs() * O.U * (up.abs() + down.abs())).sum() / (2 * step)
    limit = (exact - (value * d).sum()).abs() + noise + ((bound + O.U * value.abs()) * d.abs()).sum()
    assert (got - (grad.double() * d).sum()).abs() <= limit
    assert limit <= 0.05 * (value * d).abs().sum()


def test_two_captured_steps_replay_as_eager(dev):
    import jakal_net as J

    made = [_made(dev, 130, 16384, torch.bfloat16), _made(dev, 77, 1001, torch.float32)]
    made[0][1][::5] = -100

    def step(z, t):
        leaf = z.detach().requires_grad_()
        loss = J.cross_entropy(leaf, t)
        return [loss.detach(), *torch.autograd.grad(loss, leaf)]

    want = [step(*m) for m in made]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for m in made:
            step(*m)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for m in made:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*m))
    for rep in range(3):
        for out in outs:
            for v in out:
                v.fill_(float("nan"))
        for graph in graphs:
            graph.replay()
        torch.randn(1 << 20, device=dev).sum()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for a, b in zip(out, w):
                assert torch.equal(a, b), f"replay {rep}"


@pytest.mark.parametrize("rows,classes", [(1030, 1100), (1024, 2048), (1500, 4096), (1201, 4099), (1025, 8192),
                                          (511, 9000), (513, 9000)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_rows(dev, rows, classes, dtype):
    z, t = _made(dev, rows, classes, O.DTYPES[dtype], seed=3)
    t[::7] = -100
    _case(dev, z, t, what=f"{rows}x{classes} {dtype}")


@pytest.mark.parametrize("rows,classes", [((1 << 15) + 9, 65537), (200003, 1000), (100003, 2047)])
def test_more_logits_than_the_cache_or_31_bits(dev, rows, classes):
    import jakal_net as J

    z = torch.empty(rows, classes, device=dev, dtype=torch.bfloat16).normal_(std=2.0)
    t = torch.randint(0, classes, (rows,), device=dev)
    leaf = z.requires_grad_()
    loss = J.cross_entropy(leaf, t, reduction="none")
    (grad,) = torch.autograd.grad(loss, leaf, torch.ones(rows, device=dev))
    for at in (slice(0, 3), slice(rows - 3, rows)):
        want = O.cross_entropy(z.detach()[at], t[at], reduction="none")
        O.close("far loss", loss[at], *want["loss"])
        O.close("far grad", grad[at], want["grad"][0], want["grad"][1] + O.half(z.dtype) * want["grad"][0].abs()
                + O.floor(z.dtype))


def test_refusals(dev):
    import jakal_net as J
    import jakal_net_native as jn

    z, t = _made(dev, 4, 10, torch.float32)
    with pytest.raises(NotImplementedError):
        J.cross_entropy(z.double(), t)
    assert J.cross_entropy(z.double(), t, implementation="kernel").dtype is torch.float64
    for call in (lambda: J.cross_entropy(z, t[:3]), lambda: J.cross_entropy(z, t.float()),
                 lambda: J.cross_entropy(z, t, reduction="max"), lambda: J.cross_entropy(z, t.cpu()),
                 lambda: J.cross_entropy(torch.randn(4, 0, device=dev), t), lambda: jn.cross_entropy(z.cpu(), t.cpu())):
        with pytest.raises(RuntimeError):
            call()
    leaf = z.requires_grad_()
    (g,) = torch.autograd.grad(J.cross_entropy(leaf, t), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
