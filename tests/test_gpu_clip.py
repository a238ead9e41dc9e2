"""The gradients' global norm and clipping on the HIP library against float64:
lists longer than a launch takes, empty and scalar tensors, every mix of types,
unaligned views, in place and into other buffers, infinities and NaN, captured
calls, and the whole step of the Progressive-B model."""

import math

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


SHAPES = [(3, 5), (), (0, 4), (1,), (4096,), (4097,), (64, 513), (255,), (2, 3, 4, 5), (70001,)]


def _list(dev, shapes, dtypes, seed=0, scale=0.01, offset=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, s in enumerate(shapes):
        flat = torch.randn(offset + math.prod(s), generator=g) * scale
        out.append(flat.to(dtypes[i % len(dtypes)]).to(dev)[offset:].view(s))
    return out


def _norm_bound(want):
    return (3 * O.U) * want + 1e-45


def _check(grads, out, norm, max_norm, kind=2.0, what=""):
    """out and norm against the definition; grads: the values before."""
    want = O.grads_norm(grads, kind)
    assert norm.dtype is torch.float32 and norm.shape == ()
    assert abs(float(norm) - want) <= _norm_bound(want), f"{what} norm {float(norm)} for {want}"
    factor = min(1.0, max_norm / (want + 1e-6))
    for g, o in zip(grads, out):
        value = g.double() * factor
        # the factor and the product round to fp32, the result to its type
        O.close(f"{what} {tuple(g.shape)}", o, value,
                value.abs() * (4 * O.U + O.half(o.dtype)) + O.floor(o.dtype))


@pytest.mark.parametrize("kind", [2.0, float("inf")])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("limit", [0.25, 4.0, 0.0, float("inf")])
def test_in_place(dev, dtype, kind, limit):
    import jakal_net as J

    dtypes = list(O.DTYPES.values()) if dtype == "mixed" else [O.DTYPES[dtype]]
    grads = _list(dev, SHAPES, dtypes)
    before = [g.clone() for g in grads]
    max_norm = limit * O.grads_norm(before, kind) if math.isfinite(limit) else limit
    norm = J.clip_grads(grads, max_norm, kind)
    if limit > 1.0:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        max_norm = 1e30
    _check(before, grads, norm, max_norm, kind, dtype)
    assert torch.equal(J.grad_norm(before, kind), norm)


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtype", list(O.DTYPES))
@pytest.mark.parametrize("out_dtype", list(O.DTYPES))
def test_into_other_buffers(dev, dtype, out_dtype, offset):
    import jakal_net as J

    grads = _list(dev, SHAPES, [O.DTYPES[dtype]], seed=2, offset=offset)
    for limit in (0.3, 3.0):
        # guard elements around every output stay as they were
        pads = [torch.full((g.numel() + 2 + offset,), 7.0, device=dev, dtype=O.DTYPES[out_dtype]) for g in grads]
        out = [p[1 + offset:1 + offset + g.numel()].view(g.shape) for p, g in zip(pads, grads)]
        before = [g.clone() for g in grads]
        max_norm = limit * O.grads_norm(grads)
        norm = J.clip_grads(grads, max_norm, out=out)
        _check(before, out, norm, max_norm, 2.0, f"{dtype} to {out_dtype}")
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        assert all(bool((p[:1 + offset] == 7).all()) and float(p[-1]) == 7.0 for p in pads)


@pytest.mark.parametrize("phase", [(0, 0), (1, 1), (3, 3), (5, 1), (2, 6), (7, 7), (1, 0), (4, 4)])
@pytest.mark.parametrize("dtype,out_dtype", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp16")])
def test_views_of_flat_buffers(dev, dtype, out_dtype, phase):
    """Gradients and outputs as unpadded views of two flat buffers, at any element of them."""
    import jakal_net as J

    sizes = [5, 8192, 3, 8193, 1, 2, 20001, 16384, 7]
    g = torch.Generator().manual_seed(6)
    total = sum(sizes)
    flat = (torch.randn(total + 8, generator=g) * 0.01).to(O.DTYPES[dtype]).to(dev)[phase[0]:phase[0] + total]
    out = torch.full((total + 16,), 7.0, device=dev, dtype=O.DTYPES[out_dtype])
    grads, outs = list(flat.split(sizes)), list(out[phase[1] + 1:phase[1] + 1 + total].split(sizes))
    max_norm = 0.3 * O.grads_norm(grads)
    _check(grads, outs, J.clip_grads(grads, max_norm, out=outs), max_norm, 2.0, f"phase {phase}")
    assert bool((out[:phase[1] + 1] == 7).all()) and bool((out[phase[1] + 1 + total:] == 7).all())
    before = [t.clone() for t in grads]
    _check(before, grads, J.clip_grads(grads, max_norm), max_norm, 2.0, f"phase {phase} in place")


@pytest.mark.parametrize("count", [1, 139, 140, 141, 163, 164, 165, 300, 1000])
def test_long_lists(dev, count):
    import jakal_net as J

    shapes = [((i * 37) % 900 + 1,) for i in range(count)]
    grads = _list(dev, shapes, [torch.float32, torch.bfloat16], seed=3)
    before = [g.clone() for g in grads]
    max_norm = 0.5 * O.grads_norm(before)
    _check(before, grads, J.clip_grads(grads, max_norm), max_norm, 2.0, f"{count} tensors")


@pytest.mark.parametrize("sizes", [(9_000_000, 17, 9_000_001), (30_000_003,)])
def test_large_tensors(dev, sizes):
    import jakal_net as J

    grads = [torch.empty(n, device=dev).normal_(std=1e-3) for n in sizes]
    before = [g.clone() for g in grads]
    max_norm = 0.5 * O.grads_norm(before)
    norm = J.clip_grads(grads, max_norm)
    _check(before, grads, norm, max_norm, 2.0, "large")
    # the sum has one order: the same list gives the same norm bit for bit
    assert torch.equal(J.grad_norm(before), norm) and torch.equal(J.grad_norm(before), norm)


def test_more_than_2_31_elements(dev):
    import jakal_net as J

    n = (1 << 31) + 4101
    g = torch.zeros(n, device=dev, dtype=torch.bfloat16)
    g[0], g[1 << 31], g[-1] = 3.0, 4.0, 12.0
    norm = J.clip_grads([g], 1.3)
    assert float(norm) == 13.0
    got = [float(g[i]) for i in (0, 1 << 31, n - 1)]
    assert got == pytest.approx([0.3, 0.4, 1.2], rel=2 ** -8 + 1e-6)
    assert float(J.grad_norm([g], float("inf"))) == got[2]


def test_squares_beyond_fp32(dev):
    import jakal_net as J

    g = torch.tensor([3.0e25, 4.0e25], device=dev)
    assert float(J.clip_grads([g], 10.0)) == pytest.approx(5.0e25, rel=1e-6)
    assert g.tolist() == pytest.approx([6.0, 8.0], rel=1e-6)
    tiny = torch.tensor([3.0e-25, 4.0e-25], device=dev)
    assert float(J.grad_norm(tiny)) == pytest.approx(5.0e-25, rel=1e-6)


@pytest.mark.parametrize("kind", [2.0, float("inf")])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_not_finite(dev, bad, kind):
    """An infinite norm scales by 0 (and makes its infinities NaN), a NaN one makes all NaN."""
    import jakal_net as J

    g = [torch.ones(5000, device=dev), torch.ones(7, device=dev)]
    g[0][4500] = bad
    p = [torch.nn.Parameter(torch.zeros_like(t)) for t in g]
    for q, t in zip(p, g):
        q.grad = t.clone()
    with pytest.raises(RuntimeError, match="cannot be clipped"):
        J.clip_grad_norm_(p, 1.0, kind, error_if_nonfinite=True)
    assert all(torch.equal(q.grad.nan_to_num(2.0), t.nan_to_num(2.0)) for q, t in zip(p, g))
    norm = J.clip_grad_norm_(p, 1.0, kind)
    if math.isnan(bad):
        assert math.isnan(float(norm)) and all(bool(torch.isnan(q.grad).all()) for q in p)
    else:
        assert float(norm) == float("inf") and not p[1].grad.any()
        assert int(torch.isnan(p[0].grad).sum()) == 1 and float(p[0].grad.nan_to_num().abs().sum()) == 0.0


def test_parameters(dev):
    import jakal_net as J

    shared = torch.nn.Parameter(torch.zeros(300, device=dev))
    other = torch.nn.Parameter(torch.zeros(20, 30, device=dev))
    idle = torch.nn.Parameter(torch.zeros(5, device=dev))
    shared.grad, other.grad = torch.randn(300, device=dev), torch.randn(20, 30, device=dev)
    before = [shared.grad.clone(), other.grad.clone()]
    version = shared.grad._version
    norm = J.clip_grad_norm_([shared, other, idle, shared], 1.0)
    _check(before, [shared.grad, other.grad], norm, 1.0)
    assert shared.grad._version > version and idle.grad is None
    want = torch.nn.utils.clip_grad_norm_([torch.nn.Parameter(b) for b in before], 1.0)  # no gradients: 0
    assert float(J.clip_grad_norm_([idle], 1.0)) == float(want) == 0.0
    assert float(J.grad_norm([])) == 0.0 and float(J.grad_norm([torch.zeros(0, device=dev)])) == 0.0


def test_orders_of_axes(dev):
    """Transposed gradients are scaled where they are; other strides are copied or refused."""
    import jakal_net as J

    g = torch.randn(30, 40, device=dev).t()
    before = g.clone()
    _check([before], [g], J.clip_grads([g], 2.0), 2.0)
    out = torch.empty(40, 30, device=dev)
    g = torch.randn(30, 40, device=dev).t()
    _check([g], [out], J.clip_grads([g], 2.0, out=[out]), 2.0)
    turned = torch.empty(30, 40, device=dev).t()
    _check([g], [turned], J.clip_grads([g], 2.0, out=[turned]), 2.0)
    _check([out], [turned], J.clip_grads([out], 1.0, out=[turned]), 1.0)
    wide = torch.randn(40, 60, device=dev)
    _check([wide[:, ::2]], [out], J.clip_grads([wide[:, ::2]], 2.0, out=[out]), 2.0)
    for bad in (wide[:, ::2], torch.randn(1, 60, device=dev).expand(40, 60)):
        with pytest.raises(NotImplementedError):
            J.clip_grads([bad], 2.0)


def test_two_captured_calls_replay_as_eager(dev):
    import jakal_net as J

    lists = [_list(dev, SHAPES * 20, [torch.float32, torch.bfloat16], seed=5), _list(dev, SHAPES, [torch.float32])]
    outs = [[torch.empty(g.shape, device=dev) for g in grads] for grads in lists]
    want = []
    for grads, out in zip(lists, outs):
        norm = J.clip_grads(grads, 0.01, out=out)
        want.append([norm.clone()] + [o.clone() for o in out])
    torch.cuda.synchronize()
    graphs, norms = [], []
    for grads, out in zip(lists, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            norms.append(J.clip_grads(grads, 0.01, out=out))
    for rep in range(3):
        for out in outs:
            for o in out:
                o.fill_(float("nan"))
        for graph in graphs:
            graph.replay()
        torch.randn(1 << 20, device=dev).sum()
        torch.cuda.synchronize()
        for w, norm, out in zip(want, norms, outs):
            assert all(torch.equal(a, b) for a, b in zip(w, [norm] + out)), f"replay {rep}"


def test_pending_negations(dev):
    """Tensors whose negation torch has put off are refused, and taken once it is carried out."""
    import jakal_net as J

    a, b = torch.randn(50, device=dev), torch.empty(50, device=dev)
    late, before = torch._neg_view(a), a.clone()
    for call in (lambda: J.grad_norm([late]), lambda: J.clip_grads([late], 1.0),
                 lambda: J.clip_grads([late], 1.0, out=[b]), lambda: J.clip_grads([b.fill_(2.0)], 1.0, out=[late])):
        with pytest.raises(NotImplementedError):
            call()
        assert torch.equal(a, before)
    J.clip_grads([late.resolve_neg()], float("inf"), out=[b])
    assert torch.equal(b, -a)


def test_refusals(dev):
    import jakal_net as J

    a, b = torch.randn(50, device=dev), torch.randn(100, device=dev)
    value, runtime, limits = ValueError, RuntimeError, NotImplementedError
    for error, call in (
            (value, lambda: J.clip_grads([a], -1.0)), (value, lambda: J.clip_grads([a], float("nan"))),
            (value, lambda: J.clip_grads([a], 1.0, out=[a, b])), (value, lambda: J.clip_grads([a], 1.0, out=[b])),
            (value, lambda: J.clip_grads([a], 1.0, out=[None])),
            (value, lambda: J.clip_grads([a], 1.0, out=[torch.zeros(50, device=dev, requires_grad=True)])),
            (limits, lambda: J.clip_grads([a], 1.0, 1.0)), (limits, lambda: J.grad_norm([a.double()])),
            (limits, lambda: J.grad_norm([a.to_sparse()])),
            (runtime, lambda: J.clip_grads([a, b.cpu()], 1.0)),
            # shared memory: a tensor twice, an output over another gradient, halves that overlap
            (runtime, lambda: J.clip_grads([a, a], 1.0)), (runtime, lambda: J.clip_grads([a, a[3:20]], 1.0)),
            (runtime, lambda: J.clip_grads([b[:50], b[50:]], 1.0, out=[b[50:], b[:50]])),
            (runtime, lambda: J.clip_grads([b[:50]], 1.0, out=[b[1:51]])),
            (runtime, lambda: J.clip_grads([b[:50]], 1.0, out=[b[:50].view(torch.bfloat16)[:50]]))):
        before = (a.clone(), b.clone())
        with pytest.raises(error):
            call()
        assert torch.equal(a, before[0]) and torch.equal(b, before[1])
    # reading a tensor twice, and two halves of one buffer, are ordinary
    assert float(J.grad_norm([a, a])) == pytest.approx(math.sqrt(2) * float(J.grad_norm([a])), rel=1e-6)
    J.clip_grads([b[:50], b[50:]], 1.0)
    assert float(J.grad_norm(b)) == pytest.approx(1.0, rel=1e-5)
