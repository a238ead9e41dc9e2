"""Operators on microscaled numbers as programs use them: under autocast, in
torch.compile and captured graphs, on side streams, with views and saved-tensor
hooks, in the Progressive-B step and its 4-bit head."""

import pytest
import torch
from torch.nn import functional as F

import mx_oracle as M
import step_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


def _leaves(dev, rows, dim, hidden, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev)

    return [t.requires_grad_() for t in (rand(rows), rand(rows, dim), rand(dim, scale=0.2), rand(dim),
                                         rand(hidden, dim, scale=dim ** -0.5), rand(hidden))]


def _block(state, val, weight, bias, w, b, q):
    """An update, a head's first layer and activation, and a frozen 4-bit layer behind them."""
    import jakal_net as J

    t, y = J.stabilize(state, val, weight, bias, scale=0.5, saved="e4m3")
    h = J.gelu(J.linear(y, w, b, saved="e4m3"), saved="e4m3")
    return t, J.mx_linear(h, q, activations="e2m1"), J.mx_linear(h, q)


def _step(leaves, q, run=_block):
    outs = run(*leaves, q)
    return [*outs, *torch.autograd.grad(outs, leaves, [torch.full_like(o, 0.5) for o in outs])]


def _frozen(dev, out, dim, seed=9):
    import jakal_net as J

    w = torch.randn(out, dim, generator=torch.Generator().manual_seed(seed)) * dim ** -0.5
    return J.mx_quantize(w.to(dev), "e2m1")


@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_together(dev, dtype):
    """The operators one behind the other, as a head with an update before it: each gradient is what the next one's
    formula makes of it in float64, at the values that were kept."""
    import jakal_net as J

    kind = O.DTYPES[dtype]
    leaves, q = _leaves(dev, 70, 96, 160, kind), _frozen(dev, 200, 160)
    state, val, weight, bias, w, b = leaves
    t, y = J.stabilize(state, val, weight, bias, scale=0.5, saved="e4m3")
    h = J.linear(y, w, b, saved="e4m3")
    a = J.gelu(h, saved="e4m3")
    out = J.mx_linear(a, q)
    g = torch.randn(out.shape, generator=torch.Generator().manual_seed(4)).to(kind).to(dev)
    ga, gh, gy = torch.autograd.grad(out, [a, h, y], g, retain_graph=True)
    gw, gb, gv = torch.autograd.grad(out, [w, b, val], g)
    wq = J.mx_dequantize(q).double()
    kept = lambda x: M.quantize(x, "e4m3")[0].to(dev)
    for name, got, (value, bound) in (
            ("out", out, M.product(a.detach(), wq.t())), ("grad_a", ga, M.product(g, wq)),
            ("grad_h", gh, M.gelu_slope(kept(h), ga)), ("grad_w", gw, M.product(gh.t(), kept(y))),
            ("grad_b", gb, M.sums(gh)), ("grad_y", gy, M.product(gh, w.detach())),
            ("grad_val", gv, [x.to(dev) for x in M.kept_norm(val.detach().cpu(), weight.detach().cpu(), 1e-5, 0.5,
                                                             gy.cpu())["grad_x"]])):
        O.close(f"{dtype} {name}", got, value, bound + O.half(kind) * value.abs() + O.floor(kind))


def test_repeats_bit_for_bit_and_on_another_stream(dev):
    leaves, q = _leaves(dev, 3000, 256, 520, torch.bfloat16), _frozen(dev, 1000, 520)
    want = _step(leaves, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _step(leaves, q)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_two_captured_steps_replay_as_eager(dev):
    """Two steps of other sizes in two graphs, replayed in turn with new inputs and eager work between."""
    sizes = [(300, 256, 512), (77, 100, 136)]
    made = [_leaves(dev, *s, torch.bfloat16, seed=i) for i, s in enumerate(sizes)]
    frozen = [_frozen(dev, 264, s[2]) for s in sizes]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for m, q in zip(made, frozen):
            _step(m, q)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for m, q in zip(made, frozen):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_step(m, q))
    for rep in range(4):
        with torch.no_grad():
            for m in made:
                m[1].copy_(torch.randn(m[1].shape, generator=torch.Generator().manual_seed(50 + rep)))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for m, q, out in zip(made, frozen, outs):
            fresh = [t.detach().clone().requires_grad_() for t in m]
            for a, b in zip(out, _step(fresh, q)):
                assert torch.equal(a, b), f"replay {rep}"


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled(dev, backend):
    leaves, q = _leaves(dev, 37, 64, 96, torch.float32), _frozen(dev, 40, 96)
    torch._dynamo.reset()
    compiled = torch.compile(_block, backend=backend, fullgraph=True)
    for a, b in zip(_step(leaves, q, compiled), _step(leaves, q)):
        assert a.dtype is b.dtype and torch.equal(a, b)
    torch._dynamo.reset()


def test_autocast(dev):
    import jakal_net as J

    _, x, _, _, w, b = _leaves(dev, 20, 64, 96, torch.float32)
    q = _frozen(dev, 40, 96)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        h = J.linear(x, w, b, saved="e4m3")
        y = J.mx_linear(h, q, torch.zeros(40, device=dev))
    assert h.dtype is torch.bfloat16 and y.dtype is torch.bfloat16
    want = J.linear(x.bfloat16(), w.bfloat16(), b.bfloat16(), saved="e4m3")
    assert torch.equal(h, want)
    for a, c in zip(torch.autograd.grad(h.float().sum(), [x, w, b]), torch.autograd.grad(want.float().sum(), [x, w, b])):
        assert a.dtype is torch.float32 and torch.equal(a, c)
    norm = J.LayerNorm(64, saved="e4m3").to(dev)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert norm(x.bfloat16()).dtype is torch.float32


def test_views_and_leading_axes(dev):
    """Values with several axes, transposed, sliced, off 16 bytes, negated late; weights that are views."""
    import jakal_net as J

    base = torch.randn(3, 70, 5, 66, generator=torch.Generator().manual_seed(2)).to(dev).bfloat16()
    w = torch.randn(48, 65, device=dev).bfloat16()[:, 1:]
    b = torch.randn(48, device=dev).bfloat16()
    q = _frozen(dev, 48, 64)
    views = [base[:, :, :, 1:65], base.transpose(1, 2)[..., :64], base[::2, 3, :, :64], base[0, 0, 0, 2:66],
             torch._neg_view(base)[..., :64]]
    off = torch.zeros(48 * 32 + 1, dtype=torch.uint8, device=dev)[1:].view(48, 32)
    off.copy_(q.codes)
    loose = J.MXTensor(off, q.scales.t().contiguous().t(), "e2m1", 64)
    for v in views:
        solid = v.resolve_neg().clone(memory_format=torch.contiguous_format)
        a, c = v.detach().requires_grad_(), solid.requires_grad_()
        linear = lambda t: J.linear(t, w, b, saved="e4m3")
        # (the library's product may add the bias of a strided input after a rounding)
        assert torch.equal(linear(a), F.linear(a.resolve_neg(), w, b)) and torch.equal(linear(c), F.linear(c, w, b))
        for run in (linear, lambda t: J.gelu(t, saved="e4m3"), lambda t: J.layer_norm(t, saved="e4m3"),
                    lambda t: J.mx_linear(t, loose, b), lambda t: J.mx_linear(t, q, b, activations="e2m1")):
            y, z = run(a), run(c)
            assert y.shape == z.shape and (run is linear or torch.equal(y, z))
            g = torch.randn(z.shape, device=dev).bfloat16()
            left, right = torch.autograd.grad(y, a, g)[0].float(), torch.autograd.grad(z, c, g)[0].float()
            assert bool(((left - right).abs() <= 2 * O.half(torch.bfloat16) * right.abs() + 1e-6).all())
        assert torch.equal(J.mx_linear(solid, loose, b), J.mx_linear(solid, q, b))


def test_expanded_gradients_and_shared_inputs(dev):
    """A sum's gradient has no memory of its own; the same tensor as input, weight and bias' maker."""
    import jakal_net as J

    x = torch.randn(64, 64, device=dev, requires_grad=True)
    J.linear(x, x, x[0], saved="e4m3").sum().backward()
    k = M.quantize(x, "e4m3")[0].to(dev)
    xs = x.detach().double()
    want = xs.sum(0).expand(64, 64) + k.sum(0).expand(64, 64)
    want = want.clone()
    want[0] += 64.0
    bound = 2 * O.U * 64 * (xs.abs().sum(0) + k.abs().sum(0)).expand(64, 64) + 4 * O.U * (want.abs() + 64)
    O.close("shared", x.grad, want, bound)


def test_empty_batches(dev):
    import jakal_net as J

    q = _frozen(dev, 40, 64)
    x = torch.empty(0, 5, 64, device=dev, requires_grad=True)
    w, b = torch.randn(8, 64, device=dev, requires_grad=True), torch.randn(8, device=dev, requires_grad=True)
    s, lw = torch.empty(0, 5, device=dev, requires_grad=True), torch.ones(64, device=dev, requires_grad=True)
    y = J.linear(x, w, b, saved="e4m3")
    grads = torch.autograd.grad(y.sum(), [x, w, b])
    assert y.shape == (0, 5, 8) and grads[0].shape == x.shape
    assert not grads[1].any() and not grads[2].any()
    for out in (J.gelu(x, saved="e4m3"), J.mx_linear(x, q), J.mx_linear(x, q, activations="e2m1")):
        assert torch.autograd.grad(out.sum(), x)[0].shape == x.shape
    t, y = J.stabilize(s, x, lw, saved="e4m3")
    gs, gx, gl = torch.autograd.grad(t.sum() + y.sum(), [s, x, lw])
    assert gs.shape == s.shape and gx.shape == x.shape and not gl.any()


def test_rows_that_are_not_finite_stay_alone(dev):
    import jakal_net as J

    inf, nan = float("inf"), float("nan")
    for dim, out in ((96, 40), (2048, 300)):
        q = _frozen(dev, out, dim)
        for rows in (5, 90):
            for dtype in O.DTYPES.values():
                x = torch.randn(rows, dim, generator=torch.Generator().manual_seed(rows)).to(dtype)
                clean = x.to(dev)
                x[1, 3], x[3, dim - 1], x[4, 7] = nan, inf, -inf
                x = x.to(dev)
                bad = torch.zeros(rows, dtype=torch.bool, device=dev)
                bad[[1, 3, 4]] = True
                for acts in (None, "e2m1"):
                    y, z = J.mx_linear(x, q, activations=acts), J.mx_linear(clean, q, activations=acts)
                    assert torch.equal(y[~bad], z[~bad]) and bool((~torch.isfinite(y[bad])).any(-1).all())
                g = torch.randn(rows, dim, device=dev).to(dtype)
                a, c = x.detach().requires_grad_(), clean.detach().requires_grad_()
                for run in (lambda t: J.gelu(t, saved="e4m3"), lambda t: J.layer_norm(t, saved="e4m3")):
                    u, v = (torch.autograd.grad(run(t), t, g)[0] for t in (a, c))
                    assert torch.equal(u[~bad], v[~bad]) and bool(torch.isnan(u[bad]).any(-1).all())
        # gradients that are not finite, through a frozen weight
        a = clean.detach().requires_grad_()
        g = torch.randn(rows, out, device=dev).to(clean.dtype)
        good, = torch.autograd.grad(J.mx_linear(a, q), a, g)
        g[2, 1] = nan
        u, = torch.autograd.grad(J.mx_linear(a, q), a, g)
        keep = torch.arange(rows, device=dev) != 2
        assert torch.equal(u[keep], good[keep]) and bool(torch.isnan(u[2]).all())


def test_inputs_changed_before_the_backward(dev):
    """The input may change, since its codes are kept; the weight may not."""
    import jakal_net as J

    w = torch.randn(8, 64, device=dev, requires_grad=True)
    base = torch.randn(5, 64, device=dev, requires_grad=True)
    want = torch.autograd.grad(J.linear(base * 1.0, w, saved="e4m3").sum(), w)[0]
    x = base * 1.0
    y = J.linear(x, w, saved="e4m3")
    with torch.no_grad():
        x.zero_()
    assert torch.equal(torch.autograd.grad(y.sum(), w)[0], want)
    used = w * 1.0
    y = J.linear(base, used, saved="e4m3")
    with torch.no_grad():
        used.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = J.gelu(base, saved="e4m3")
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float() if t.dtype is torch.uint8 else t):
        y = J.gelu(base, saved="e4m3")
    with pytest.raises(RuntimeError, match="another device, type or size"):
        y.sum().backward()
    with torch.autograd.graph.save_on_cpu():
        y = J.gelu(base, saved="e4m3")
    assert torch.equal(torch.autograd.grad(y.sum(), base)[0],
                       torch.autograd.grad(J.gelu(base, saved="e4m3").sum(), base)[0])


def test_what_is_kept(dev):
    """Nothing of the input's own size stays with the graph."""
    import jakal_net as J

    sizes = []

    def pack(t):
        sizes.append((t.dtype, t.numel() * t.element_size()))
        return t

    x = torch.randn(64, 512, device=dev, requires_grad=True)
    w = torch.randn(16, 512, device=dev, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        J.linear(x, w, saved="e4m3"), J.gelu(x, saved="e4m3"), J.layer_norm(x, saved="e4m3")
    kept = [n for dtype, n in sizes if dtype is torch.uint8]
    assert kept and max(kept) == 64 * 512 and all(n <= 64 * 512 for _, n in sizes)


def test_transforms_and_second_derivatives(dev):
    import jakal_net as J

    x = torch.randn(3, 4, 64, device=dev)
    q = _frozen(dev, 8, 64)
    for run in (lambda t: J.gelu(t, saved="e4m3"), lambda t: J.layer_norm(t, saved="e4m3"), lambda t: J.mx_linear(t, q)):
        assert torch.equal(torch.func.vmap(run)(x), run(x))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: run(t).pow(3).sum())(x)
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(run, (x,), (x,))
        leaf = x.clone().requires_grad_()
        g, = torch.autograd.grad(run(leaf).pow(3).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.sum().backward()


def test_refusals(dev):
    import jakal_net as J

    x = torch.randn(6, 64, device=dev)
    q = _frozen(dev, 8, 64)
    w, b = torch.randn(8, 64, device=dev), torch.randn(8, device=dev)
    for call in (lambda: J.linear(x, w.bfloat16(), saved="e4m3"), lambda: J.linear(x, w, b.half(), saved="e4m3"),
                 lambda: J.linear(x, w[:, :60], saved="e4m3"), lambda: J.linear(x, w, b[1:], saved="e4m3"),
                 lambda: J.linear(x, w.cpu(), saved="e4m3"), lambda: J.mx_linear(x, q.to("cpu")),
                 lambda: J.mx_linear(x, q, b.half()), lambda: J.mx_linear(x, q, b.cpu()),
                 lambda: J.linear(x, w[:0], saved="e4m3"), lambda: J.gelu(x[:, :0], saved="e4m3"),
                 lambda: J.stabilize(x[1:, 0], x, saved="e4m3"), lambda: J.layer_norm(x, w[0, 1:], saved="e4m3"),
                 lambda: torch.ops.jakal_net_hip.mx_weight_grad(x, q.codes, q.scales, 64, False),
                 lambda: torch.ops.jakal_net_hip.mx_values(q.codes, q.scales, 1, 96, torch.float32),
                 lambda: torch.ops.jakal_net_hip.mx_values(q.codes, q.scales, 1, 64, torch.float64),
                 lambda: torch.ops.jakal_net_hip.gelu_backward(x[1:], *torch.ops.jakal_net_hip.mx_codes(x, 0))):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: J.gelu(x.double(), saved="e4m3"), lambda: J.mx_quantize(x.double()),
                 lambda: J.linear(x.double(), w.double(), saved="e4m3")):
        with pytest.raises(NotImplementedError):
            call()
    # where the library declines, "kernel" takes the PyTorch form
    assert J.gelu(x.double(), saved="e4m3", implementation="kernel").dtype is torch.float64
    assert J.mx_quantize(x.double(), implementation="kernel").codes.is_cuda


def test_more_than_2_31_elements(dev):
    """Quantising and the activation past 32-bit element numbers: the ends against the same rows alone."""
    import jakal_net as J

    rows, dim = 70_001, 32_000  # 2.24e9
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device=dev)
    for at in range(0, rows, 10_000):
        x[at:at + 10_000].normal_()
    q = J.mx_quantize(x)
    y = J.gelu(x.requires_grad_(), saved="e4m3")
    for at in (0, rows - 3):
        part = x.detach()[at:at + 3].clone()
        alone = J.mx_quantize(part)
        assert torch.equal(q.codes[at:at + 3], alone.codes) and torch.equal(q.scales[at:at + 3], alone.scales)
        assert torch.equal(y.detach()[at:at + 3], J.gelu(part, saved="e4m3"))
    del q
    g = torch.ones(1, device=dev, dtype=torch.bfloat16).expand(rows, dim)
    grad, = torch.autograd.grad(y, x, g)
    part = x.detach()[-3:].clone().requires_grad_()
    assert torch.equal(grad[-3:], torch.autograd.grad(J.gelu(part, saved="e4m3").sum(), part)[0])


def _model(activations=None, seed=7, dim=32):
    from jakal_net.progressive import ProgressiveBConfig, ProgressiveBStep

    cfg = ProgressiveBConfig(vocab=97, dim=dim, prefix=48, query=8, rank=8, topk=4, s_window=6, warmup=1, blocks=2,
                             expanded=24, compressed=8, refine=1, query_refine=2)
    torch.manual_seed(seed)
    model = ProgressiveBStep(cfg, activations=activations)
    g = torch.Generator().manual_seed(seed + 1)
    return model, [torch.randint(0, cfg.vocab - 1, (2, n), generator=g) for n in (cfg.prefix, cfg.query)]


def test_step_that_keeps_8_bits(dev, monkeypatch):
    """The loss is the plain step's to the bit; its norms, linears and activation all keep e4m3, and the head's
    gradients are their formulas at the kept inputs."""
    import jakal_net_native as jn
    from jakal_net.progressive import train_step

    calls = {}
    for name in ("layer_norm", "stabilize", "layer_norm_saved", "stabilize_saved", "linear_saved", "gelu_saved"):
        op = getattr(jn, name)
        monkeypatch.setattr(jn, name, lambda *a, _op=op, _n=name, **k: calls.__setitem__(_n, calls.get(_n, 0) + 1) or _op(*a, **k))
    plain, (prefix, target) = _model()
    model, _ = _model("e4m3")
    plain, model, prefix, target = plain.to(dev), model.to(dev), prefix.to(dev), target.to(dev)
    a = plain(prefix, target)
    assert set(calls) == {"layer_norm", "stabilize"}
    counts = dict(calls)
    calls.clear()
    seen = {}
    model.head[0].register_forward_hook(lambda m, i, o: seen.update(x=i[0].detach(), h=o.detach()))
    model.head[2].register_forward_hook(lambda m, i, o: seen.update(a=i[0].detach()))
    b = model(prefix, target)
    assert torch.equal(a, b)
    assert calls == {"layer_norm_saved": counts["layer_norm"], "stabilize_saved": counts["stabilize"], "linear_saved": 3,
                     "gelu_saved": 1}
    logits = model.query_logits(model.encode_prefix(prefix), target).detach()
    b.backward()
    g = torch.softmax(logits.double(), -1)
    g = (g - F.one_hot(target, 97)).reshape(-1, 97) / target.numel()
    x, h, act = (seen[n].reshape(-1, seen[n].shape[-1]) for n in ("x", "h", "a"))
    first, last = model.head[0], model.head[2]
    want, bound = M.product(g.t(), M.quantize(act, "e4m3")[0].to(dev))
    # the loss' gradient is off by some units of its own: 64 of them for 97 classes' sum and exponentials
    O.close("head.2", last.weight.grad, want, bound + 64 * O.U * (g.abs().t() @ act.abs().double() + g.abs().sum(0)[:, None]))
    ga, _ = M.product(g, last.weight.detach())
    gh, _ = M.gelu_slope(M.quantize(h, "e4m3")[0].to(dev), ga)
    want, bound = M.product(gh.t(), M.quantize(x, "e4m3")[0].to(dev))
    O.close("head.0", first.weight.grad, want,
            bound + 512 * O.U * ((g.abs() @ last.weight.detach().abs().double() * 1.2).t() @ x.abs().double()))
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    loss, norm = train_step(model, opt, prefix, target, max_norm=1.0, autocast=dict(device_type="cuda", dtype=torch.bfloat16))
    assert bool(torch.isfinite(loss)) and bool(torch.isfinite(norm))


@pytest.mark.parametrize("activations", [None, "e2m1"])
def test_head_of_4_bits(dev, activations, monkeypatch):
    """A trained model's head made ready for answering: its logits are the products' at the rounded weights."""
    import jakal_net as J
    import jakal_net_native as jn

    model, (prefix, target) = _model(dim=64)
    model, prefix, target = model.to(dev).eval(), prefix.to(dev), target.to(dev)
    weights = [m.weight.detach() for m in model.head if isinstance(m, torch.nn.Linear)]
    biases = [m.bias.detach() for m in model.head if isinstance(m, torch.nn.Linear)]
    calls = []
    op = jn.mx_linear
    monkeypatch.setattr(jn, "mx_linear", lambda *a, **k: calls.append(a[4]) or op(*a, **k))
    model.quantize_head(activations)
    with torch.no_grad():
        s = model.encode_prefix(prefix)
        seen = {}
        model.head[0].register_forward_hook(lambda m, i, o: seen.update(x=i[0], h=o))
        logits = model.query_logits(s, target)
    assert calls == [activations, activations]
    rounded = lambda x: x.double().cpu() if activations is None else M.quantize(x, activations)[0]
    for x, y, w, b in ((seen["x"], seen["h"], weights[0], biases[0]), (F.gelu(seen["h"]), logits, weights[1], biases[1])):
        flat = x.reshape(-1, x.shape[-1])
        value, bound = M.product(rounded(flat), M.quantize(w, "e2m1")[0].t(), b.cpu())
        O.close("head", y.reshape(-1, y.shape[-1]), value, bound + O.U * value.abs())
    # gradients reach what lies before the head
    loss = model(prefix, target)
    loss.backward()
    assert model.head_norm.weight.grad is not None and bool(torch.isfinite(model.embed.weight.grad).all())
    state = model.state_dict()
    again, _ = _model(dim=64)
    again = again.to(dev).quantize_head(activations)
    again.load_state_dict(state)
    with torch.no_grad():
        assert torch.equal(again.query_logits(again.encode_prefix(prefix), target), logits)


@pytest.mark.parametrize("kind", ["cpu", "order", "checkpoint", "reentrant checkpoint"])
def test_saved_tensors_that_come_back(dev, kind):
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
    from torch.utils.checkpoint import checkpoint

    leaves, q = _leaves(dev, 40, 96, 64, torch.bfloat16), _frozen(dev, 48, 64)
    run = lambda *t: sum(o.float().sum() for o in _block(*t, q))
    want = torch.autograd.grad(run(*leaves), leaves)
    if kind == "cpu":
        with save_on_cpu():
            loss = run(*leaves)
    elif kind == "order":
        other = lambda t: t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t.clone()
        with saved_tensors_hooks(lambda t: t, other):
            loss = run(*leaves)
    else:
        loss = checkpoint(run, *leaves, use_reentrant=kind.startswith("reentrant"))
    loss.backward()
    assert all(torch.equal(p.grad, g) for p, g in zip(leaves, want))


def test_captured_training_steps_that_keep_8_bits(dev):
    """Whole steps (loss, clipping, AdamW under autocast) of two models in two graphs, replayed in turn."""
    from jakal_net.progressive import train_step

    steps = []
    for seed in (11, 12):
        model, batch = _model("e4m3", seed)
        model = model.to(dev)
        opt = torch.optim.AdamW(model.parameters(), lr=1e-3, capturable=True)
        prefix, target = (t.to(dev) for t in batch)
        cast = dict(device_type="cuda", dtype=torch.bfloat16, cache_enabled=False)
        steps.append((model, opt, lambda m=model, o=opt, p=prefix, t=target: train_step(m, o, p, t, max_norm=0.1, autocast=cast)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _, _, step in steps:
            for _ in range(2):
                step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    tensors = lambda m, o: [p.data for p in m.parameters()] + [v for s in o.state.values() for v in s.values() if torch.is_tensor(v)]
    kept = [[t.clone() for t in tensors(m, o)] for m, o, _ in steps]

    def restore():
        for (m, o, _), saved in zip(steps, kept):
            for t, v in zip(tensors(m, o), saved):
                t.copy_(v)
        torch.cuda.synchronize()

    want = []
    for m, _, step in steps:
        loss, norm = step()
        want.append([loss.clone(), norm.clone()] + [p.data.clone() for p in m.parameters()])
        del loss, norm
    restore()
    graphs, outs = [], []
    for _, _, step in steps:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for rep in range(3):
        restore()
        for graph in graphs:
            graph.replay()
        torch.randn(1 << 20, device=dev).sum()
        torch.cuda.synchronize()
        for (m, _, _), (loss, norm), w in zip(steps, outs, want):
            got = [loss, norm] + [p.data for p in m.parameters()]
            assert all(torch.equal(a, b) for a, b in zip(got, w)), f"replay {rep}"


def test_compiled_training_step(dev):
    torch._dynamo.reset()
    model, (prefix, target) = _model("e4m3")
    model, prefix, target = model.to(dev), prefix.to(dev), target.to(dev)
    used = list(model.parameters())
    loss = model(prefix, target)
    want = torch.autograd.grad(loss, used, allow_unused=True)
    again = torch.compile(model, backend="aot_eager")(prefix, target)
    got = torch.autograd.grad(again, used, allow_unused=True)
    torch._dynamo.reset()
    # the same kernels between decomposed torch operators: fp32 roundings apart
    assert float(again.detach()) == pytest.approx(float(loss.detach()), rel=1e-5)
    # which may move a kept value by a step of its code (2^-3 of itself), in few places
    for p, a, b in zip(used, want, got):
        a, b = (torch.zeros_like(p) if t is None else t for t in (a, b))
        assert float((a - b).norm()) <= 2.0 ** -3 * float(a.norm()) + 1e-7


def test_products_past_32_bits(dev):
    """Outputs and gradients of more than 2^31 elements: the last rows against float64, and sums over all of them."""
    import jakal_net as J

    rows, dim, out = 140_003, 64, 16_384  # 2.29e9
    x = torch.empty(rows, dim, device=dev, dtype=torch.bfloat16).normal_().requires_grad_()
    q = _frozen(dev, out, dim)
    w = J.mx_dequantize(q).double()
    for acts in (None, "e2m1"):
        y = J.mx_linear(x, q, activations=acts)
        a = x.detach()[-3:].double() if acts is None else M.quantize(x.detach()[-3:], acts)[0].to(dev)
        value, bound = M.product(a, w.t())
        O.close(f"{acts} y", y[-3:], value, bound + O.half(torch.bfloat16) * value.abs() + O.floor(torch.bfloat16))
        del y
    g = torch.empty(rows, out, device=dev, dtype=torch.bfloat16)
    for at in range(0, rows, 20_000):
        g[at:at + 20_000].normal_()
    gx = torch.ops.jakal_net_hip.mx_input_grad(g, q.codes, q.scales, dim)
    value, bound = M.product(g[-3:], w)
    O.close("grad_x", gx[-3:], value, bound + O.half(torch.bfloat16) * value.abs() + O.floor(torch.bfloat16))
    codes, scales = torch.ops.jakal_net_hip.mx_codes(x.detach(), 0)
    gw, gb = torch.ops.jakal_net_hip.mx_weight_grad(g, codes, scales, dim, True)
    some = [0, 5, out - 1]
    value, bound = M.product(g[:, some].t(), M.quantize(x.detach(), "e4m3")[0].to(dev))
    O.close("grad_w", gw[some], value, bound + O.half(torch.bfloat16) * value.abs())
    value, bound = M.sums(g[:, some])
    O.close("grad_b", gb[some], value, bound + O.half(torch.bfloat16) * value.abs())


def test_calls_on_two_streams_at_once(dev):
    leaves, q = [_leaves(dev, 900, 128, 520, torch.bfloat16, seed=i) for i in range(2)], _frozen(dev, 1000, 520)
    want = [_step(m, q) for m in leaves]
    streams = [torch.cuda.Stream() for _ in leaves]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = _step(leaves[i], q)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
