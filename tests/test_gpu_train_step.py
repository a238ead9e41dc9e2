"""The Progressive-B training step with its norms, updates, loss and clipping on
the HIP library: against the float64 step on the CPU, and captured."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


def _model(seed, implementation="native"):
    from jakal_net.progressive import ProgressiveBConfig, ProgressiveBStep

    cfg = ProgressiveBConfig(vocab=97, dim=32, prefix=48, query=8, rank=8, topk=4, s_window=6, warmup=1, blocks=2,
                             expanded=24, compressed=8, refine=1, query_refine=2)
    torch.manual_seed(seed)
    model = ProgressiveBStep(cfg, implementation=implementation)
    g = torch.Generator().manual_seed(seed + 1)
    return model, [torch.randint(0, cfg.vocab - 1, (2, n), generator=g) for n in (cfg.prefix, cfg.query)]


class _Ops:
    """Counts the library's calls of the training-step operators."""

    def __init__(self, monkeypatch):
        import jakal_net_native as jn

        self.calls = {}
        for name in ("layer_norm", "stabilize", "cross_entropy", "clip_grads"):
            op = getattr(jn, name)
            monkeypatch.setattr(jn, name, lambda *a, _op=op, _n=name, **k: self._count(_n) or _op(*a, **k))

    def _count(self, name):
        self.calls[name] = self.calls.get(name, 0) + 1


@pytest.mark.parametrize("share", [0.5, 3.0])
def test_clipped_step_against_float64(dev, share, monkeypatch):
    """Loss, norm and update of one step; the limit at half the norm, and above it."""
    from jakal_net.progressive import train_step

    ref, (prefix, target) = _model(7, "reference")
    ref = ref.double()
    native, _ = _model(7)
    native.load_state_dict({k: v.float() for k, v in ref.state_dict().items()})
    native = native.to(dev)
    # the float64 step's own norm sets the limit
    loss = ref(prefix, target)
    loss.backward()
    grads = [p.grad for p in ref.parameters() if p.grad is not None]
    norm = float(torch.linalg.vector_norm(torch.cat([g.reshape(-1) for g in grads])))
    limit = share * norm
    ops = _Ops(monkeypatch)
    before = [p.detach().clone() for p in native.parameters()]
    opt = torch.optim.SGD(native.parameters(), lr=1.0)
    got_loss, got_norm = train_step(native, opt, prefix.to(dev), target.to(dev), max_norm=limit)
    assert set(ops.calls) == {"layer_norm", "stabilize", "cross_entropy", "clip_grads"}
    assert ops.calls["cross_entropy"] == ops.calls["clip_grads"] == 1 and ops.calls["stabilize"] >= 10
    # the step's fp32 gradients agree with float64 to about 1e-4 of their norm (tests/test_gpu_progressive.py)
    assert float(got_loss) == pytest.approx(float(loss.detach()), rel=1e-5)
    assert float(got_norm) == pytest.approx(norm, rel=1e-3)
    factor = min(1.0, limit / (norm + 1e-6))
    moved = torch.cat([(b - p.detach()).double().cpu().reshape(-1) for b, p, q in
                       zip(before, native.parameters(), ref.parameters()) if q.grad is not None])
    want = torch.cat([g.reshape(-1) for g in grads]) * factor
    assert float(torch.linalg.vector_norm(moved - want)) <= 2e-3 * norm


def test_two_captured_clipped_steps_replay_as_eager(dev):
    """The whole step of two models in two graphs, replayed in turn from the same
    parameters with eager work between, gives the eager updates bit for bit."""
    from jakal_net.progressive import train_step

    steps = []
    for seed in (11, 12):
        model, batch = _model(seed)
        model = model.to(dev)
        opt = torch.optim.AdamW(model.parameters(), lr=1e-3, capturable=True)
        prefix, target = (t.to(dev) for t in batch)
        autocast = dict(device_type="cuda", dtype=torch.bfloat16, cache_enabled=False)
        steps.append((model, opt, lambda m=model, o=opt, p=prefix, t=target: train_step(m, o, p, t, max_norm=0.1,
                                                                                       autocast=autocast)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _, _, step in steps:
            for _ in range(2):
                step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()

    def tensors(model, opt):
        return [p.data for p in model.parameters()] + [v for st in opt.state.values() for v in st.values()
                                                       if torch.is_tensor(v)]

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
            assert float(norm) > 0.1, "the step has to clip"
            assert all(torch.equal(a, b) for a, b in zip(got, w)), f"replay {rep}"


def _update_and_loss(dev):
    """A layer update and a loss over its values, and the leaves it starts from."""
    import jakal_net as J

    g = torch.Generator().manual_seed(3)
    leaves = [torch.randn(shape, generator=g).to(dev).requires_grad_() for shape in ((2, 9), (2, 9, 40), (40,), (40,))]
    target = torch.randint(0, 40, (2, 9), generator=g).to(dev)

    def run(state, val, weight, bias):
        out, y = J.stabilize(state, val, weight, bias, scale=0.5)
        return J.cross_entropy(y, target) + out.square().sum()

    return run, leaves


def _other_order(t):
    """t, its elements in another order in memory."""
    return t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t.clone()


@pytest.mark.parametrize("kind", ["cpu", "order", "checkpoint", "reentrant checkpoint"])
def test_saved_tensors_that_come_back(dev, kind):
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
    from torch.utils.checkpoint import checkpoint

    run, leaves = _update_and_loss(dev)
    want = torch.autograd.grad(run(*leaves), leaves)
    if kind == "cpu":
        with save_on_cpu():
            loss = run(*leaves)
    elif kind == "order":
        with saved_tensors_hooks(lambda t: t, _other_order):
            loss = run(*leaves)
    else:
        loss = checkpoint(run, *leaves, use_reentrant=kind.startswith("reentrant"))
    loss.backward()
    assert all(torch.equal(p.grad, g) for p, g in zip(leaves, want))


@pytest.mark.parametrize("change", [torch.Tensor.bfloat16, torch.Tensor.cpu, lambda t: t.reshape(-1)[:1],
                                    lambda t: t.reshape(-1).repeat(2)], ids=["type", "device", "shorter", "longer"])
def test_saved_tensors_that_come_back_changed_raise(dev, change):
    import jakal_net as J
    from torch.autograd.graph import saved_tensors_hooks

    _, (state, val, weight, bias) = _update_and_loss(dev)
    target = torch.zeros(2, 9, dtype=torch.long, device=dev)
    with saved_tensors_hooks(lambda t: t, change):
        losses = [J.layer_norm(val, weight, bias).sum(), J.stabilize(state, val)[0].sum(), J.cross_entropy(val, target)]
    for loss in losses:
        with pytest.raises(RuntimeError, match="came back"):
            loss.backward()
