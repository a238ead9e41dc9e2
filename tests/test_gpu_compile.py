"""The training-step operators inside torch.compile and under the tracing that it
does: whole graphs with their backward, changing sizes, lists that are written,
and the Progressive-B step."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _fresh():
    torch._dynamo.reset()
    yield
    torch._dynamo.reset()


def _leaves(dev, rows, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    made = [torch.randn(shape, generator=g).to(dtype).to(dev).requires_grad_()
            for shape in ((2, rows), (2, rows, dim))]
    made += [torch.randn(dim, generator=g).to(dev).requires_grad_() for _ in range(2)]
    target = torch.randint(0, dim, (2, rows), generator=g).to(dev)
    target[0, 0] = -100
    return made, target


def _update(state, val, weight, bias, target):
    import jakal_net as J

    t, y = J.stabilize(state, val, weight, bias, scale=0.5)
    z = J.layer_norm(y, weight)
    return t, J.cross_entropy(z, target), J.cross_entropy(z, target, reduction="none")


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_whole_graph_with_its_backward(dev, backend, dtype):
    leaves, target = _leaves(dev, 37, 64, dtype)
    compiled = torch.compile(_update, backend=backend, fullgraph=True)
    results = []
    for run in (_update, compiled):
        t, loss, each = run(*leaves, target)
        seeds = [torch.ones_like(t), torch.ones_like(loss), torch.full_like(each, 0.25)]
        results.append([t, loss, each, *torch.autograd.grad([t, loss, each], leaves, seeds)])
    for eager, graph in zip(*results):
        assert eager.dtype is graph.dtype and torch.equal(eager, graph)


def test_sizes_that_change(dev):
    compiled = torch.compile(_update, backend="aot_eager", fullgraph=True, dynamic=True)
    for rows, dim in ((5, 32), (9, 32), (70, 48), (1, 48), (513, 96)):
        leaves, target = _leaves(dev, rows, dim, torch.float32, seed=rows)
        results = []
        for run in (_update, compiled):
            t, loss, each = run(*leaves, target)
            results.append([t, loss, each, *torch.autograd.grad(t.sum() + loss + each.sum(), leaves)])
        for eager, graph in zip(*results):
            assert torch.equal(eager, graph), (rows, dim)


def test_without_gradients_and_on_views(dev):
    import jakal_net as J

    def run(x, target):
        return J.layer_norm(x[1:, 1:]), J.cross_entropy(x[1:, 1:], target, reduction="none")

    x, target = torch.randn(9, 33, device=dev), torch.randint(0, 32, (8,), device=dev)
    for context in (torch.no_grad, torch.inference_mode):
        torch._dynamo.reset()
        with context():
            for a, b in zip(run(x, target), torch.compile(run, backend="aot_eager", fullgraph=True)(x, target)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("limit", [0.5, 100.0])
def test_lists_in_a_graph(dev, limit):
    """In place, into buffers, and a norm alone; what the graph leaves in the tensors is what the eager call leaves."""
    import jakal_net as J

    def run(a, b, c, out_b):
        first = J.grad_norm([a, b, c])
        norm = J.clip_grads([a, b], limit, out=[a, out_b])
        return first, norm, J.clip_grads([c], limit, float("inf")), a + 1, out_b * 2

    def made():
        g = torch.Generator().manual_seed(5)
        return [torch.randn(s, generator=g).to(dev) for s in ((70, 3), (9001,), (4, 5))] + [torch.zeros(9001, device=dev)]

    eager, graph = made(), made()
    want = run(*eager)
    got = torch.compile(run, backend="aot_eager", fullgraph=True)(*graph)
    for a, b in zip([*want, *eager], [*got, *graph]):
        assert torch.equal(a, b)


def test_under_autocast(dev):
    leaves, target = _leaves(dev, 20, 32, torch.float32)
    weight = torch.randn(32, 32, device=dev)

    def run(val):
        import jakal_net as J

        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = J.layer_norm(val @ weight, leaves[2], leaves[3])
            return J.cross_entropy(y @ weight, target)

    results = [(loss, *torch.autograd.grad(loss, leaves[1:]))
               for loss in (run(leaves[1]), torch.compile(run, backend="aot_eager", fullgraph=True)(leaves[1]))]
    for eager, graph in zip(*results):
        assert torch.equal(eager, graph)


def test_operators_below_autograd_match_their_fake_forms(dev):
    ops = torch.ops.jakal_net_hip
    g = torch.Generator().manual_seed(1)
    x, gy, w = (torch.randn(s, generator=g).to(dev) for s in ((6, 40), (6, 40), (40,)))
    s, gs, stats = (torch.randn(n, generator=g).to(dev) for n in ((6,), (6,), (6, 2)))
    t, count = torch.randint(0, 40, (6,), generator=g).to(dev), torch.tensor(6.0, device=dev)
    calls = [(ops.row_norm_forward, (s, x, w, w, 1e-5, 0.5, True)),
             (ops.row_norm_backward, (gs, gy, s, x, w, stats, 0.5, torch.float32, [True] * 4)),
             (ops.loss_forward, (x, t, -100, 2, True)), (ops.loss_backward, (count, x, t, stats, count, -100, 2)),
             (ops.list_norm, ([x, w], 0)), (ops.list_clip, ([x, w], [gy, torch.zeros_like(w)], 0.5, 0))]
    for op, args in calls:
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))


def test_operators_below_autograd_refuse_what_does_not_fit(dev):
    ops = torch.ops.jakal_net_hip
    x, w = torch.randn(6, 40, device=dev), torch.randn(40, device=dev)
    s, stats, t = torch.randn(6, device=dev), torch.randn(6, 2, device=dev), torch.zeros(6, dtype=torch.int64, device=dev)
    one = torch.ones((), device=dev)
    none = [False] * 4
    for call in (lambda: ops.row_norm_forward(s[1:], x, w, w, 1e-5, 1.0, True),
                 lambda: ops.row_norm_forward(s, x, w[1:], w, 1e-5, 1.0, True),
                 lambda: ops.row_norm_backward(None, x[1:], None, x, w, stats, 1.0, torch.float32, [False, True, False, False]),
                 lambda: ops.row_norm_backward(None, None, None, x, w, stats, 1.0, torch.float32, [False, True, False, False]),
                 lambda: ops.row_norm_backward(None, x, None, x, w, stats[1:], 1.0, torch.float32, none),
                 lambda: ops.row_norm_backward(None, x, None, x, w, stats, 1.0, torch.bfloat16, [False, False, False, True]),
                 lambda: ops.row_norm_backward(s, None, None, x, w, stats, 1.0, torch.float32, [True, False, False, False]),
                 lambda: ops.row_norm_backward(None, x, None, x, None, stats, 1.0, torch.float32, [False, False, True, False]),
                 lambda: ops.loss_forward(x, t[1:], -100, 2, True),
                 lambda: ops.loss_backward(one, x, t, stats[1:], one, -100, 2),
                 lambda: ops.loss_backward(one, x, t, stats, None, -100, 2),
                 lambda: ops.loss_backward(one, x, t, stats, one, -100, 0),
                 lambda: ops.list_clip([x], [x.t()], 1.0, 0), lambda: ops.list_clip([x], [], 1.0, 0),
                 lambda: ops.list_norm([x[:, :3]], 0), lambda: ops.list_norm([], 0), lambda: ops.list_clip([], [], 1.0, 0)):
        with pytest.raises((RuntimeError, ValueError)):
            call()


def test_the_progressive_step(dev):
    """The model compiles as it did with torch's own norms and loss: the ctypes propagation ops break the graph."""
    from jakal_net.progressive import ProgressiveBConfig, ProgressiveBStep

    cfg = ProgressiveBConfig(vocab=97, dim=32, prefix=48, query=8, rank=8, topk=4, s_window=6, warmup=1, blocks=1,
                             expanded=24, compressed=8, refine=1, query_refine=1)
    torch.manual_seed(3)
    model = ProgressiveBStep(cfg).to(dev)
    g = torch.Generator().manual_seed(4)
    prefix, target = (torch.randint(0, 96, (2, n), generator=g).to(dev) for n in (cfg.prefix, cfg.query))
    loss = model(prefix, target)
    used = list(model.parameters())
    want = torch.autograd.grad(loss, used, allow_unused=True)
    again = torch.compile(model, backend="aot_eager")(prefix, target)
    got = torch.autograd.grad(again, used, allow_unused=True)
    # the same kernels between decomposed torch operators: fp32 roundings apart
    assert float(again.detach()) == pytest.approx(float(loss.detach()), rel=1e-5)
    for p, a, b in zip(used, want, got):
        # (a compiled graph gives zeros for a parameter that the loss does not reach)
        a, b = (torch.zeros_like(p) if t is None else t for t in (a, b))
        assert float((a - b).norm()) <= 1e-4 * float(a.norm()) + 1e-7
