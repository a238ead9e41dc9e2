"""Layer updates whose norm is not a bare layer norm: other modules in its place,
subclasses, parametrisations and hooks are called, as any module is."""

import pytest
import torch
from torch import nn

import jakal_net as J


def _layer(seed=0):
    g = torch.Generator().manual_seed(seed)
    layer = J.Layer(dim=12, num_nodes=5, state=torch.randn(2, 5, generator=g), val=torch.randn(2, 5, 12, generator=g))
    return layer, J.LayerDelta(delta_state=layer.state + 1, delta_val=layer.val * 2)


class _Shifted(J.LayerNorm):
    def forward(self, x):
        return super().forward(x) + 3.0


class _Doubled(nn.Module):
    def forward(self, weight):
        return weight * 2


def _norms():
    parametrised = J.LayerNorm(12)
    nn.utils.parametrize.register_parametrization(parametrised, "weight", _Doubled())
    return dict(identity=nn.Identity(), axes=nn.LayerNorm((5, 12)), rms=nn.RMSNorm(12),
                chain=nn.Sequential(nn.LayerNorm(12), nn.Tanh()), subclass=_Shifted(12), parametrised=parametrised)


@pytest.mark.parametrize("kind", list(_norms()))
@pytest.mark.parametrize("scale", [1.0, 0.25])
def test_other_modules_are_called(kind, scale):
    norm = _norms()[kind]
    layer, delta = _layer()
    kept = J.stabilize_layer(layer, norm)
    assert torch.equal(kept.val, norm(layer.val)) and torch.equal(kept.state, torch.tanh(layer.state))
    moved = J.stabilize_layer(layer, norm, delta, scale)
    assert torch.equal(moved.val, norm(delta.delta_val * scale))
    assert torch.equal(moved.state, torch.tanh(delta.delta_state * scale))


@pytest.mark.parametrize("make", [nn.LayerNorm, J.LayerNorm])
def test_hooks_run(make):
    layer, delta = _layer(1)
    calls = []
    norm = make(12)
    handles = [norm.register_forward_pre_hook(lambda m, args: calls.append("before")),
               norm.register_forward_hook(lambda m, args, out: calls.append("after") or out + 1.0),
               norm.register_full_backward_hook(lambda m, gi, go: calls.append("backward"))]
    moved = J.stabilize_layer(layer, norm, delta, 0.5)
    assert calls == ["before", "after"]
    moved.val.sum().backward()
    assert calls == ["before", "after", "backward"]
    for h in handles:
        h.remove()
    assert torch.equal(J.stabilize_layer(layer, norm, delta, 0.5).val + 1.0, moved.val) and len(calls) == 3


def test_a_forward_of_its_own_runs():
    layer, _ = _layer(2)
    norm = J.LayerNorm(12)
    plain = norm(layer.val)
    norm.forward = lambda x, _forward=norm.forward: _forward(x) * 2.0
    assert torch.equal(J.stabilize_layer(layer, norm).val, plain * 2.0)


def test_the_model_takes_another_norm_and_calls_hooks():
    from jakal_net.progressive import ProgressiveBConfig, ProgressiveBStep

    cfg = ProgressiveBConfig(vocab=97, dim=32, prefix=48, query=8, rank=8, topk=4, s_window=6, warmup=1, blocks=1,
                             expanded=24, compressed=8, refine=1, query_refine=1)
    g = torch.Generator().manual_seed(3)
    prefix, target = (torch.randint(0, 96, (2, n), generator=g) for n in (48, 8))
    torch.manual_seed(4)
    model = ProgressiveBStep(cfg, implementation="streaming")
    plain = model(prefix, target)
    widths = []
    model.s_norm.register_forward_hook(lambda m, args, out: widths.append(out.shape[-1]))
    assert torch.equal(model(prefix, target), plain) and len(widths) >= 3 and set(widths) == {32}
    model.s_norm = nn.RMSNorm(32)
    assert bool(torch.isfinite(model(prefix, target)))
