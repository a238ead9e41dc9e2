"""Layer updates on the HIP library with norms that have to be called."""

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu


def test_a_hooked_norm_gives_what_the_fused_update_gives():
    """scale * val is rounded once more on its way to the called norm; by a power of two it is exact."""
    import jakal_net as J

    g = torch.Generator().manual_seed(0)
    state, val = (torch.randn(s, generator=g).cuda().requires_grad_() for s in ((3, 7), (3, 7, 64)))
    delta = J.LayerDelta(delta_state=state, delta_val=val)
    layer = J.Layer(dim=64, num_nodes=7, state=state.detach(), val=val.detach())
    norm = J.LayerNorm(64).cuda()
    fused = J.stabilize_layer(layer, norm, delta, 0.25)
    grads = torch.autograd.grad(fused.val.square().sum(), [val, norm.weight, norm.bias])
    seen = []
    norm.register_forward_hook(lambda m, args, out: seen.append(out))
    called = J.stabilize_layer(layer, norm, delta, 0.25)
    assert len(seen) == 1 and torch.equal(called.val, fused.val)
    assert torch.allclose(called.state, fused.state, rtol=4e-7, atol=1e-9)
    for a, b in zip(grads, torch.autograd.grad(called.val.square().sum(), [val, norm.weight, norm.bias])):
        assert torch.equal(a, b)
    other = J.stabilize_layer(layer, nn.Identity(), delta, 0.25)
    assert torch.equal(other.val, val * 0.25)
