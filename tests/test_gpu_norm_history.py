"""Which outputs of a stabilisation carry history: the state's where the state does,
the values' where the values, weight or bias do, as in the PyTorch form."""

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", [c for n in range(4) for c in itertools.combinations(("state", "val", "weight"), n)])
def test_history_follows_each_outputs_inputs(which):
    import jakal_net as J

    g = torch.Generator().manual_seed(1)
    shapes = dict(state=(3, 5), val=(3, 5, 24), weight=(24,))
    made = {n: torch.randn(s, generator=g).cuda() for n, s in shapes.items()}
    seeds = [torch.randn(s, generator=g).cuda() for s in ((3, 5), (3, 5, 24))]
    full = {n: v.clone().requires_grad_() for n, v in made.items()}
    want = dict(zip(full, torch.autograd.grad(J.stabilize(**full, scale=0.5), list(full.values()), seeds)))
    part = {n: v.clone().requires_grad_(n in which) for n, v in made.items()}
    outs = J.stabilize(**part, scale=0.5)
    history = [e.requires_grad for e in outs]
    assert history == ["state" in which, "val" in which or "weight" in which]
    assert history == [e.requires_grad for e in J.stabilize(**part, scale=0.5, implementation="reference")]
    if which:
        ends = [(e, s) for e, s in zip(outs, seeds) if e.requires_grad]
        grads = torch.autograd.grad([e for e, _ in ends], [part[n] for n in which], [s for _, s in ends])
        assert all(torch.equal(got, want[n]) for n, got in zip(which, grads))
