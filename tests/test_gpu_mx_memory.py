"""What a Progressive-B step holds between its forward and its backward, with its activations kept in 8 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _held(dev, activations):
    """Bytes that the loss' graph holds, after a step that makes the libraries' own allocations."""
    from jakal_net.progressive import ProgressiveBConfig, ProgressiveBStep

    cfg = ProgressiveBConfig(vocab=997, dim=128, prefix=256, query=32, rank=16, topk=8, s_window=16, warmup=2, blocks=2,
                             expanded=96, compressed=32, refine=2, query_refine=2)
    torch.manual_seed(7)
    model = ProgressiveBStep(cfg, activations=activations).to(dev)
    prefix, target = (torch.randint(0, cfg.vocab - 1, (8, n), device=dev) for n in (cfg.prefix, cfg.query))
    for _ in range(2):
        model.zero_grad(set_to_none=True)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = model(prefix, target)
        held = torch.cuda.memory_allocated() - before
        loss.backward()
        del loss
    return held


def test_a_step_holds_less(monkeypatch):
    """Each update's values, fp32, are kept as codes and scales (33 bytes a run of 32) but for two that other layers
    hold as well: the embedded prefix and the feedback, from which the first states are made."""
    import jakal_net_native as jn

    dev = torch.device("cuda:0")
    plain = _held(dev, None)
    sizes = []
    op = jn.stabilize_saved
    monkeypatch.setattr(jn, "stabilize_saved", lambda state, val, *a, **k: sizes.append(val.numel()) or op(state, val, *a, **k))
    kept = _held(dev, "e4m3")
    updates = sorted(sizes[:len(sizes) // 2])[:-2]
    assert len(updates) > 8
    # codes and scales are allocations of their own, in steps of 512 bytes
    least = sum(n * 4 - n * 33 // 32 - 1024 for n in updates)
    print(f"held {plain} and {kept} bytes, {least} from {len(updates)} updates")
    assert plain - kept >= least
