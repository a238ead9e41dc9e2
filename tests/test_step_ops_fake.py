"""The training-step operators on tensors without memory: sizes, types and
history as the real ones have them, and no kernel called (there is no GPU here)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norms_of_fake_tensors(dtype):
    import jakal_net as J

    with FakeTensorMode():
        base = torch.empty(5, 7, 33, device="cuda", dtype=dtype)
        val = base[1:, :, 1:].requires_grad_()  # a view with an offset, not contiguous
        state = torch.empty(4, 7, device="cuda", requires_grad=True)
        w, b = (torch.empty(32, device="cuda", requires_grad=True) for _ in range(2))
        y = J.layer_norm(val, w, b)
        assert y.shape == val.shape and y.dtype is dtype and y.device.type == "cuda" and y.is_contiguous()
        assert y.requires_grad and not J.layer_norm(val.detach()).requires_grad
        t, y = J.stabilize(state, val, w, scale=0.5)
        assert t.shape == state.shape and t.dtype is state.dtype and y.shape == val.shape and t.requires_grad
        assert J.layer_norm(torch.empty(0, 8, device="cuda")).shape == (0, 8)
        for call in (lambda: J.layer_norm(val, w[1:]), lambda: J.stabilize(state[1:], val), lambda: J.layer_norm(val, eps=-1.0),
                     lambda: J.layer_norm(torch.empty(3, 0, device="cuda")), lambda: J.layer_norm(val.double())):
            with pytest.raises(RuntimeError):
                call()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_of_fake_tensors(reduction):
    import jakal_net as J

    with FakeTensorMode():
        z = torch.empty(4, 6, 50, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        for kind in (torch.int64, torch.int32):
            loss = J.cross_entropy(z, torch.empty(4, 6, device="cuda", dtype=kind), reduction=reduction)
            assert loss.shape == ((4, 6) if reduction == "none" else ()) and loss.dtype is torch.float32
            assert loss.requires_grad and loss.device.type == "cuda"
        with pytest.raises(RuntimeError):
            J.cross_entropy(z, torch.empty(4, 5, device="cuda", dtype=torch.int64), reduction=reduction)


def test_lists_of_fake_tensors():
    import jakal_net as J

    with FakeTensorMode():
        grads = [torch.empty(s, device="cuda", dtype=k) for s, k in (((3, 4), torch.float32), ((), torch.bfloat16),
                                                                    ((0,), torch.float32))]
        out = [torch.empty(g.shape, device="cuda") for g in grads]
        for norm in (J.grad_norm(grads), J.grad_norm([grads[0].t()], float("inf")), J.clip_grads(grads, 1.0),
                     J.clip_grads(grads, 1.0, out=out), J.clip_grads([torch.empty(4, 3, device="cuda").t()], 1.0,
                                                                    out=[out[0]])):
            assert norm.shape == () and norm.dtype is torch.float32 and norm.device.type == "cuda"
        with pytest.raises(ValueError):
            J.clip_grads(grads, 1.0, out=out[::-1])


def test_history_of_fake_outputs():
    import jakal_net as J

    with FakeTensorMode():
        state, val = torch.empty(4, device="cuda"), torch.empty(4, 8, device="cuda")
        for a, b in ((True, False), (False, True), (True, True), (False, False)):
            t, y = J.stabilize(state.detach().requires_grad_(a), val.detach().requires_grad_(b))
            assert (t.requires_grad, y.requires_grad) == (a, b)
