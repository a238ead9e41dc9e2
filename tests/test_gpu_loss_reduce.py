"""Sum and mean of the losses of many rows, on both sides of the row count from
which many workgroups reduce them."""

import ctypes

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


@pytest.mark.parametrize("rows", [1, 1023, 32768, 32769, 40961, 200003, 1 << 20, (1 << 24) - 1])
@pytest.mark.parametrize("reduction", [1, 2])
def test_whole_numbers_reduce_exactly(rows, reduction):
    """Losses of 0 to 15: the 64-bit sums are exact, so is their rounding; the workspace between guards."""
    import jakal_net_native as jn

    gen = torch.Generator("cuda").manual_seed(rows)
    loss = torch.randint(0, 16, (rows,), device="cuda", generator=gen).float()
    target = torch.randint(-3, 3, (rows,), device="cuda", generator=gen)
    target[-1] = 2
    loss[target == -3] = 0.0
    out = torch.full((2,), -1.0, device="cuda")
    need = jn._LIB.jn_cross_entropy_reduce_workspace_bytes(rows)
    assert (need > 0) == (rows > 32768) and need <= 4096
    guard = 256
    ws = torch.full((guard + need + guard,), 171, device="cuda", dtype=torch.uint8)
    rc = jn._LIB.jn_cross_entropy_reduce(_p(loss), _p(target), rows, -3, reduction, _p(out[:1]), _p(out[1:]),
                                         ctypes.c_void_p(ws.data_ptr() + guard), need,
                                         ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    total, count = float(loss.double().sum()), int((target != -3).sum())
    want = total / count if reduction == 2 else total
    assert out.tolist() == torch.tensor([want, count], dtype=torch.float64).float().tolist()
    assert bool((ws[:guard] == 171).all()) and bool((ws[guard + need:] == 171).all())


@pytest.mark.parametrize("rows,classes,dtype", [(32768, 37, "fp32"), (32769, 37, "fp32"), (200003, 130, "bf16"),
                                                (1000003, 8, "fp16")])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_many_rows_with_ignored_ones(rows, classes, dtype, reduction):
    import jakal_net as J

    gen = torch.Generator("cuda").manual_seed(classes)
    z = (torch.randn(rows, classes, device="cuda", generator=gen) * 2.5).to(O.DTYPES[dtype]).requires_grad_()
    t = torch.randint(0, classes, (rows,), device="cuda", generator=gen)
    t[torch.rand(rows, device="cuda", generator=gen) < 0.2] = -100
    t[0], t[-1] = -100, 1
    loss = J.cross_entropy(z, t, reduction=reduction)
    (grad,) = torch.autograd.grad(loss, z)
    want = O.cross_entropy(z.detach(), t, -100, reduction)
    O.close("loss", loss, want["loss"][0], want["loss"][1] + O.U * want["loss"][0].abs())
    value, bound = want["grad"]
    O.close("grad", grad, value, bound + O.half(z.dtype) * value.abs() + O.floor(z.dtype))
    # the rows' own losses, summed in 64 bits, round to the same number (their order is nothing to 2^-53)
    rows_sum = float(J.cross_entropy(z.detach(), t, reduction="none").double().sum())
    exact = rows_sum / int((t != -100).sum()) if reduction == "mean" else rows_sum
    assert abs(float(loss.detach()) - exact) <= (O.U + rows * 2.0 ** -52) * abs(exact)


def test_nothing_counts_in_many_rows():
    import jakal_net as J

    z = torch.randn(40000, 5, device="cuda", requires_grad=True)
    t = torch.full((40000,), 3, device="cuda")
    assert bool(torch.isnan(J.cross_entropy(z, t, ignore_index=3)))
    loss = J.cross_entropy(z, t, ignore_index=3, reduction="sum")
    (grad,) = torch.autograd.grad(loss, z)
    assert float(loss.detach()) == 0.0 and not grad.any()


def test_two_captured_losses_of_many_rows_replay_as_eager():
    import jakal_net as J

    made = [(torch.randn(n, 33, device="cuda"), torch.randint(0, 33, (n,), device="cuda")) for n in (70001, 33333)]

    def step(z, t):
        leaf = z.detach().requires_grad_()
        loss = J.cross_entropy(leaf, t)
        return [loss.detach(), *torch.autograd.grad(loss, leaf)]

    want = [step(*m) for m in made]
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
        torch.randn(1 << 20, device="cuda").sum()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for a, b in zip(out, w):
                assert torch.equal(a, b), f"replay {rep}"
