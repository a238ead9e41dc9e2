"""The vocabulary loss at the most classes it takes and at more rows than its grids
have places for."""

import math

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("classes", [(1 << 31) - 1, (1 << 30) + 3])
def test_the_most_classes(classes):
    """One row of bf16 logits.  A sum of 1024 threads has classes / 65,536 steps of 64 terms a thread, whose roundings
    (with those of the terms and the join) bound the loss; the gradient's elements have that and their own."""
    import jakal_net as J

    z = torch.empty(1, classes, device="cuda", dtype=torch.bfloat16)
    gen = torch.Generator("cuda").manual_seed(classes)
    total, top = 0.0, float("-inf")
    for part in z.view(-1).split(1 << 28):
        part.normal_(std=2.0, generator=gen)
        top = max(top, float(part.max()))
    for part in z.view(-1).split(1 << 28):
        total += float(torch.exp(part.double() - top).sum())
    log = math.log(total)
    steps = (classes // 65536 + 64 + 16) * O.U
    for t in (0, classes // 2 + 1, classes - 1):
        target = torch.tensor([t], device="cuda")
        leaf = z.detach().requires_grad_()
        loss = J.cross_entropy(leaf, target)
        zt = float(z[0, t])
        # (4 roundings of each exponential's argument, of which the mean under the softmax is below log(classes))
        e_log = steps + 4 * O.U * math.log(classes) + O.U * log
        assert abs(float(loss.detach()) - (log + top - zt)) <= e_log + 4 * O.U * (log + top - zt)
        (grad,) = torch.autograd.grad(loss, leaf)
        for at in (0, 1, 7, classes // 2, classes // 2 + 1, classes - 9, classes - 2, classes - 1):
            away = top - float(z[0, at])
            p = math.exp(-away - log)
            want = p - (at == t)
            bound = p * (O.U * (6 * away + 6 * log + 8) + e_log) + (O.half(z.dtype) + 2 * O.U) * abs(want)
            assert abs(float(grad[0, at]) - want) <= bound, (t, at)
        del grad, leaf, loss


@pytest.mark.parametrize("rows,classes,dtype", [((1 << 22) + 9, 6, "fp32"), ((1 << 20) + 5, 1040, "bf16")])
def test_more_rows_than_workgroups(rows, classes, dtype):
    import jakal_net as J

    gen = torch.Generator("cuda").manual_seed(rows)
    kind = O.DTYPES[dtype]
    z = torch.empty(rows, classes, device="cuda", dtype=kind).normal_(std=2.0, generator=gen)
    t = torch.randint(0, classes, (rows,), device="cuda", generator=gen)
    t[3::7] = -100
    t[-1] = classes - 1
    leaf = z.requires_grad_()
    loss = J.cross_entropy(leaf, t, reduction="none")
    (grad,) = torch.autograd.grad(loss, leaf, torch.ones(rows, device="cuda"))
    z = z.detach()
    for at in (slice(0, 70), slice(rows // 2, rows // 2 + 70), slice(rows - 70, rows)):
        want = O.cross_entropy(z[at], t[at], reduction="none")
        value, bound = want["loss"]
        O.close("loss", loss[at], value, bound + O.U * value.abs())
        value, bound = want["grad"]
        O.close("grad", grad[at], value, bound + O.half(kind) * value.abs() + O.floor(kind))
    whole = J.cross_entropy(z, t)
    rows_sum, count = float(loss.detach().double().sum()), int((t != -100).sum())
    assert abs(float(whole) - rows_sum / count) <= (O.U + rows * 2.0 ** -52) * rows_sum / count
    assert not grad[t == -100].any()
