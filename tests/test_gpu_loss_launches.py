"""Which losses take one launch: the line was drawn where a captured call is faster
on either side of it."""

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu


def _kernels(call):
    import jakal_net_native as jn

    jn.profile_enable(True)
    try:
        jn.profile_collect()
        call()
        torch.cuda.synchronize()
        return {name: launches for name, (launches, _) in jn.profile_collect().items()}
    finally:
        jn.profile_enable(False)


@pytest.mark.parametrize("rows,classes,dtype,one", [(1, 10, "fp32", True), (16, 4000, "fp32", True),
                                                    (16, 8000, "bf16", True), (17, 10, "fp32", False),
                                                    (64, 1000, "bf16", False), (1, 8192, "fp32", True),
                                                    (1, 8193, "fp32", False), (1, 64000, "bf16", False),
                                                    (16, 4100, "fp32", False)])
def test_one_launch_for_a_row_a_wave(rows, classes, dtype, one):
    import jakal_net as J

    z = torch.randn(rows, classes, device="cuda").to(O.DTYPES[dtype])
    t = torch.randint(0, classes, (rows,), device="cuda")
    t[::3] = -100
    t[-1] = 0
    names = _kernels(lambda: J.cross_entropy(z, t))
    assert names == ({"loss_small_kernel": 1} if one else {"loss_forward_kernel": 1, "loss_reduce_kernel": 1}), names
    value, bound = O.cross_entropy(z, t)["loss"]
    O.close("loss", J.cross_entropy(z, t), value, bound + O.U * value.abs())
    # the reduction "none" takes the other kernel: the same losses
    each = J.cross_entropy(z, t, reduction="none")
    assert float(J.cross_entropy(z, t, reduction="sum")) == pytest.approx(float(each.double().sum()), rel=1e-6)
