"""Which layer norm backwards take one launch: the line was drawn where a captured
call is faster on either side of it."""

import pytest
import torch

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


@pytest.mark.parametrize("rows,dim,one", [(64, 64, True), (65, 64, False), (16, 512, True), (17, 512, False),
                                          (2, 4096, True), (3, 4096, False), (2, 8192, True), (3, 8192, False)])
def test_one_launch_for_two_steps_of_rows(rows, dim, one):
    import jakal_net as J

    x, g = torch.randn(rows, dim, device="cuda").requires_grad_(), torch.randn(rows, dim, device="cuda")
    w, b = (torch.ones(dim, device="cuda").requires_grad_() for _ in range(2))
    y = J.layer_norm(x, w, b)
    names = _kernels(lambda: torch.autograd.grad(y, [x, w, b], g))
    want = {"norm_backward_kernel": 1} if one else {"norm_backward_kernel": 1, "norm_columns_finish_kernel": 1}
    assert names == want, names
