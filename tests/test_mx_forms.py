"""The PyTorch forms of the operators on microscaled numbers: values of one axis and of none,
autocast, meta tensors, complex ones."""

import pytest
import torch

import mx_oracle as M
import step_oracle as O

MODES = ["reference", "streaming", "kernel", "native"]


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("acts", [None, "e2m1"])
def test_values_of_one_axis(mode, acts):
    """A bias' gradient of a single row is the output's gradient."""
    import jakal_net as J

    x, b, g = _rand(1, 50).requires_grad_(), _rand(3, 9).requires_grad_(), _rand(2, 9)
    weight, w = J.mx_quantize(_rand(4, 9, 50), "e2m1"), M.quantize(_rand(4, 9, 50), "e2m1")[0]
    y = J.mx_linear(x, weight, b, activations=acts, implementation=mode)
    assert y.shape == (9,)
    gx, gb = torch.autograd.grad(y, (x, b), g)
    assert torch.equal(gb, g)
    value, bound = M.product(g[None], w)
    O.close("grad_x", gx[None], value, bound + O.U * value.abs())


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("cast", [False, True])
@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_norms_under_autocast_give_what_they_give_without_saved(dtype, cast, mode):
    """CPU autocast leaves a norm's values in their type, as it leaves torch's layer norm."""
    _norms_with_and_without_saved(torch.device("cpu"), dtype, cast, mode)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["reference", "native"])
@pytest.mark.parametrize("cast", [False, True])
@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_norms_under_autocast_on_the_gpu(dtype, cast, mode):
    """GPU autocast takes torch's layer norm in fp32."""
    _norms_with_and_without_saved(torch.device("cuda:0"), dtype, cast, mode)


def _norms_with_and_without_saved(dev, dtype, cast, mode):
    import jakal_net as J

    kind = O.DTYPES[dtype]
    state, x = (_rand(i, *s).to(dev, kind).requires_grad_() for i, s in ((1, (3, 7)), (2, (3, 7, 40))))
    # (torch's own layer norm on the GPU takes parameters of the values' type)
    weight = (1 + 0.1 * _rand(3, 40)).to(dev, torch.float32 if cast or dev.type == "cpu" else kind).requires_grad_()
    with torch.autocast(dev.type, dtype=torch.bfloat16, enabled=cast):
        y, want = (J.layer_norm(x, weight, saved=s, implementation=mode) for s in ("e4m3", None))
        t, z = J.stabilize(state, x, weight, scale=0.4, saved="e4m3", implementation=mode)
        plain = J.stabilize(state, x, weight, scale=0.4, implementation=mode)
    for got, expected in ((y, want), (t, plain[0]), (z, plain[1])):
        assert got.dtype is expected.dtype and torch.equal(got, expected)
    for out in (y, z):
        gx, gw = torch.autograd.grad(out.float().sum(), (x, weight), retain_graph=True)
        assert gx.dtype is kind and gw.dtype is weight.dtype


@pytest.mark.parametrize("mode", ["reference", "streaming"])
def test_meta_tensors(mode):
    """Shapes and types without memory, for which there is no autocast."""
    import jakal_net as J

    x, w, b = (torch.empty(*s, device="meta", requires_grad=True) for s in ((4, 7, 50), (9, 50), (9,)))
    weight = J.mx_quantize(torch.empty(9, 50, device="meta"), "e2m1", implementation=mode)
    assert weight.codes.shape == (9, 32) and weight.device.type == "meta"
    for y in (J.linear(x, w, b, saved="e4m3", implementation=mode), J.mx_linear(x, weight, b, implementation=mode),
              J.mx_linear(x, weight, b, activations="e2m1", implementation=mode)):
        assert y.shape == (4, 7, 9) and [g.shape for g in torch.autograd.grad(y.sum(), (x, b))] == [x.shape, b.shape]
    for kind in (torch.float32, torch.bfloat16):
        v = x.detach().to(kind).requires_grad_()
        for y in (J.gelu(v, saved="e4m3", implementation=mode), J.layer_norm(v, saved="e4m3", implementation=mode)):
            assert y.shape == x.shape and y.dtype is kind and torch.autograd.grad(y.sum(), v)[0].shape == x.shape


@pytest.mark.parametrize("mode", MODES)
def test_a_tensor_without_axes_is_refused(mode):
    """As the library refuses it: with a RuntimeError that names the shape."""
    import jakal_net as J

    x = torch.tensor(1.0, requires_grad=True)
    for call in (lambda: J.mx_quantize(x, implementation=mode), lambda: J.gelu(x, saved="e4m3", implementation=mode),
                 lambda: J.layer_norm(x, saved="e4m3", implementation=mode),
                 lambda: J.linear(x, torch.ones(3, 1), saved="e4m3", implementation=mode),
                 lambda: J.mx_linear(x, J.mx_quantize(torch.ones(3, 1), "e2m1"), implementation=mode)):
        with pytest.raises(RuntimeError, match=r"shape \(\)"):
            call()


@pytest.mark.parametrize("mode", MODES)
def test_complex_values_are_refused(mode):
    """Microscaled numbers are real: the imaginary parts would be lost."""
    import jakal_net as J

    x = torch.complex(_rand(1, 3, 32), _rand(2, 3, 32))
    weight = J.mx_quantize(_rand(4, 9, 32), "e2m1")
    for call in (lambda: J.mx_quantize(x, implementation=mode), lambda: J.gelu(x, saved="e4m3", implementation=mode),
                 lambda: J.linear(x, x, saved="e4m3", implementation=mode),
                 lambda: J.layer_norm(x, saved="e4m3", implementation=mode),
                 lambda: J.mx_linear(x, weight, implementation=mode),
                 lambda: J.mx_linear(x, weight, activations="e2m1", implementation=mode)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_dequantising_to_other_types_is_declined_for_tensors_without_memory_too():
    """A traced call takes the form that the call itself takes."""
    import jakal_net as J
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q = J.mx_quantize(torch.empty(3, 64, device="cuda"), "e2m1")
        for kind in (torch.float64, torch.int32):
            with pytest.raises(NotImplementedError):
                J.mx_dequantize(q, kind)
            assert J.mx_dequantize(q, kind, implementation="kernel").dtype is kind
        assert J.mx_dequantize(q, torch.float16).dtype is torch.float16
