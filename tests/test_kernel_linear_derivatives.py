"""Derivatives of a kernel-mode Linear beyond the first, and torch.func's transforms over it: for float32 rows above KERNEL_MAX_ROWS its product is torch's own."""

import pytest
import torch
import torch.nn as nn

from llmquant.core.scheme import QuantizationArgs, QuantizationScheme
from llmquant.quantizers import KernelQuantLinear
from llmquant.quantizers.kernel import _FrozenCodes


@pytest.fixture
def no_kernels(monkeypatch):
    """On the CPU: a module of groups that no kernel takes, whose product is torch's own."""
    import llmquant.quantizers.kernel as kernel

    monkeypatch.setattr(kernel, "load_extension", lambda: type("None", (), {"wq_gemv": None})())


def linear(inp, out, group, bits, bias=True, heads=None, dtype=torch.float32, device="cpu"):
    gen = torch.Generator().manual_seed(inp + out)
    source = nn.Linear(inp, out, bias=bias)
    with torch.no_grad():
        for p in source.parameters():
            p.copy_(torch.randn(p.shape, generator=gen) / inp ** 0.5)
    weights = QuantizationArgs(num_bits=bits, strategy="group", group_size=group, head_dim=heads)
    return KernelQuantLinear.from_linear(source.to(dtype).to(device), QuantizationScheme(weights=weights, input_activations=None))


@pytest.mark.parametrize("inp, group, heads", [(36, 12, None), (30, 12, None)])
@pytest.mark.parametrize("bits", [8, 4])
def test_differentiated_twice(no_kernels, inp, group, heads, bits):
    """The gradient is itself a function that can be differentiated (64 bits, on the CPU)."""
    module = linear(inp, 10, group, bits, heads=heads, dtype=torch.float64)
    x = torch.randn(2, 3, inp, dtype=torch.float64, generator=torch.Generator().manual_seed(1), requires_grad=True)

    def call(x, bias):
        module.bias = nn.Parameter(bias.detach()) if bias is not module.bias else bias
        return _FrozenCodes.apply(x, bias, module)

    assert torch.autograd.gradcheck(call, (x, module.bias))
    assert torch.autograd.gradgradcheck(lambda x: _FrozenCodes.apply(x, module.bias, module), (x,))
    # a penalty on a gradient's norm, as module(x) gives it
    weight = module._real_weight(torch.float64)
    first, = torch.autograd.grad(module(x).square().sum(), x, create_graph=True)
    got, = torch.autograd.grad(first.square().sum(), x)
    y = x.detach().flatten(0, 1) @ weight.T + module.bias
    assert torch.allclose(got.flatten(0, 1), 2 * (2 * y @ weight) @ (2 * weight.T @ weight))


def check_transforms(module, x, rtol):
    """Against the dense weight that the codes stand for."""
    from torch.func import grad, hessian, jacrev, jvp, vjp, vmap

    weight, bias = module._real_weight(x.dtype), module.bias

    def dense(x):
        return x @ weight.T + bias

    def close(a, b):
        assert a.shape == b.shape and (a - b).norm() <= rtol * b.norm()

    close(grad(lambda x: module(x).sin().sum())(x), grad(lambda x: dense(x).sin().sum())(x))
    way = torch.randn(module(x).shape, generator=torch.Generator().manual_seed(2)).to(x)
    close(vjp(module, x)[1](way)[0], vjp(dense, x)[1](way)[0])
    close(jvp(module, (x,), (x.cos(),))[1], jvp(dense, (x,), (x.cos(),))[1])
    small = x.flatten()[: 6 * module.in_features].reshape(6, -1)
    close(jacrev(module)(small), jacrev(dense)(small))
    close(vmap(module)(x.reshape(2, -1, x.shape[-1])), dense(x).reshape(2, -1, module.out_features))
    close(hessian(lambda x: module(x).sin().sum())(small), hessian(lambda x: dense(x).sin().sum())(small))
    y = small.clone().requires_grad_()
    close(torch.autograd.functional.jacobian(module, y, vectorize=True), torch.autograd.functional.jacobian(dense, y, vectorize=True))


@pytest.mark.parametrize("inp, group, heads", [(36, 12, None), (30, 12, None)])
def test_transforms(no_kernels, inp, group, heads):
    check_transforms(linear(inp, 10, group, 8, heads=heads), torch.randn(14, inp, generator=torch.Generator().manual_seed(3)), 1e-5)


# (float32 against float32, sums of 128 and 136 products in another order: below 2 x 136 x 2^-24 of the magnitudes' sum, here at most 32 times a result's norm)
@pytest.mark.gpu
@pytest.mark.parametrize("inp, heads", [(128, None), (120, None), (128, 64)])
@pytest.mark.parametrize("bits", [8, 4])
def test_transforms_on_the_device(inp, heads, bits):
    module = linear(inp, 136, 128, bits, heads=heads, device="cuda")
    check_transforms(module, torch.randn(14, inp, generator=torch.Generator().manual_seed(3)).cuda(), 1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 6, 70, 300])
@pytest.mark.parametrize("inp, heads", [(128, None), (200, None), (192, 64)])
def test_differentiated_twice_on_the_device(inp, heads, rows, dtype):
    """d/dx of |d/dx (sum of y^2 / 2)|^2 / 2 = y W W^T W of the weight that the codes stand for."""
    module = linear(inp, 136, 128, 4, bias=False, heads=heads, dtype=dtype, device="cuda")
    x = torch.randn(rows, inp, generator=torch.Generator().manual_seed(rows)).to("cuda", dtype).requires_grad_()
    first, = torch.autograd.grad(module(x).float().square().sum() / 2, x, create_graph=True)
    got, = torch.autograd.grad(first.float().square().sum() / 2, x)
    weight = module._real_weight(dtype).double()
    u = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    # four products, each of sums in fp32 (at most 200 terms) rounded to the type, and what the later ones make of that
    want, tol, size = x.detach().double(), 0.0, torch.linalg.matrix_norm(weight, 2)
    for matrix in (weight.T, weight, weight.T, weight):
        sums = 208 * 2.0 ** -24 * (want.abs() @ matrix.abs()).norm()
        want = want @ matrix
        tol = tol * size + sums + u * (want.norm() + tol * size + sums)
    assert (got.double() - want).norm() <= tol


@pytest.mark.parametrize("inp, out, rows, dtype, plain", [
    (2048, 2048, 4, torch.float32, False), (2048, 2048, 64, torch.float32, False), (2048, 2048, 65, torch.float32, True), (2048, 2048, 320, torch.float32, True),
    (2048, 2048, 4095, torch.float32, True), (2048, 2048, 4096, torch.float32, False), (4096, 4096, 1023, torch.float32, True), (4096, 4096, 1024, torch.float32, False),
    (8192, 1024, 16, torch.float32, False), (8192, 1024, 17, torch.float32, True), (2048, 2048, 320, torch.bfloat16, False), (2048, 2048, 65, torch.float16, False)])
def test_where_the_gradient_is_torchs_own(no_kernels, inp, out, rows, dtype, plain):
    module = KernelQuantLinear(torch.zeros(out, inp // 128, 128, dtype=torch.int8), torch.ones(out, inp // 128), None,
                               QuantizationScheme(weights=QuantizationArgs(num_bits=8, strategy="group", group_size=128), input_activations=None), inp)
    assert module._plain(torch.empty(rows, inp, dtype=dtype, device="meta")) == plain
    assert module._plain(torch.empty(1, rows, inp, dtype=dtype, device="meta")) == plain
    a_scale_a_row = QuantizationScheme(weights=QuantizationArgs(num_bits=8, strategy="channel"), input_activations=None)
    module = KernelQuantLinear(torch.zeros(out, 1, inp, dtype=torch.int8), torch.ones(out, 1), None, a_scale_a_row, inp)
    assert module._plain(torch.empty(rows, inp, dtype=dtype, device="meta")) == plain


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 64, 65, 320, 321, 1023, 1030])
def test_one_gradient_on_both_sides(rows):
    """float32, the codes' gradient and torch's own against the weight in 64 bits."""
    module = linear(256, 136, 128, 8, device="cuda")
    x = torch.randn(rows, 256, generator=torch.Generator().manual_seed(rows)).cuda()
    way = torch.randn(rows, 136, generator=torch.Generator().manual_seed(1)).cuda()
    weight = module._real_weight(torch.float32).double()
    want, size = way.double() @ weight, way.double().abs() @ weight.abs()
    y = x.clone().requires_grad_()
    assert module._plain(y) == (rows > 64)
    for out in (module(y), _FrozenCodes.apply(y, module.bias, module)):
        with torch.no_grad():
            assert torch.equal(out, module(x))
        got, = torch.autograd.grad(out, y, way)
        assert ((got.double() - want).abs() <= (6 * 136 + 72) * 2.0 ** -24 * size + 2.0 ** -22 * size + 2.0 ** -23 * want.abs()).all()


def test_codes_from_inference_mode(no_kernels):
    """A model that was quantized in inference mode has gradients by its input."""
    with torch.inference_mode():
        module = linear(36, 10, 12, 8, bias=False)
    assert module.qdata.is_inference()
    x = torch.randn(6, 36, generator=torch.Generator().manual_seed(1), requires_grad=True)
    got, = torch.autograd.grad(_FrozenCodes.apply(x, None, module), x, torch.ones(6, 10))
    with torch.inference_mode():
        want = torch.ones(6, 10) @ module._real_weight(torch.float32)
    assert torch.allclose(got, want)


def test_codes_written_before_the_backward_pass_are_an_error(no_kernels):
    module = linear(36, 10, 12, 8)
    x = torch.randn(6, 36, generator=torch.Generator().manual_seed(1), requires_grad=True)
    out = _FrozenCodes.apply(x, module.bias, module)
    module.qdata.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
