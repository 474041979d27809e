"""Learning where sizes, strides and memory end: rows far apart, what a call touches beside its outputs. Bounds as in test_gpu_vocab_loss.py and
test_gpu_lora.py."""

import pytest
import torch
from test_gpu_learning_edges import ext, loss_and_gradients, same  # noqa: F401 (ext: a fixture)
from test_gpu_lora import call, call_grad, make
from test_gpu_vocab_loss import case, quantized

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def room():
    """6 GB of memory, for rows that lie far apart."""
    held = torch.zeros(3 << 30, dtype=torch.bfloat16, device="cuda")
    yield held
    del held
    torch.cuda.empty_cache()


def apart(room, rows, stride):
    """The same rows, `stride` elements from one to the next."""
    assert (rows.shape[0] - 1) * stride + rows.shape[1] <= room.numel()
    return room.view(rows.dtype).as_strided(rows.shape, (stride, 1)).copy_(rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, stride", [(129, 1 << 24), (160, 1 << 24), (300, 8421504), (300, 8421512), (66, 1 << 25)])
def test_rows_of_the_loss_far_apart(ext, room, rows, stride, dtype):  # noqa: F811
    """Tiles take rows that span 4 GiB and more from where they lie, each its own (a multiple of 2^24 elements apart, an offset that wraps falls on another row)."""
    c = case(rows, 515, 128, dtype, 0, rows)
    want = loss_and_gradients(ext, c)
    assert same(loss_and_gradients(ext, (apart(room, c[0], stride), *c[1:])), want)


@pytest.mark.parametrize("rows, stride", [(321, 8421504), (321, 8421512), (340, 9000000), (40, 1 << 25)])
def test_rows_of_a_linears_gradient_far_apart(ext, room, rows, stride):  # noqa: F811
    gen = torch.Generator(device="cuda").manual_seed(rows)
    stored, scale, _ = quantized(gen, 512, 256, 8)
    grad = torch.randn(rows, 512, generator=gen, device="cuda").bfloat16()
    want = ext.wq_linear_grad(grad, stored, scale)
    if rows <= 320:   # (few rows by their own offsets, of 64 bits, but not over 2^24 elements apart)
        with pytest.raises(RuntimeError, match="row stride"):
            ext.wq_linear_grad(apart(room, grad, stride), stored, scale)
        return
    assert torch.equal(ext.wq_linear_grad(apart(room, grad, stride), stored, scale), want)


def test_rows_of_a_request_far_apart(ext, room):  # noqa: F811
    c = make([25, 7], [1, 0], 2, 64, 128, 136, torch.bfloat16)
    low = torch.empty(32, 64, device="cuda")
    want = [call(ext, c, low=low), *call_grad(ext, c, low)]
    for stride in (93400000, 95443712):
        far = dict(c, x=apart(room, c["x"], stride))
        assert torch.equal(call(ext, far), want[0])
        assert torch.equal(call_grad(ext, dict(c, grad=apart(room, c["grad"], stride)), low)[0], want[1])
