"""Cross entropy over a vocabulary and its gradient (vocab_loss, vocab_loss_grad), and the gradient of a quantized Linear
(wq_linear_grad), against the formulas in 64 bits.

Tolerances are bounds, element by element, of what the kernels may lose. u: half a step of the type (bf16 2^-8, fp16 2^-11,
fp32 2^-24). A sum of K products in fp32, in any order, is off by at most (K + 8) 2^-24 times the sum of their magnitudes; with
fp32 inputs the six products of planes make 6 K, and the three left out 2^-22 more at the most. A logit's bound is d; lse is off by the largest d
and by what exp, log and a sum of positive terms round (128 + V / 256 additions). P = (p - [target]) g is off by p g 2 d, by u of itself and,
in fp16, by half the smallest step (2^-25) times the power of two that g is scaled by. Results are sums of those, rounded once."""

import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
F32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ext():
    from llmquant.hip import load_extension

    return load_extension()


def quantized(gen, out, inp, bits, group=128, out_group=0):
    """(stored codes, scales, codes as float) of random values."""
    most = 127 if bits == 8 else 7
    codes = torch.randint(-most - 1, most + 1, (out, inp // group, group), generator=gen, device="cuda")
    rows = out if not out_group else -(-out // out_group)
    scale = torch.exp(0.3 * torch.randn(rows, inp // group, generator=gen, device="cuda")) * (0.05 / most)
    stored = codes.to(torch.int8)
    if bits == 4:
        biased = (codes + 8).to(torch.uint8)
        stored = biased[..., 0::2] | (biased[..., 1::2] << 4)
    return stored.contiguous(), scale, codes.float()


def dense_of(codes, scale, dtype, out_group=0):
    """The weight that codes and scales stand for: the fp32 product, rounded to the type."""
    rows = scale if not out_group else scale.repeat_interleave(out_group, 0)[: codes.shape[0]]
    return (codes * rows[..., None]).to(dtype).flatten(1)


def sum_error(terms, dtype):
    """Relative to the sum of magnitudes: what a sum of that many products loses."""
    if dtype == torch.float32:
        return (6 * terms + 8) * F32 + 2.0 ** -22
    return (terms + 8) * F32


def expected(hidden, weight, targets, grad, ignore, dtype):
    """Values in 64 bits and their bounds: (losses, lse, dh, dW), each a pair."""
    h, w = hidden.double(), weight.double()
    vocab, width = w.shape
    counted = targets != ignore
    safe = torch.where(counted, targets, 0)
    logits, size = h @ w.T, h.abs() @ w.abs().T
    d = (sum_error(width, dtype) * size).amax(-1)                        # of any logit of the row
    lse = torch.logsumexp(logits, -1)
    chosen = logits.gather(1, safe[:, None])[:, 0]
    losses = torch.where(counted, lse - chosen, 0.0)
    lse_tol = d + (128 + vocab / 256) * F32 + 4 * F32 * (lse.abs() + math.log(vocab) + 20)
    loss_tol = 2 * d + (128 + vocab / 256) * F32 + 4 * F32 * (losses.abs() + math.log(vocab) + 20)
    if grad is None:
        return (losses, loss_tol), (lse, lse_tol)
    g = torch.where(counted, grad.double(), 0.0)
    p = torch.exp(logits - lse[:, None])
    part = p.clone()
    part[torch.arange(len(safe), device=part.device), safe] -= 1.0
    part *= g[:, None]
    scale = 2.0 ** math.floor(math.log2(g.abs().max().item())) if g.abs().max() > 0 else 1.0
    p_tol = p * g.abs()[:, None] * (2 * (d + lse_tol) + 8 * F32)[:, None] + U[dtype] * 1.01 * part.abs()
    if dtype == torch.float16:
        p_tol = p_tol + torch.where(g != 0, scale * 2.0 ** -25, 0.0)[:, None]
    dh, dw = part @ w, part.T @ h
    dh_tol = p_tol @ w.abs() + sum_error(vocab + 64, dtype) * (part.abs() @ w.abs())
    dw_tol = p_tol.T @ h.abs() + sum_error(len(g) + 64, dtype) * (part.abs().T @ h.abs())
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return ((losses, loss_tol), (lse, lse_tol), (dh, dh_tol + U[dtype] * (dh.abs() + dh_tol) + small),
            (dw, dw_tol + U[dtype] * (dw.abs() + dw_tol) + small))


def close(got, want, what=""):
    value, tol = want
    off = (got.double() - value).abs()
    assert (off <= tol).all(), f"{what}: {(off - tol).max().item()} beyond, off by {off.max().item()}, {(off > tol).sum().item()} of {off.numel()}"


def case(rows, vocab, width, dtype, bits, seed, group=None, out_group=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if bits:
        group = group or (128 if width % 128 == 0 else 8)
        weight, scale, codes = quantized(gen, vocab, width, bits, group, out_group)
        dense = dense_of(codes, scale, dtype, out_group)
    else:
        weight = dense = (0.1 * torch.randn(vocab, width, generator=gen, device="cuda")).to(dtype)
        scale = None
    targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    hidden = torch.randn(rows, width, generator=gen, device="cuda")
    hidden = (hidden + 6 * torch.rand(rows, 1, generator=gen, device="cuda") * dense[targets].float()).to(dtype)
    grad = torch.randn(rows, generator=gen, device="cuda") / max(rows, 1)
    return hidden, weight, scale, dense, targets, grad


SIZES = [(1, 8, 8), (3, 300, 72), (64, 256, 64), (65, 257, 128), (130, 1000, 256), (17, 5003, 200), (300, 771, 96), (1, 40000, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("rows, vocab, width", SIZES)
def test_loss_and_gradients(ext, rows, vocab, width, bits, dtype):
    hidden, weight, scale, dense, targets, grad = case(rows, vocab, width, dtype, bits, rows + vocab)
    if rows > 2:
        targets[::3] = -100
    losses, lse = ext.vocab_loss(hidden, weight, targets, -100, scale)
    want = expected(hidden, dense, targets, grad, -100, dtype)
    close(losses, want[0], "losses")
    close(lse, want[1], "lse")
    assert (losses[targets == -100] == 0).all()
    dh, dw = ext.vocab_loss_grad(hidden, weight, targets, lse, grad, -100, scale, 0, not bits)
    close(dh, want[2], "dh")
    assert (dh[targets == -100] == 0).all()
    if bits:
        assert dw is None
    else:
        close(dw, want[3], "dw")
        again, none = ext.vocab_loss_grad(hidden, weight, targets, lse, grad, -100)
        assert none is None and torch.equal(again, dh)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, out, width, bits, group, keep, out_group", [
    (1, 8, 128, 8, 128, 128, 0), (5, 64, 256, 4, 128, 128, 0), (64, 200, 384, 8, 128, 64, 0), (65, 512, 128, 4, 128, 128, 64),
    (300, 136, 640, 4, 64, 64, 0), (700, 1032, 512, 8, 128, 128, 0), (257, 2048, 264, 8, 8, 8, 0),
])
def test_linear_grad(ext, rows, out, width, bits, group, keep, out_group, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    stored, scale, codes = quantized(gen, out, width, bits, group, out_group)
    weight = dense_of(codes, scale, dtype, out_group).unflatten(1, (-1, group))[..., :keep].flatten(1).double()
    grad = torch.randn(rows, out, generator=gen, device="cuda").to(dtype)
    got = ext.wq_linear_grad(grad, stored, scale, out_group, keep)
    want, size = grad.double() @ weight, grad.double().abs() @ weight.abs()
    tol = sum_error(out + 64, dtype) * size
    close(got, (want, tol + U[dtype] * (want.abs() + tol)))
