"""Learning where sizes, types and memory end: rows far apart, weights of rows far apart, what a call touches beside its outputs. Bounds as in
test_gpu_vocab_loss.py and test_gpu_lora.py."""

import math
import random

import pytest
import torch
from test_gpu_learning_edges import ext, loss_and_gradients, same  # noqa: F401 (ext: a fixture)
from test_gpu_lora import backward as lora_backward
from test_gpu_lora import call, call_grad, make
from test_gpu_lora import close as lora_close
from test_gpu_vocab_loss import DTYPES, F32, U, case, close, dense_of, quantized, sum_error

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


def bounded(c, learned):
    """(dh, dW) in 64 bits with their bounds (those of test_gpu_vocab_loss.py), where an entry of P is off by half a step of the type and, in fp16, by at most half
    a step of 2^-38 of the power of two below |g|, the row's own or, where the weight learns, the largest."""
    hidden, _, _, dense, targets, grad = c
    dtype, (h, w, g) = hidden.dtype, (t.double() for t in (hidden, dense, grad))
    logits, size = h @ w.T, h.abs() @ w.abs().T
    d = (sum_error(h.shape[1], dtype) * size).amax(-1)
    lse = torch.logsumexp(logits, -1)
    lse_tol = d + (128 + len(w) / 256) * F32 + 4 * F32 * (lse.abs() + math.log(len(w)) + 20)
    p = torch.exp(logits - lse[:, None])
    part = p.clone()
    part[torch.arange(len(h), device="cuda"), targets] -= 1.0
    part *= g[:, None]
    p_tol = p * g.abs()[:, None] * (2 * (d + lse_tol) + 8 * F32)[:, None] + U[dtype] * 1.01 * part.abs()
    small = 0.0
    if dtype == torch.float16:
        power = torch.exp2(torch.floor(torch.log2(g.abs())))
        p_tol, small = p_tol + 2.0 ** -39 * (power.max() if learned else power[:, None]), 2.0 ** -25
    out = []
    for value, tol in ((part @ w, p_tol @ w.abs() + sum_error(len(w) + 64, dtype) * (part.abs() @ w.abs())),
                       (part.T @ h, p_tol.T @ h.abs() + sum_error(len(h) + 64, dtype) * (part.abs().T @ h.abs()))):
        out.append((value, tol + U[dtype] * (value.abs() + tol) + small))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("bits, spread", [(0, 10), (8, 10), (8, 20)])
def test_rows_of_unlike_weight(ext, bits, spread, rows, dtype):  # noqa: F811
    """Gradients of losses that count unlike, over a head with a common part in all its rows: what a row of little weight has of the softmax must not be lost
    beside the largest (p is about 2^-15 here), nor a token's row of dW that is no row's target."""
    vocab, width = 20011, 256
    gen = torch.Generator(device="cuda").manual_seed(rows + spread)
    common = 0.5 * torch.randn(width, generator=gen, device="cuda")
    weight, scale = (common + 0.05 * torch.randn(vocab, width, generator=gen, device="cuda")).to(dtype), None
    dense = weight
    if bits:
        codes = (weight.float() * 48).round().clamp(-128, 127).unflatten(1, (-1, 128))
        scale = (1 + torch.rand(vocab, width // 128, generator=gen, device="cuda")) / 64
        weight, dense = codes.to(torch.int8), dense_of(codes, scale, dtype)
    hidden = torch.randn(rows, width, generator=gen, device="cuda").to(dtype)
    targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    grad = 2.0 ** (6 if spread == 10 else 13) * torch.exp2(-spread * torch.rand(rows, generator=gen, device="cuda"))
    grad *= torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    c = hidden, weight, scale, dense, targets, grad
    for learned in (False, True)[: 1 if bits else 2]:
        _, _, dh, dw = loss_and_gradients(ext, c, learned)
        want = bounded(c, learned)
        close(dh, want[0], "dh")
        if learned:
            close(dw, want[1], "dW")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rank, lengths, adapters, slots", [
    (64, [1500], [700], 1024), (64, [1100, 1200], [40, 3], 64), (16, [4000, 0, 7, 4100], [9, 2, -1, 0], 12), (128, [1300, 900], [1, 1], 2), (8, [5000], [5], 6)])
def test_gradients_of_a_bank_with_idle_slots(ext, rank, lengths, adapters, slots, dtype):  # noqa: F811
    """Long slots among slots without rows, in pieces; zeros for the others. Where as many slots can have rows, as in a bank of their own."""
    c = make(lengths, adapters, slots, rank, 136, 128, dtype)
    low = torch.empty(sum(lengths), rank, device="cuda")
    call(ext, c, low=low)
    gx, ga, gb = call_grad(ext, c, low)
    used = sorted({a for a in adapters if a >= 0})
    if len(used) == len(adapters):   # (otherwise pieces may be of other lengths)
        alone = dict(c, lora_a=c["lora_a"][used].contiguous(), lora_b=c["lora_b"][used].contiguous(), scaling=c["scaling"][used].contiguous(),
                     adapter=torch.tensor([used.index(a) for a in adapters], dtype=torch.int32, device="cuda"))
        hx, ha, hb = call_grad(ext, alone, low)
        assert torch.equal(gx, hx) and torch.equal(ga[used], ha) and torch.equal(gb[used], hb)
    idle = [s for s in range(slots) if s not in used]
    assert not ga[idle].any() and not gb[idle].any()
    for got, pair in zip((gx, ga, gb), lora_backward(c, c["x"].double(), low, dtype, False)):
        lora_close(got, pair)


class Walled:
    """Memory in which every piece that is handed out has walls of a known pattern before and behind it."""

    WALL = 1 << 16

    def __init__(self, nbytes):
        self.held = torch.full((nbytes,), 0xA5, dtype=torch.uint8, device="cuda")
        self.at, self.pieces = 0, []

    def take(self, nbytes):
        begin = self.at + self.WALL
        self.at = (begin + nbytes + 255) // 256 * 256
        assert self.at + self.WALL <= self.held.numel()
        self.pieces.append((begin, begin + nbytes))
        return self.held.data_ptr() + begin

    def whole(self):
        at = 0
        for begin, end in [*self.pieces, (self.held.numel(), 0)]:
            if not bool((self.held[at:begin] == 0xA5).all()):
                return False
            at = end
        return True


def malformed(rows, sequences, seed):
    """Starts that decrease, repeat, leave the rows on both sides."""
    rng = random.Random(seed)
    edge = [0, rows, -9, rows + 50, -2 ** 31, 2 ** 31 - 1]
    return [rng.choice([rng.randint(0, rows), rng.randint(-rows, 2 * rows), *edge][: 2 + rng.randint(0, 6)]) for _ in range(sequences + 1)]


@pytest.mark.parametrize("rows, sequences, slots, rank", [(256, 8, 2, 8), (300, 70, 5, 64), (5000, 3, 9, 16), (4500, 130, 1, 128), (40, 200, 200, 16), (2500, 1, 3, 64)])
@pytest.mark.parametrize("seed", range(3))
def test_malformed_starts_write_within_what_a_call_was_given(rows, sequences, slots, rank, seed):
    """Nothing is promised of the results, but that no byte beside the outputs and the workspace changes: a wall on both sides of each, every start clamped to the
    rows, pieces, virtual rows and records counted from sizes alone."""
    from llmquant.hip.build import load_capi

    lib, bf16, inp, out = load_capi(), 2, 72, 136
    c = make([rows], [0], slots, rank, inp, out, torch.bfloat16)
    adapter = torch.tensor([random.Random(seed + 9).randint(-1, slots) for _ in range(sequences)], dtype=torch.int32, device="cuda")
    start = torch.tensor(malformed(rows, sequences, seed), dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    add = lib.llmq_lora_add_workspace_bytes(rows, sequences, 1, inp, rank, bf16)
    back = lib.llmq_lora_grad_workspace_bytes(rows, sequences, 1, inp, out, rank, slots, bf16)
    sizes = dict(out=2 * rows * out, low=4 * rows * rank, add=add, gx=2 * rows * inp, ga=2 * slots * rank * inp, gb=2 * slots * rank * out, back=back)
    room = Walled(sum(sizes.values()) + 16 * Walled.WALL)
    to = {name: room.take(n) for name, n in sizes.items()}
    weights = [c[k].data_ptr() for k in ("lora_a", "lora_b", "scaling")]
    assert lib.llmq_lora_add(c["x"].data_ptr(), inp, c["base"].data_ptr(), out, *weights, adapter.data_ptr(), start.data_ptr(), to["out"], to["low"], to["add"], add,
                             rows, sequences, inp, out, rank, slots, bf16, stream) == 0, lib.llmq_last_error()
    torch.cuda.synchronize()
    assert room.whole(), "lora_add"
    low = torch.randn(rows, rank, device="cuda")
    assert lib.llmq_lora_grad(c["grad"].data_ptr(), out, c["x"].data_ptr(), inp, None, low.data_ptr(), *weights, adapter.data_ptr(), start.data_ptr(),
                              c["grad_base"].data_ptr(), inp, to["gx"], to["ga"], to["gb"], to["back"], back, rows, sequences, inp, out, rank, slots, bf16,
                              stream) == 0, lib.llmq_last_error()
    torch.cuda.synchronize()
    assert room.whole(), "lora_grad"
