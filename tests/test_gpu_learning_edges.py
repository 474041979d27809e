"""Where the operators of learning can go wrong: few rows past a weight as it lies, rows that do not count, garbage in masked places, strides, offsets past
32 bits, captured calls, other streams, repeated calls, refusals. Bounds are those of test_gpu_vocab_loss.py and test_gpu_lora.py."""

import math

import pytest
import torch
from test_gpu_lora import backward as lora_backward
from test_gpu_lora import call, call_grad, make
from test_gpu_lora import close as lora_close
from test_gpu_lora import forward as lora_forward
from test_gpu_vocab_loss import DTYPES, U, case, close, dense_of, expected, quantized, sum_error

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.fixture(scope="module")
def ext():
    from llmquant.hip import load_extension

    return load_extension()


def loss_and_gradients(ext, c, want_weight=None, ignore=-100, out_group=0):
    hidden, weight, scale, _, targets, grad = c
    losses, lse = ext.vocab_loss(hidden, weight, targets, ignore, scale, out_group)
    learned = scale is None if want_weight is None else want_weight
    dh, dw = ext.vocab_loss_grad(hidden, weight, targets, lse, grad, ignore, scale, out_group, learned)
    return losses, lse, dh, dw


def same(a, b):
    return all((x is None and y is None) or torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def replays(work, change, outputs_of, times=3):
    """Captures work(), replays it after each change(i) and checks every replay against an eager run, with eager work between."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for i in range(times):
        change(i)
        graph.replay()
        torch.cuda.synchronize()
        got = [None if t is None else t.clone() for t in outputs_of(captured)]
        assert same(got, outputs_of(work())), f"replay {i}"
    return graph, captured


# ---- few rows -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("rows, vocab, width, group, out_group", [
    (1, 1, 128, 128, 0), (1, 63, 256, 128, 0), (16, 64, 128, 128, 0), (17, 1000, 384, 384, 0), (33, 2049, 256, 128, 0), (64, 5003, 512, 256, 0),
    (48, 129, 1024, 128, 64), (31, 8191, 256, 128, 100), (2, 70001, 128, 128, 0),
    (65, 700, 192, 64, 0), (100, 3001, 256, 256, 0), (128, 515, 384, 128, 7), (129, 515, 384, 128, 0), (300, 130, 128, 128, 0), (512, 333, 256, 128, 0),
    (513, 333, 256, 128, 0)])
def test_few_rows(ext, rows, vocab, width, group, out_group, bits, dtype):
    c = case(rows, vocab, width, dtype, bits, rows * vocab, group, out_group if bits else 0)
    hidden, weight, scale, dense, targets, grad = c
    if rows > 4:
        targets[1::4] = -100
    losses, lse, dh, dw = loss_and_gradients(ext, c, out_group=out_group if bits else 0)
    want = expected(hidden, dense, targets, grad, -100, dtype)
    for got, pair, what in zip((losses, lse, dh, dw), want, ("losses", "lse", "dh", "dW")):
        if got is not None:
            close(got, pair, what)
    assert (dh[targets == -100] == 0).all() and (losses[targets == -100] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, out, width, bits, group, keep, out_group", [
    (1, 4104, 256, 8, 128, 128, 0), (16, 24, 128, 4, 8, 8, 0), (17, 136, 384, 8, 128, 72, 0), (33, 1032, 128, 4, 128, 128, 100), (48, 8, 2048, 8, 64, 64, 0),
    (128, 2056, 256, 4, 256, 256, 0), (129, 520, 136, 8, 8, 8, 3), (256, 264, 1024, 8, 128, 128, 0), (257, 264, 1024, 8, 128, 128, 0), (320, 2056, 256, 4, 128, 128, 0),
    (321, 264, 256, 8, 128, 128, 0)])
def test_few_rows_of_a_linear(ext, rows, out, width, bits, group, keep, out_group, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows + out)
    stored, scale, codes = quantized(gen, out, width, bits, group, out_group)
    weight = dense_of(codes, scale, dtype, out_group).unflatten(1, (-1, group))[..., :keep].flatten(1).double()
    grad = torch.randn(rows, out, generator=gen, device="cuda").to(dtype)
    got = ext.wq_linear_grad(grad, stored, scale, out_group, keep)
    tol = sum_error(out + 64, dtype) * (grad.double().abs() @ weight.abs())
    want = grad.double() @ weight
    close(got, (want, tol + U[dtype] * (want.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0.0)))
    bad = grad.clone()
    bad[rows // 2] = NAN
    other = ext.wq_linear_grad(bad, stored, scale, out_group, keep)
    assert other[rows // 2].isnan().all()
    rest = torch.arange(rows, device="cuda") != rows // 2
    assert torch.equal(other[rest], got[rest])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("rows", [1, 20, 64, 65, 700])
@pytest.mark.parametrize("same", [False, True])
def test_a_target_loses_nothing_to_rounding(ext, rows, bits, dtype, same):
    """Logits near each other: P is (p - [target]) g with p of about 1 / 3000, and the entries of the targets, which rounding to 16 bits would leave u off, are
    nearly all of it. What is left over the results' own rounding is the others' u p, together below u / 50 (their 3000 independent errors of at most u / 3000 each)."""
    vocab, width = 3000, 256
    hidden, weight, scale, dense, targets, grad = case(rows, vocab, width, dtype, bits, rows)
    hidden = (hidden / 64).to(dtype)
    if same:
        targets[:] = 1717   # (all rows on one token: its row of dW has a term from each)
    grad = torch.full_like(grad, 1 / 1.37)
    _, _, dh, dw = loss_and_gradients(ext, (hidden, weight, scale, dense, targets, grad))
    want = expected(hidden, dense, targets, grad, -100, dtype)
    for got, (value, _) in ((dh, want[2]), (dw, want[3])):
        if got is not None:
            own = (value.to(dtype).double() - value).norm()
            assert (got.double() - value).norm() <= 1.05 * own + 0.02 * U[dtype] * value.norm()


# ---- rows that do not count -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("rows", [3, 40, 300])
@pytest.mark.parametrize("garbage", [NAN, float("inf"), -float("inf"), "lowest"])
def test_garbage_in_rows_that_do_not_count(ext, rows, bits, dtype, garbage):
    c = case(rows, 700, 256, dtype, bits, rows)
    hidden, weight, scale, dense, targets, grad = c
    targets[::2] = -100
    clean = loss_and_gradients(ext, c)
    hidden = hidden.clone()
    hidden[::2] = torch.finfo(dtype).min if garbage == "lowest" else garbage
    grad = grad.clone()
    grad[::2] = NAN
    dirty = loss_and_gradients(ext, (hidden, weight, scale, dense, targets, grad))
    counted = targets != -100
    assert torch.equal(dirty[0], clean[0]) and torch.equal(dirty[1][counted], clean[1][counted])
    assert torch.equal(dirty[2], clean[2])
    assert bits or torch.equal(dirty[3], clean[3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [5, 100])
def test_targets_outside_make_nan_of_their_own_row(ext, rows, dtype):
    c = case(rows, 500, 128, dtype, 8, 1)
    good = loss_and_gradients(ext, c)
    hidden, weight, scale, dense, targets, grad = c
    wrong = targets.clone()
    for row, target in ((0, 500), (1, -1), (2, 1 << 40), (3, -(1 << 62))):
        wrong[row] = target
    losses, lse, dh, _ = loss_and_gradients(ext, (hidden, weight, scale, dense, wrong, grad))
    assert losses[:4].isnan().all() and dh[:4].isnan().all()
    assert torch.equal(lse, good[1]) and torch.equal(losses[4:], good[0][4:]) and torch.equal(dh[4:], good[2][4:])
    inside = loss_and_gradients(ext, (hidden, weight, scale, dense, targets, grad), ignore=int(targets[0]))   # ignore_index may be a token
    assert (inside[0][targets == targets[0]] == 0).all() and (inside[2][targets == targets[0]] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [0, 1, 7, 64, 90])
def test_no_row_counts(ext, rows, dtype):
    c = case(rows, 300, 64, dtype, 0, 1)
    c[4].fill_(-100)
    losses, _, dh, dw = loss_and_gradients(ext, c)
    assert losses.shape == (rows,) and (losses == 0).all() and dh.shape == (rows, 64) and (dh == 0).all() and (dw == 0).all()
    if rows:
        hidden, weight, scale, dense, targets, grad = case(rows, 300, 64, dtype, 0, 1)
        _, _, dh, dw = loss_and_gradients(ext, (hidden, weight, scale, dense, targets, torch.zeros_like(grad)))
        assert (dh == 0).all() and (dw == 0).all()


# ---- magnitudes -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [5, 130])
@pytest.mark.parametrize("size, grad_size", [(1000.0, 1.0), (30.0, 1e-9), (0.01, 3e5), (1.0, 1e30)])
def test_large_logits_and_far_gradients(ext, rows, size, grad_size):
    """fp16 gradients beyond its range where they come out so; P's own range is a power of two away from the gradients'."""
    dtype = torch.float16
    hidden, weight, scale, dense, targets, grad = case(rows, 400, 128, dtype, 0, 3)
    hidden = (hidden.float() * size / 10).clamp(-60000, 60000).to(dtype)
    grad = grad * grad_size
    losses, lse, dh, dw = loss_and_gradients(ext, (hidden, weight, scale, dense, targets, grad))
    want = expected(hidden, dense, targets, grad, -100, dtype)
    close(losses, want[0], "losses")
    close(lse, want[1], "lse")
    for got, (value, tol) in ((dh, want[2]), (dw, want[3])):
        inside = value.abs() + tol < 65000
        assert ((got.double() - value).abs() <= tol)[inside].all()
        assert got[value.abs() - tol > 65536].isinf().all()


def test_differences(ext):
    """The gradients against central differences of the losses: fp32, in which the losses' own rounding (2e-6) over the step leaves 2e-6 / 2 h."""
    from llmquant.hip import vocab_cross_entropy

    gen = torch.Generator(device="cuda").manual_seed(5)
    hidden = torch.randn(9, 64, generator=gen, device="cuda", requires_grad=True)
    weight = (0.3 * torch.randn(203, 64, generator=gen, device="cuda")).requires_grad_()
    targets = torch.randint(0, 203, (9,), generator=gen, device="cuda")
    targets[4] = -100
    vocab_cross_entropy(hidden, weight, targets).backward()
    h = 2.0 ** -6
    for leaf in (hidden, weight):
        way = torch.randn(leaf.shape, generator=gen, device="cuda")
        way /= way.norm()
        with torch.no_grad():
            sides = [vocab_cross_entropy(*(t + s * h * way if t is leaf else t for t in (hidden, weight)), targets).double() for s in (1, -1)]
        slope = (sides[0] - sides[1]) / (2 * h)
        assert abs(slope - (leaf.grad.double() * way.double()).sum()) < 2e-6 / h + h * h


# ---- strides, offsets -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [6, 130])
def test_strided_expanded_and_odd_tensors(ext, rows, dtype):
    c = case(rows, 260, 128, dtype, 0, 11)
    hidden, weight, _, dense, targets, grad = c
    want = loss_and_gradients(ext, c)
    wide = torch.full((rows, 3, 136), NAN, dtype=dtype, device="cuda")
    wide[:, 1, :128] = hidden
    odd = torch.empty(rows * 128 + 1, dtype=dtype, device="cuda")[1:].view(rows, 128).copy_(hidden)
    turned = hidden.t().contiguous().t()
    spread = torch.zeros(rows, 5, dtype=torch.long, device="cuda")
    spread[:, 2] = targets
    for h in (wide[:, 1, :128], odd, turned):
        assert same(loss_and_gradients(ext, (h, weight, None, dense, spread[:, 2], grad)), want)
    one = grad[:1].expand(rows)   # as sum().backward() gives it
    row = hidden[:1].expand(rows, 128)
    assert same(loss_and_gradients(ext, (row, weight, None, dense, targets, one)),
                loss_and_gradients(ext, (row.contiguous(), weight, None, dense, targets, one.contiguous())))
    stored, scale, _ = quantized(torch.Generator(device="cuda").manual_seed(2), 128, 256, 8)
    got = ext.wq_linear_grad(hidden, stored, scale)
    for h in (wide[:, 1, :128], odd, turned):
        assert torch.equal(ext.wq_linear_grad(h, stored, scale), got)


@pytest.mark.parametrize("rows", [3, 70])
def test_a_vocabulary_past_32_bits(ext, rows):
    """2^31.2 elements, zeros but for the first and last hundred rows: the zeros have logits of nothing and no part in dh."""
    dtype, vocab, width = torch.bfloat16, 610_000, 4096
    gen = torch.Generator(device="cuda").manual_seed(rows)
    weight = torch.zeros(vocab, width, dtype=dtype, device="cuda")
    weight[:100] = 0.05 * torch.randn(100, width, generator=gen, device="cuda")
    weight[-100:] = 0.05 * torch.randn(100, width, generator=gen, device="cuda")
    hidden = torch.randn(rows, width, generator=gen, device="cuda").to(dtype)
    targets = torch.randint(0, 100, (rows,), generator=gen, device="cuda")
    targets[1::2] += vocab - 100
    grad = torch.ones(rows, device="cuda")
    losses, lse = ext.vocab_loss(hidden, weight, targets, -100)
    dh, none = ext.vocab_loss_grad(hidden, weight, targets, lse, grad, -100)
    some = torch.cat([weight[:100], weight[-100:]]).double()
    h = hidden.double()
    logits = h @ some.T
    want = torch.logsumexp(torch.cat([logits, torch.full((rows, 1), math.log(vocab - 200), device="cuda", dtype=torch.float64)], 1), -1)
    at = torch.where(targets < 100, targets, targets - vocab + 200)
    d = (sum_error(width, dtype) * (h.abs() @ some.abs().T)).amax()
    far = 2 * d + (128 + vocab / 64) * 2.0 ** -24 + 1e-5
    assert ((lse - want).abs() < far).all() and ((losses - (want - logits[torch.arange(rows), at])).abs() < 2 * far).all()
    p = torch.exp(logits - want[:, None])
    part = p.clone()
    part[torch.arange(rows), at] -= 1
    value = part @ some
    tol = (4 * far * p + 1.01 * U[dtype] * part.abs()) @ some.abs() + sum_error(vocab, dtype) * (part.abs() @ some.abs())
    close(dh, (value, tol + U[dtype] * (value.abs() + tol)), "dh")


# ---- captured, on other streams, again ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows, bits", [(7, 0), (40, 4), (200, 0), (200, 8)])
def test_captured_losses(ext, rows, bits, dtype):
    c = case(rows, 1300, 256, dtype, bits, 21)
    gen = torch.Generator(device="cuda").manual_seed(22)

    def change(i):
        c[0].copy_(torch.randn(c[0].shape, generator=gen, device="cuda"))
        c[4].copy_(torch.randint(0, 1300, (rows,), generator=gen, device="cuda"))
        c[4][: i * rows // 3] = -100
        c[5].copy_(torch.randn(rows, generator=gen, device="cuda"))

    first = replays(lambda: loss_and_gradients(ext, c), change, list)
    second = replays(lambda: loss_and_gradients(ext, c), change, list)   # two graphs of the same inputs, a workspace each
    for i in range(2):
        change(i)
        first[0].replay()
        second[0].replay()
        torch.cuda.synchronize()
        assert same(first[1], second[1]) and same(first[1], loss_and_gradients(ext, c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [9, 300])
def test_captured_gradient_of_a_linear(ext, rows, dtype):
    gen = torch.Generator(device="cuda").manual_seed(3)
    stored, scale, _ = quantized(gen, 264, 512, 8)
    grad = torch.randn(rows, 264, generator=gen, device="cuda").to(dtype)
    replays(lambda: [ext.wq_linear_grad(grad, stored, scale)], lambda i: grad.copy_(torch.randn(rows, 264, generator=gen, device="cuda")), list)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("codes", [False, True])
def test_captured_adapters(ext, codes, dtype):
    """Who has which adapter, and whose rows are whose, change between replays."""
    c = make([40, 1, 30, 9, 0, 48], [0, 1, -1, 2, 1, 0], 3, 16, 256, 136, dtype)
    low = torch.empty(128, 16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(9)
    spans = [[0, 1, 2, 3, 4, 5, 128], [0, 0, 0, 0, 100, 128, 128], [5, 30, 31, 60, 70, 71, 120]]

    def work():
        out = call(ext, c, low=low)
        if codes:
            stored, scale = ext.quant_group_codes(c["x"], 8, 128)
            grads = call_grad(ext, c, low, x=stored, x_scale=scale)
        else:
            grads = call_grad(ext, c, low, grad_base=c["grad_base"])
        return [out, low.clone(), *grads]

    def change(i):
        c["x"].copy_(torch.randn(c["x"].shape, generator=gen, device="cuda"))
        c["adapter"].copy_(torch.randint(-1, 4, (6,), generator=gen, device="cuda"))
        c["query_start"].copy_(torch.tensor(spans[i % 3], dtype=torch.int32))

    replays(work, change, list)


def test_a_captured_step_of_autograd(ext):
    from llmquant.hip import vocab_cross_entropy

    gen = torch.Generator(device="cuda").manual_seed(1)
    hidden = torch.randn(50, 256, generator=gen, device="cuda").bfloat16().requires_grad_()
    weight = (0.1 * torch.randn(999, 256, generator=gen, device="cuda")).bfloat16().requires_grad_()
    targets = torch.randint(0, 999, (50,), generator=gen, device="cuda")
    upstream = torch.rand(50, generator=gen, device="cuda")

    def work():
        losses = vocab_cross_entropy(hidden, weight, targets, reduction="none")
        return [losses.detach(), *torch.autograd.grad(losses, (hidden, weight), upstream)]

    replays(work, lambda i: upstream.copy_(torch.rand(50, generator=gen, device="cuda")), list)


@pytest.mark.parametrize("rows", [12, 150])
def test_on_another_stream_and_again(ext, rows):
    c = case(rows, 1500, 256, torch.bfloat16, 0, 31)
    a = make([rows], [0], 1, 16, 256, 512, torch.bfloat16)
    low = torch.empty(rows, 16, device="cuda")
    stored, scale, _ = quantized(torch.Generator(device="cuda").manual_seed(4), 512, 256, 4)

    def work():
        out = call(ext, a, low=low)
        return [*loss_and_gradients(ext, c), out, *call_grad(ext, a, low), ext.wq_linear_grad(a["grad"], stored, scale)]

    want = work()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(10_000_000)
        got = work()
    side.synchronize()
    assert same(got, want)
    for _ in range(3):
        assert same(work(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows, slots, rank, inp, out", [
    (1, 2, 16, 2048, 2056), (5, 3, 24, 72, 513 * 8), (64, 48, 16, 4096, 4096), (65, 48, 16, 4096, 4096), (600, 2, 8, 64, 8), (3, 2, 128, 512, 1000),
    (3, 2, 128, 520, 1000), (2, 1, 8, 8, 8), (11, 5, 40, 1032, 264)])
def test_single_rows_in_one_launch_and_in_two(ext, rows, slots, rank, inp, out, dtype):
    adapters = [(5 * b) % (slots + 2) - 1 for b in range(rows)]
    c = make([1] * rows, adapters, slots, rank, inp, out, dtype, seed=rank, step=True)
    low = torch.full((rows, rank), NAN, device="cuda")
    got = call(ext, c, low=low)
    want, want_low = lora_forward(c, dtype)
    lora_close(low, want_low, "low")
    lora_close(got, want, "out")
    nobody = torch.tensor([not 0 <= a < slots for a in adapters], device="cuda")
    assert torch.equal(got[nobody], c["base"][nobody]) and (low[nobody] == 0).all()
    in_place = c["base"].clone()
    call(ext, dict(c, base=in_place), out=in_place)
    assert torch.equal(in_place, got)
    c["x"][nobody] = NAN
    assert torch.equal(call(ext, c), got)


# ---- adapters -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_of_nobody(ext, dtype):
    """Rows in front of the first request, behind the last, and of requests without an adapter: base to the bit, whatever x holds there, and no part in
    the banks' gradients."""
    lengths, adapters = [7, 30, 12, 50, 11], [-1, 1, -5, 0, 2]
    c = make(lengths, adapters, 3, 16, 128, 264, dtype)
    start = c["query_start"]
    start[0], start[-1] = 7, 99   # rows 0 .. 6 and 99 .. of no request; adapter of the last: 2, with no row left
    start[1] = 7
    nobody = torch.ones(110, dtype=torch.bool, device="cuda")
    nobody[7:37] = nobody[49:99] = False
    clean = call(ext, c)
    want, want_low = lora_forward(c, dtype)
    c["x"][nobody], c["grad"][nobody] = NAN, float("inf")
    c["base"][nobody] = -0.0
    low = torch.full((110, 16), NAN, device="cuda")
    out = call(ext, c, low=low)
    assert torch.equal(out[~nobody], clean[~nobody])
    lora_close(out[~nobody], (want[0][~nobody], want[1][~nobody]) if isinstance(want, tuple) else want, "out")
    assert torch.equal(out[nobody].view(torch.uint8), c["base"][nobody].view(torch.uint8))
    assert (low[nobody] == 0).all()
    low[nobody] = NAN
    gx, ga, gb = call_grad(ext, c, low, grad_base=c["grad_base"])
    assert torch.equal(gx[nobody], c["grad_base"][nobody])
    assert (call_grad(ext, c, low)[0][nobody] == 0).all()
    c["x"][nobody], c["grad"][nobody], low[nobody] = 0, 0, 0
    wants = lora_backward(c, c["x"].double(), low, dtype)
    lora_close(ga, wants[1], "gA")
    lora_close(gb, wants[2], "gB")
    assert (ga[2] == 0).all() and (gb[2] == 0).all()


@pytest.mark.parametrize("rank", [8, 32, 64, 128])
@pytest.mark.parametrize("lengths", [[1, 20, 3], [200]])
@pytest.mark.parametrize("tiny", [False, True])
def test_rows_of_unlike_magnitude_in_half(ext, lengths, rank, tiny):
    """fp16 rows from 2^-20 to 2^12 and banks down to its subnormal numbers: what lies between the two products has an exponent of its own for each row."""
    dtype = torch.float16
    c = make(lengths, list(range(len(lengths))), len(lengths), rank, 256, 264, dtype, seed=rank)
    rows = sum(lengths)
    gen = torch.Generator(device="cuda").manual_seed(rank)
    size = 2.0 ** torch.randint(-20, 10, (rows, 1), generator=gen, device="cuda")
    c["x"] = (c["x"].float() * size).to(dtype)
    c["base"].zero_()
    c["lora_b"] = (c["lora_b"].float() * (1e-6 if tiny else 1e-2)).to(dtype)
    c["scaling"] = c["scaling"] * (300.0 if tiny else 0.01)
    low = torch.empty(rows, rank, device="cuda")
    out = call(ext, c, low=low)
    want, want_low = lora_forward(c, dtype)
    lora_close(low, want_low, "low")
    lora_close(out, want, "out")
    c["x"][0, 0] = float("inf")
    bad = call(ext, c)
    assert bad[0].isnan().any() and torch.equal(bad[1:], out[1:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("lengths, adapters, slots, rank", [
    ([1030], [0], 1, 24), ([1000, 20], [1, 0], 2, 40), ([700, 700, 700], [0, 2, 0], 4, 72), ([1500, 1300], [0, 1], 2, 128), ([2500], [2], 3, 64), ([2100, 1, 3], [1, 1, 0], 2, 16),
    ([5, 900], [3, 1], 5, 8)])
def test_gradients_of_banks_in_one_piece_and_in_several(ext, lengths, adapters, slots, rank, codes, dtype):
    """Around 1024 rows a slot and 1024 and 2048 rows together, where the sums over rows are cut otherwise; slots without rows are zero."""
    c = make(lengths, adapters, slots, rank, 256, 136, dtype, seed=rank)
    low = torch.empty(sum(lengths), rank, device="cuda")
    call(ext, c, low=low)
    values, more = c["x"].double(), {}
    if codes:
        stored, scale = ext.quant_group_codes(c["x"], 8, 128)
        values, more = (stored.double().unflatten(1, (-1, 128)) * scale.double()[..., None]).flatten(1), dict(x=stored, x_scale=scale)
    grads = call_grad(ext, c, low, grad_base=c["grad_base"], **more)
    for got, pair, what in zip(grads, lora_backward(c, values, low, dtype), ("gx", "gA", "gB")):
        lora_close(got, pair, what)
    for slot in set(range(slots)) - set(adapters):
        assert (grads[1][slot] == 0).all() and (grads[2][slot] == 0).all()
    assert same(call_grad(ext, c, low, grad_base=c["grad_base"], **more), grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_slots_no_rows_no_requests(ext, dtype):
    c = make([3, 2], [0, 1], 0, 8, 64, 72, dtype)
    assert torch.equal(call(ext, c), c["base"])
    gx, ga, gb = call_grad(ext, c, torch.zeros(5, 8, device="cuda"), grad_base=c["grad_base"])
    assert torch.equal(gx, c["grad_base"]) and ga.shape == (0, 8, 64) and gb.shape == (0, 72, 8)
    c = make([0, 0], [0, 1], 2, 8, 64, 72, dtype)
    assert call(ext, c).shape == (0, 72)
    gx, ga, gb = call_grad(ext, c, torch.zeros(0, 8, device="cuda"))
    assert gx.shape == (0, 64) and (ga == 0).all() and (gb == 0).all()
    c = make([4], [0], 2, 8, 64, 72, dtype)
    c["adapter"], c["query_start"] = c["adapter"][:0], c["query_start"][:1]
    low = torch.full((4, 8), NAN, device="cuda")
    assert torch.equal(call(ext, c, low=low), c["base"]) and (low == 0).all()
    gx, ga, gb = call_grad(ext, c, low)
    assert (gx == 0).all() and (ga == 0).all() and (gb == 0).all()
    c["adapter"], c["query_start"] = torch.tensor([-2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    assert torch.equal(call(ext, c), c["base"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_rows_of_adapters(ext, dtype):
    c = make([40, 25], [1, 0], 2, 16, 128, 136, dtype)
    low = torch.empty(65, 16, device="cuda")
    want, grads = call(ext, c, low=low), None
    grads = call_grad(ext, c, low, grad_base=c["grad_base"])
    for kind in ("wide", "odd", "turned"):
        d = dict(c)
        for name in ("x", "base", "grad", "grad_base"):
            t = c[name]
            if kind == "wide":
                room = torch.full((65, 2, t.shape[1] + 8), NAN, dtype=dtype, device="cuda")
                room[:, 1, :t.shape[1]] = t
                d[name] = room[:, 1, :t.shape[1]]
            elif kind == "odd":
                d[name] = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t)
            else:
                d[name] = t.t().contiguous().t()
        assert torch.equal(call(ext, d), want), kind
        assert same(call_grad(ext, d, low, grad_base=d["grad_base"]), grads), kind
    one = dict(c, grad=c["grad"][:1].expand(65, 136))
    assert same(call_grad(ext, one, low), call_grad(ext, dict(c, grad=one["grad"].contiguous()), low))


def test_differences_of_adapters():
    """_LoraAdd against central differences, fp32; the function is of third order in all of its inputs together, so that the step's error is of h^2."""
    from llmquant.quantizers.adapters import _LoraAdd

    c = make([5, 0, 20, 3], [1, 0, -1, 0], 2, 8, 40, 24, torch.float32)
    leaves = {k: c[k].clone().requires_grad_() for k in ("x", "base", "lora_a", "lora_b")}
    upstream = c["grad"] / c["grad"].norm()

    def value(t):
        out = _LoraAdd.apply(t["x"], t["base"], t["lora_a"], t["lora_b"], c["scaling"], c["adapter"], c["query_start"], 16)
        return (out.double() * upstream.double()).sum()

    value(leaves).backward()
    gen = torch.Generator(device="cuda").manual_seed(0)
    h = 2.0 ** -5
    for name, leaf in leaves.items():
        way = torch.randn(leaf.shape, generator=gen, device="cuda")
        way /= way.norm()
        with torch.no_grad():
            slope = (value(dict(leaves, **{name: leaf + h * way})) - value(dict(leaves, **{name: leaf - h * way}))) / (2 * h)
        # (linear in each: what is left is the rounding of the outputs, 2^-24 of values of a few units with weights of norm 1)
        assert abs(slope - (leaf.grad.double() * way.double()).sum()) < 2.0 ** -20 / h, name


def test_starts_that_decrease_stay_within_their_memory(ext):
    """Not allowed, and nothing is promised of the results; what they touch is the outputs', and the next call is right."""
    c = make([32] * 8, [0, 1] * 4, 2, 8, 64, 64, torch.bfloat16)
    good = c["query_start"].clone()
    low = torch.empty(256, 8, device="cuda")
    want = [call(ext, c, low=low), *call_grad(ext, c, low)]
    c["query_start"] = torch.tensor([0, 256, 0, 256, -9, 300, 0, 256, 0], dtype=torch.int32, device="cuda")
    call(ext, c, low=low)
    call_grad(ext, c, low)
    torch.cuda.synchronize()
    c["query_start"] = good
    assert same([call(ext, c, low=low), *call_grad(ext, c, low)], want)


def test_copied_and_saved_banks():
    """A copy of a model has banks and requests of its own; a state dict holds the banks."""
    import copy

    from llmquant.quantizers import add_adapters, adapter_parameters, use_adapters
    from test_gpu_adapters import build

    _, model = build(torch.float32, layers=1)
    add_adapters(model, rank=8, slots=2)
    gen = torch.Generator(device="cuda").manual_seed(0)
    with torch.no_grad():
        for p in adapter_parameters(model):
            p.copy_(0.05 * torch.randn(p.shape, generator=gen, device="cuda"))
    ids = torch.randint(0, 1000, (2, 9), generator=gen, device="cuda")
    use_adapters(model, [0, 1])
    with torch.no_grad():
        want = model(ids).logits
        twin = copy.deepcopy(model)
        use_adapters(twin, [-1, -1])
        bare = twin(ids).logits
        assert torch.equal(model(ids).logits, want) and not torch.equal(bare, want)
        use_adapters(twin, [0, 1])
        assert torch.equal(twin(ids).logits, want)
        _, other = build(torch.float32, layers=1)
        add_adapters(other, rank=8, slots=2)
        banks = {k: v for k, v in model.state_dict().items() if "adapters" in k}
        missing, unexpected = other.load_state_dict(banks, strict=False)
        assert not unexpected and not any("adapters" in k for k in missing) and len(banks) == 3 * 7
        use_adapters(other, [0, 1])
        assert torch.equal(other(ids).logits, want)


def test_a_captured_step_keeps_the_starts_it_reads():
    from llmquant.quantizers.adapters import AdapterBatch, LoraAdapters

    batch = AdapterBatch("cuda")
    bank = LoraAdapters(64, 64, 8, 2, 16.0, torch.bfloat16, "cuda", batch).requires_grad_(False)
    gen = torch.Generator(device="cuda").manual_seed(0)
    bank.lora_b.copy_(torch.randn(bank.lora_b.shape, generator=gen, device="cuda"))
    x, base = (torch.randn(12, 64, generator=gen, device="cuda").bfloat16() for _ in range(2))
    batch.select([0, 1], torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda"))
    want = bank(x, base.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = bank(x, base.clone())
    batch.select([1, 0])   # (the tensor of starts is nobody's else)
    noise = [torch.full((3,), 7, dtype=torch.int32, device="cuda") for _ in range(64)]
    batch.select([0, 1])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    del noise


# ---- refusals of the bindings ---------------------------------------------------------------------------------------------------------
def test_refusals(ext):
    hidden, weight, _, _, targets, grad = case(4, 40, 64, torch.bfloat16, 0, 0)
    lse = torch.zeros(4, device="cuda")
    stored, scale, _ = quantized(torch.Generator(device="cuda").manual_seed(0), 40, 64, 8, 64)
    for args, what in (((hidden.cpu(), weight, targets, -100), "CUDA"), ((hidden.double(), weight, targets, -100), "hidden"),
                       ((hidden, weight.float(), targets, -100), "weight must be"), ((hidden, weight.t().contiguous().t(), targets, -100), "contiguous"),
                       ((hidden, weight.cpu(), targets, -100), "weight must be"), ((hidden, weight, targets.int(), -100), "int64"),
                       ((hidden, weight, targets[:3], -100), "int64"), ((hidden, weight, targets.cpu(), -100), "int64"),
                       ((hidden[0], weight, targets, -100), "rows"), ((hidden[:, :60], weight[:, :60].contiguous(), targets, -100), "multiple of 8"),
                       ((hidden, weight, targets, -100, None, 4), "out_group"), ((hidden, stored[:, :, :32].contiguous(), targets, -100, scale), "")):
        with pytest.raises(RuntimeError, match=what or None):
            ext.vocab_loss(*args)
    for args, what in (((hidden, weight, targets, lse[:3], grad, -100), "lse"), ((hidden, weight, targets, lse, grad.double(), -100), "grad"),
                       ((hidden, stored, targets, lse, grad, -100, scale, 0, True), "no gradient")):
        with pytest.raises(RuntimeError, match=what or None):
            ext.vocab_loss_grad(*args)
    g = torch.zeros(3, 40, dtype=torch.bfloat16, device="cuda")
    for args, what in (((g.cpu(), stored, scale), "CUDA"), ((g[:, :32], stored, scale), "grad must be"), ((g, stored, scale.double()), ""),
                       ((g, stored, scale, 0, 72), "keep_per_group"), ((g, stored, scale, 0, 12), "keep_per_group"), ((g, stored.cpu(), scale), "")):
        with pytest.raises(RuntimeError, match=what or None):
            ext.wq_linear_grad(*args)
    c = make([4], [0], 1, 8, 64, 72, torch.bfloat16)
    low = torch.zeros(4, 8, device="cuda")
    for change, what in ((dict(x=c["x"].cpu()), ""), (dict(base=c["base"].float()), ""), (dict(lora_a=c["lora_a"].float()), "dtype"),
                         (dict(lora_a=c["lora_a"][:, :4].contiguous()), "lora_a"), (dict(lora_b=c["lora_b"].transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
                         (dict(scaling=c["scaling"].double()), "scaling"), (dict(adapter=c["adapter"].long()), "adapter"),
                         (dict(query_start=c["query_start"][:1]), "query_start"), (dict(query_start=None), "one row"),
                         (dict(x=c["x"][:3]), ""), (dict(x=c["x"][:, :56]), "")):
        with pytest.raises(RuntimeError, match=what or None):
            call(ext, c | change)
        if "base" not in change:
            with pytest.raises(RuntimeError, match=what or None):
                call_grad(ext, c | change, low)
    for more, what in ((dict(out=torch.empty(4, 64, dtype=torch.bfloat16, device="cuda")), "out must be"), (dict(low=low.half()), "low must be"),
                       (dict(out=c["x"].new_zeros(8, 72)[::2]), "out must be")):
        with pytest.raises(RuntimeError, match=what or None):
            call(ext, c, **more)
    both = torch.zeros(8 * 72, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="share memory"):
        call(ext, dict(c, base=both[:288].view(4, 72)), out=both[72:360].view(4, 72))
    with pytest.raises(RuntimeError, match="x_scale"):
        call_grad(ext, c, low, x=c["x"].to(torch.int8), x_scale=torch.ones(4, 1, device="cuda"))
    with pytest.raises(RuntimeError, match="grad_base"):
        call_grad(ext, c, low, grad_base=c["grad_base"][:2])
    with pytest.raises(RuntimeError, match="at most 1024"):
        many = make([4], [0], 1025, 8, 8, 8, torch.bfloat16)
        call_grad(ext, many, low)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second device")
def test_on_the_tensors_device(ext):
    c = [t if t is None else t.to("cuda:1") for t in case(20, 300, 128, torch.bfloat16, 0, 0)]
    here = loss_and_gradients(ext, [t if t is None else t.to("cuda:0") for t in c])
    there = loss_and_gradients(ext, c)
    assert all(t.device.index == 1 for t in there) and same([t.cpu() for t in there], [t.cpu() for t in here])
