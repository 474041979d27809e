"""Low-rank adapters of many requests (lora_add) and their gradients (lora_grad) against the formulas in 64 bits.

Tolerances are bounds, element by element. u: half a step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24). A sum of K products in fp32, in any
order, is off by at most (K + 24) 2^-24 times the sum of their magnitudes. What lies between the two factors (low, du) enters the second product of 16-bit
types as two bfloat16: off by 2^-16, and the products of the two small parts that are left out for fp16 are 2^-16 more. The results are rounded once."""

import ctypes

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


def middle(dtype):
    return 2.0 ** -15 if dtype != torch.float32 else F32


def smallest(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def make(lengths, adapters, slots, rank, inp, out, dtype, seed=0, step=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    rows = sum(lengths)
    starts = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    return dict(x=normal(rows, inp).to(dtype), base=normal(rows, out).to(dtype), grad=normal(rows, out).to(dtype),
                grad_base=normal(rows, inp).to(dtype), lora_a=(normal(slots, rank, inp) * inp ** -0.5).to(dtype),
                lora_b=(0.3 * normal(slots, out, rank)).to(dtype), scaling=0.5 + torch.rand(slots, generator=gen, device="cuda"),
                adapter=torch.tensor(adapters, dtype=torch.int32, device="cuda"), query_start=None if step else starts)


def spans(c):
    adapters = c["adapter"].tolist()
    starts = range(len(adapters) + 1) if c["query_start"] is None else c["query_start"].tolist()
    return [(slice(starts[b], starts[b + 1]), a) for b, a in enumerate(adapters) if 0 <= a < c["lora_a"].shape[0]]


def forward(c, dtype):
    """(out, bound), (low, bound) in 64 bits."""
    x, out = c["x"].double(), c["base"].double()
    rank = c["lora_a"].shape[1]
    low = torch.zeros(x.shape[0], rank, dtype=torch.float64, device="cuda")
    low_tol, out_tol = torch.zeros_like(low), torch.zeros_like(out)
    for rows, a in spans(c):
        la, lb, s = c["lora_a"][a].double(), c["lora_b"][a].double(), c["scaling"][a].double()
        low[rows] = x[rows] @ la.T
        low_tol[rows] = (x.shape[1] + 24) * F32 * (x[rows].abs() @ la.abs().T)
        out[rows] += s * (low[rows] @ lb.T)
        size = s * (low[rows].abs() @ lb.abs().T)
        out_tol[rows] = s * (low_tol[rows] @ lb.abs().T) + (middle(dtype) + (3 * rank + 24) * F32) * size + F32 * (size + out[rows].abs())
    touched = torch.zeros(x.shape[0], 1, device="cuda", dtype=torch.bool)
    for rows, _ in spans(c):
        touched[rows] = True
    out_tol = out_tol + torch.where(touched, U[dtype] * (out.abs() + out_tol) + smallest(dtype), 0.0)
    return (out, out_tol), (low, low_tol)


def backward(c, x, low, dtype, with_base=True):
    """Gradients of x, lora_a, lora_b with their bounds; x: the values in 64 bits."""
    grad, low = c["grad"].double(), low.double()
    gx = c["grad_base"].double() if with_base else torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    gx_tol = torch.zeros_like(gx)
    ga, gb = (torch.zeros(c[k].shape, dtype=torch.float64, device="cuda") for k in ("lora_a", "lora_b"))
    ga_tol, gb_tol = torch.zeros_like(ga), torch.zeros_like(gb)
    rank, total = ga.shape[1], grad.shape[0]
    for rows, a in spans(c):
        la, lb, s = c["lora_a"][a].double(), c["lora_b"][a].double(), c["scaling"][a].double()
        g, v = grad[rows], x[rows]
        du = s * (g @ lb)
        du_tol = s * (grad.shape[1] + 24) * F32 * (g.abs() @ lb.abs()) + 2 * F32 * du.abs()
        size = du.abs() @ la.abs()
        gx[rows] += du @ la
        gx_tol[rows] = du_tol @ la.abs() + (middle(dtype) + (3 * rank + 24) * F32) * size + F32 * (size + gx[rows].abs())
        ga[a] += du.T @ v
        ga_tol[a] += du_tol.T @ v.abs() + (middle(dtype) + (3 * total + 24) * F32) * (du.abs().T @ v.abs())
        gb[a] += s * (g.T @ low[rows])
        gb_tol[a] += (middle(dtype) + (3 * total + 24) * F32) * s * (g.abs().T @ low[rows].abs())
    pairs = []
    for value, tol in ((gx, gx_tol), (ga, ga_tol), (gb, gb_tol)):
        pairs.append((value, tol + torch.where(tol > 0, U[dtype] * (value.abs() + tol) + smallest(dtype), 0.0)))
    return pairs


def close(got, want, what=""):
    value, tol = want
    off = (got.double() - value).abs()
    assert (off <= tol).all(), f"{what}: {(off - tol).max().item()} beyond, off by {off.max().item()}, {(off > tol).sum().item()} of {off.numel()}"


def call(ext, c, **more):
    return ext.lora_add(c["x"], c["base"], c["lora_a"], c["lora_b"], c["scaling"], c["adapter"], c["query_start"], **more)


def call_grad(ext, c, low, **more):
    return ext.lora_grad(c["grad"], more.pop("x", c["x"]), low, c["lora_a"], c["lora_b"], c["scaling"], c["adapter"], c["query_start"], **more)


# (lengths of the requests, their adapters, slots, rank, in, out)
CASES = {
    "one row": ([1], [0], 1, 8, 8, 8),
    "ranks that are no whole tile": ([3, 17, 1], [1, 0, 1], 2, 24, 200, 72),
    "without, outside, empty": ([5, 0, 40, 7, 33, 0], [-1, 0, 2, 3, 1, 1], 3, 16, 264, 136),
    "same adapter again and again": ([9, 70, 9, 65, 30], [1, 1, 0, 1, 1], 2, 32, 128, 256),
    "long requests": ([300, 129, 1, 150], [0, 2, 1, 2], 4, 64, 520, 392),
    "wide rank": ([33, 100], [1, 0], 2, 128, 384, 640),
    "rank of 40 over long rows": ([200, 31], [0, 1], 2, 40, 1032, 128),
    "nobody has one": ([4, 4], [-1, 9], 2, 16, 64, 64),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", CASES)
def test_requests(ext, name, dtype):
    c = make(*CASES[name], dtype)
    low = torch.full((c["x"].shape[0], c["lora_a"].shape[1]), float("nan"), device="cuda")
    out = call(ext, c, low=low)
    want, want_low = forward(c, dtype)
    close(low, want_low, "low")
    close(out, want, "out")
    assert torch.equal(out, call(ext, c))
    in_place = c["base"].clone()
    assert ext.lora_add(c["x"], in_place, c["lora_a"], c["lora_b"], c["scaling"], c["adapter"], c["query_start"], out=in_place) is not None
    assert torch.equal(out, in_place)
    grads = call_grad(ext, c, low, grad_base=c["grad_base"])
    for got, pair, what in zip(grads, backward(c, c["x"].double(), low, dtype), ("gx", "gA", "gB")):
        close(got, pair, what)
    bare = call_grad(ext, c, low)
    close(bare[0], backward(c, c["x"].double(), low, dtype, False)[0], "gx alone")
    assert torch.equal(bare[1], grads[1]) and torch.equal(bare[2], grads[2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, slots, rank, inp, out", [(1, 3, 16, 2048, 512), (7, 4, 8, 136, 2048), (70, 9, 64, 1024, 1000), (300, 2, 128, 256, 328)])
def test_a_row_each(ext, rows, slots, rank, inp, out, dtype):
    adapters = [(7 * b) % (slots + 1) - 1 for b in range(rows)]
    c = make([1] * rows, adapters, slots, rank, inp, out, dtype, seed=rows, step=True)
    low = torch.empty(rows, rank, device="cuda")
    got = call(ext, c, low=low)
    want, want_low = forward(c, dtype)
    close(low, want_low, "low")
    close(got, want, "out")
    for grad, pair, what in zip(call_grad(ext, c, low, grad_base=c["grad_base"]), backward(c, c["x"].double(), low, dtype), ("gx", "gA", "gB")):
        close(grad, pair, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths, adapters, slots, rank, inp, out", [
    ([1], [0], 1, 8, 128, 8), ([40, 3, 90], [1, -1, 0], 2, 16, 384, 264), ([500, 20], [0, 1], 2, 64, 256, 128), ([65, 66], [0, 0], 1, 128, 640, 72)])
def test_gradients_from_codes(ext, lengths, adapters, slots, rank, inp, out, dtype):
    """x kept as the framework's own 8-bit codes: the gradients are those of the values that the codes stand for."""
    c = make(lengths, adapters, slots, rank, inp, out, dtype, seed=inp)
    codes, scale = ext.quant_group_codes(c["x"], 8, 128)
    low = torch.empty(c["x"].shape[0], rank, device="cuda")
    call(ext, c, low=low)
    values = (codes.double().unflatten(1, (-1, 128)) * scale.double()[..., None]).flatten(1)
    grads = call_grad(ext, c, low, x=codes, x_scale=scale, grad_base=c["grad_base"])
    for got, pair, what in zip(grads, backward(c, values, low, dtype), ("gx", "gA", "gB")):
        close(got, pair, what)
    plain = call_grad(ext, c, low, grad_base=c["grad_base"])
    assert torch.equal(plain[0], grads[0]) and torch.equal(plain[2], grads[2])
