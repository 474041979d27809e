"""Who has which adapter, as captured steps, several streams and calls of unlike sizes read it."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def batch_and_bank(slots=3):
    from llmquant.quantizers.adapters import AdapterBatch, LoraAdapters

    batch = AdapterBatch("cuda")
    bank = LoraAdapters(64, 64, 8, slots, 16.0, torch.bfloat16, "cuda", batch).requires_grad_(False)
    gen = torch.Generator(device="cuda").manual_seed(0)
    bank.lora_b.copy_(torch.randn(bank.lora_b.shape, generator=gen, device="cuda"))
    x, base = (torch.randn(12, 64, generator=gen, device="cuda").bfloat16() for _ in range(2))
    return batch, bank, x, base


def alone(bank, x, base, adapter, start=None):
    """The rows with their adapters, by the operator itself (in the form that the batch takes, so that the bits agree: a row each, or starts)."""
    from llmquant.hip import load_extension

    start = None if start is None else torch.tensor(start, dtype=torch.int32, device="cuda")
    return load_extension().lora_add(x, base, bank.lora_a, bank.lora_b, bank.scaling, torch.tensor(adapter, dtype=torch.int32, device="cuda"), start)


@pytest.mark.parametrize("rows", [1, 12])
def test_a_step_captured_before_anything_was_selected(rows):
    """It reads what is selected later; a fill recorded with it would take that back at every replay."""
    batch, bank, x, base = batch_and_bank()
    x, base = x[:rows], base[:rows]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = bank(x, base.clone())
    for adapter in (1, -1, 2, 0):
        batch.select([adapter])
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, bank(x, base.clone())) and torch.equal(got, alone(bank, x, base, [adapter], None if rows == 1 else [0, rows])), adapter
    batch.clear()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, base)


def test_requests_are_not_selected_for_the_first_time_in_a_capture():
    batch, bank, x, base = batch_and_bank()
    chosen = torch.tensor([2, -1, 0], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="for the first time"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            batch.select(chosen)
    torch.cuda.synchronize()
    batch.select([0, 0, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):   # (known: from now on a replay selects them)
        batch.select(chosen)
    for _ in range(3):
        batch.select([1, 1, 1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bank(x[:3], base[:3].clone()), alone(bank, x[:3], base[:3], [2, -1, 0]))


def test_starts_made_on_one_stream_are_read_on_another():
    """The next call with as many rows, on a stream that does not wait for the first one's."""
    batch, bank, x, base = batch_and_bank()
    batch.select([2, 0])
    want = alone(bank, x, base, [2, 0], [0, 6, 12])
    torch.cuda.synchronize()
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(20_000_000)
        first = bank(x, base.clone())
    with torch.cuda.stream(other):
        second = bank(x, base.clone())
    other.synchronize()
    assert torch.equal(second, want)
    torch.cuda.synchronize()
    assert torch.equal(first, want)


def test_many_prompt_lengths_beside_a_captured_step():
    from llmquant.quantizers import AdapterBatch

    batch, bank, x, base = batch_and_bank()
    batch.select([2, 0])
    want = bank(x, base.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = bank(x, base.clone())
    longer = torch.empty(2 * AdapterBatch.STARTS + 20, 64, dtype=torch.bfloat16, device="cuda")
    for n in range(2, longer.shape[0], 2):
        assert batch.rows(longer[:n])[1].tolist() == [0, n // 2, n] if n != 2 else batch.rows(longer[:n])[1] is None
    noise = [torch.full((3,), 7, dtype=torch.int32, device="cuda") for _ in range(64)]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(bank(x, base.clone()), want)
    del noise


def test_a_step_behind_a_prompt():
    """One row of each of two requests while a prompt's starts are selected: refused; with adapters that lie on the device nothing is asked of it."""
    batch, bank, x, base = batch_and_bank()
    start = torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda")
    batch.select([2, 0], start)
    assert torch.equal(bank(x, base.clone()), alone(bank, x, base, [2, 0], [0, 5, 12]))
    with pytest.raises(ValueError, match="fewer than the 12"):
        bank(x[:2], base[:2].clone())
    batch.select([2, 0])
    assert torch.equal(bank(x[:2], base[:2].clone()), alone(bank, x[:2], base[:2], [2, 0]))
    batch.select(torch.tensor([2, 0], dtype=torch.int32, device="cuda"), start)
    assert torch.equal(bank(x, base.clone()), alone(bank, x, base, [2, 0], [0, 5, 12]))
    assert torch.equal(bank(x[:2], base[:2].clone()), alone(bank, x[:2], base[:2], [2, 0], [0, 5, 12]))


def test_runtimes_from_before_the_adapters():
    """What is kept on the whole model gives way to adapters that are added through a part of it; a fused runtime in a program's hands refuses."""
    from llmquant.quantizers import add_adapters, remove_adapters, use_adapters
    from llmquant.runtime import graphed_generate, kernel_runtime
    from test_gpu_adapters import build, stir

    _, kernel = build(torch.float32, hidden=512, inter=1024, heads=8, vocab=512)
    ids = torch.randint(0, 512, (1, 12), generator=torch.Generator().manual_seed(4)).cuda()
    held = kernel_runtime(kernel, 32)
    plain = graphed_generate(kernel, ids, 12, kv_bits=8)
    assert torch.equal(held.generate(ids, 12), plain)
    add_adapters(kernel.model, rank=8, slots=2)
    stir(kernel)
    use_adapters(kernel, [1])
    want = kernel_runtime(kernel, 32).generate(ids, 12, use_graph=False)
    assert not torch.equal(want, plain)
    assert torch.equal(graphed_generate(kernel, ids, 12, kv_bits=8), want)
    with pytest.raises(RuntimeError, match="build another"):
        held.generate(ids, 12)
    remove_adapters(kernel.model)
    assert torch.equal(graphed_generate(kernel, ids, 12, kv_bits=8), plain) and torch.equal(held.generate(ids, 12), plain)


def test_a_training_step_behind_an_evaluation():
    """In inference mode with as many rows before: what was kept from it is read by autograd."""
    batch, bank, x, base = batch_and_bank()
    bank.requires_grad_(True)
    with torch.inference_mode():
        batch.select([2, 0])
        want = bank(x, base.clone())
    out = bank(x, base)
    assert torch.equal(out, want)
    out.float().square().sum().backward()
    assert bank.lora_a.grad[2].any() and bank.lora_b.grad[0].any() and not bank.lora_b.grad[1].any()
    batch.select([1, 1])
    assert not torch.equal(bank(x, base), want)


def test_a_model_of_inference_mode_learns():
    """Codes, scales, targets and starts that were made there have no gradient and are read by one."""
    from llmquant.hip import vocab_cross_entropy
    from llmquant.quantizers import KernelQuantLinear, add_adapters, use_adapters
    from test_kernel_linear_derivatives import linear

    torch.manual_seed(0)
    plain = torch.nn.Sequential(linear(128, 256, 128, 8, bias=False, device="cuda"), linear(256, 512, 128, 4, bias=False, device="cuda"))
    with torch.inference_mode():
        parts = [linear(128, 256, 128, 8, bias=False, device="cuda"), linear(256, 512, 128, 4, bias=False, device="cuda")]
        start, targets = torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda"), torch.randint(0, 512, (12,), device="cuda")
    model = torch.nn.Sequential(*parts)
    assert isinstance(model[0], KernelQuantLinear) and model[0].qdata.is_inference() and targets.is_inference()
    x = torch.randn(12, 128, device="cuda")
    grads = []
    for m, t, s in ((model, targets, start), (plain, targets.clone(), start.clone())):
        torch.manual_seed(1)
        add_adapters(m, rank=8, slots=2, targets="0", dtype=torch.float32)
        torch.nn.init.normal_(m[0].adapters.lora_b)
        use_adapters(m, [1, 0], s)
        leaf = x.clone().requires_grad_()
        vocab_cross_entropy(m[0](leaf), m[1], t).backward()
        grads.append((leaf.grad, m[0].adapters.lora_a.grad, m[0].adapters.lora_b.grad))
    assert all(torch.equal(a, b) and a.any() for a, b in zip(*grads))
