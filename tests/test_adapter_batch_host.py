"""The bookkeeping of who has which adapter, on the CPU."""

import copy

import pytest
import torch

from llmquant.quantizers import AdapterBatch


def rows(batch, *lead):
    adapter, start = batch.rows(torch.empty(*lead, 8, device="meta"))
    return adapter.tolist(), None if start is None else start.tolist()


def test_requests_of_equal_length():
    batch = AdapterBatch("cpu")
    assert rows(batch, 1) == ([-1], None) and rows(batch, 5) == ([-1], [0, 5]) and rows(batch, 1, 7) == ([-1], [0, 7])
    batch.select([3, -1, 0])
    assert rows(batch, 3) == ([3, -1, 0], None) and rows(batch, 3, 4) == ([3, -1, 0], [0, 4, 8, 12]) and rows(batch, 6) == ([3, -1, 0], [0, 2, 4, 6])
    batch.clear()
    assert rows(batch, 12) == ([-1], [0, 12])
    batch.select(torch.tensor([1, 2, 2]))
    assert rows(batch, 3, 4) == ([1, 2, 2], [0, 4, 8, 12])


def test_what_is_kept_has_an_end(monkeypatch):
    """A serving program meets any number of prompt lengths; those that captured steps read stay."""
    batch = AdapterBatch("cpu")
    first = batch.rows(torch.empty(2, 8))[1]
    monkeypatch.setattr(batch, "_capturing", lambda: True)
    held = batch.rows(torch.empty(2, 8))[1]
    made = batch.rows(torch.empty(3, 8))[1]   # (the graph's own)
    monkeypatch.undo()
    assert held is first and made.tolist() == [0, 3]
    for n in range(2, 1500):
        assert batch.rows(torch.empty(n, 8))[1].tolist() == [0, n]
        assert len(batch._starts) <= AdapterBatch.STARTS
    assert batch.rows(torch.empty(2, 8))[1] is first and len(batch._captured) == 1


def test_starts_of_a_prompt_are_no_steps():
    """A call of fewer rows than the selected requests have would lie in the first ones' ranges."""
    batch = AdapterBatch("cpu")
    start = torch.tensor([0, 4, 4, 9], dtype=torch.int32)
    batch.select([0, 1, 2], start)
    assert rows(batch, 9) == ([0, 1, 2], [0, 4, 4, 9]) and rows(batch, 3, 4) == ([0, 1, 2], [0, 4, 4, 9])   # (rows behind the last request's: nobody's)
    for lead in ((3,), (1, 3), (8,), (1,)):
        with pytest.raises(ValueError, match="fewer than the 9"):
            rows(batch, *lead)
    twin = copy.deepcopy(batch)
    with pytest.raises(ValueError, match="fewer than the 9"):
        rows(twin, 3)
    start.copy_(torch.tensor([0, 1, 2, 3], dtype=torch.int32))   # (written since: whoever wrote knows what calls come)
    assert rows(batch, 3) == ([0, 1, 2], [0, 1, 2, 3])
    with pytest.raises(ValueError, match="fewer than the 9"):
        rows(twin, 3)
    batch.select([0, 1, 2])
    assert rows(batch, 3) == ([0, 1, 2], None)
    with torch.inference_mode():
        batch.select([5], torch.tensor([0, 6], dtype=torch.int32))
        with pytest.raises(ValueError, match="fewer than the 6"):
            rows(batch, 5)
        assert rows(batch, 6) == ([5], [0, 6])
    batch.clear()
    assert rows(batch, 2) == ([-1], [0, 2])


def test_a_packed_file_says_that_it_holds_no_adapters(monkeypatch, tmp_path, recwarn):
    """What was learned beside the codes does not go with them; it is in the state dict."""
    import llmquant.quantizers.kernel as kernel
    from llmquant.core.scheme import QuantizationArgs, QuantizationScheme
    from llmquant.packing import read_packed, save_packed_model
    from llmquant.quantizers import KernelQuantLinear, add_adapters, remove_adapters

    monkeypatch.setattr(kernel, "load_extension", lambda: type("None", (), {"wq_gemv": None})())
    model = torch.nn.Module()
    scheme = QuantizationScheme(weights=QuantizationArgs(num_bits=8, strategy="group", group_size=128), input_activations=None)
    model.up_proj = KernelQuantLinear.from_linear(torch.nn.Linear(128, 16, bias=False), scheme)
    save_packed_model(model, tmp_path / "bare", "test/model")
    assert not recwarn.list
    add_adapters(model, rank=8)
    with pytest.warns(UserWarning, match="no adapters.*up_proj"):
        save_packed_model(model, tmp_path / "adapted", "test/model")
    assert (tmp_path / "bare").read_bytes() == (tmp_path / "adapted").read_bytes()
    assert sum("adapters" in name for name in model.state_dict()) == 3
    remove_adapters(model)
    recwarn.clear()
    save_packed_model(model, tmp_path / "again", "test/model")
    assert not recwarn.list and not any("adapters" in name for name in read_packed(tmp_path / "again")[0])


def test_what_is_kept_from_inference_mode_serves_training():
    batch = AdapterBatch("cpu")
    with torch.inference_mode():
        batch.select([1, 0])
        kept = batch.rows(torch.empty(6, 8))
    assert not any(t.is_inference() for t in kept)
    batch.select([0, 1])
    assert rows(batch, 6) == ([0, 1], [0, 3, 6])
