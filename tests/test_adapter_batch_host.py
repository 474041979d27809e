"""The bookkeeping of who has which adapter, on the CPU."""

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
