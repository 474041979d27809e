"""Bounds of the learning entry points that a call cannot be seen to break by its result's shape: how far rows may lie apart, what a workspace
takes. Before any device is asked for."""

import pytest
from test_learning_host import BF16, F16, F32, lib, linear, lora, lora_grad, loss, loss_grad, text  # noqa: F401 (lib: a fixture)

WIDE = "within 4 GiB"


# A lane's offset into a tile of rows has 32 bits: (rows of the tile - 1) strides and a step of 128 bytes lie below 2^32. 255 x 2 x 8421504 + 128 does.
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows, stride, fits", [(256, 8421504, True), (256, 8421512, False), (1000, 8421504, True), (1000, 8421512, False), (128, 1 << 24, True),
                                                (129, 1 << 24, False), (66, 1 << 25, False), (64, 1 << 30, True), (256, 1 << 40, False)])
def test_rows_of_the_loss_lie_within_its_tiles_reach(lib, rows, stride, fits, dtype):  # noqa: F811
    assert loss(lib, rows=rows, stride=stride, format=0, scale=None, dtype=dtype) == 1
    assert (WIDE in text(lib)) != fits and ("workspace" in text(lib)) == fits
    assert loss_grad(lib, rows=rows, stride=stride, format=0, scale=None, dtype=dtype) == 1 and "workspace" in text(lib)   # (gathers its rows)


def test_rows_that_are_staged_lie_anywhere(lib):  # noqa: F811
    for change in (dict(dtype=F32, format=0, scale=None, rows=600), dict(rows=1000, hidden=256 + 8, group=8), dict(rows=128)):
        assert loss(lib, **(dict(stride=1 << 30) | change)) == 1 and "workspace" in text(lib)


@pytest.mark.parametrize("change, fits", [
    (dict(rows=321, stride=8421504), True), (dict(rows=321, stride=8421512), False), (dict(rows=321, stride=1 << 24), False), (dict(rows=320, stride=1 << 24), True),
    (dict(rows=321, stride=1 << 24, dtype=F32), True), (dict(rows=321, stride=1 << 24, N=520), True), (dict(rows=321, stride=1 << 24, N=1 << 24), False),
    (dict(rows=321, stride=1 << 24, N=(1 << 24) - 8), False), (dict(rows=321, stride=1 << 24, N=1 << 24, dtype=F32), False)])
def test_rows_of_a_linears_gradient_lie_within_its_tiles_reach(lib, change, fits):  # noqa: F811
    assert linear(lib, **change) == 1
    assert (WIDE in text(lib)) != fits and ("workspace" in text(lib)) == fits


@pytest.mark.parametrize("change, fits", [
    (dict(stride=429496672), True), (dict(stride=429496680), False),                                # 5 x 2 x it + 512 bytes of a row
    (dict(rows=1000, stride=143165552), True), (dict(rows=1000, stride=143165560), False),          # 15 rows
    (dict(rows=1000, rank=64, stride=69273656), True), (dict(rows=1000, rank=64, stride=69273664), False),   # 31
    (dict(rows=1000, sequences=1000, rank=64, stride=143165552), True), (dict(rows=1000, rank=64, stride=34636820, dtype=F32), True),
    (dict(rows=1000, rank=64, stride=34636832, dtype=F32), False), (dict(rows=3, start=None, stride=1 << 40), True)])
def test_rows_of_a_request_lie_within_reach(lib, change, fits):  # noqa: F811
    change = dict(change)
    stride = change.pop("stride")
    for rows in (lora(lib, inp=256, x_stride=stride, **change), lora_grad(lib, out=256, base_stride=stride, **change)):
        assert rows == 1 and (WIDE in text(lib)) != fits and ("workspace" in text(lib)) == fits


@pytest.mark.parametrize("rows, sequences, inp, out, rank", [(2000, 1, 4096, 4096, 64), (4096, 2, 4096, 14336, 64), (4099, 3, 4096, 4096, 128), (20000, 5, 2048, 2048, 16)])
def test_slots_without_rows_take_their_turned_banks_alone(lib, rows, sequences, inp, out, rank):  # noqa: F811
    """A large bank of which few learn at a time: sums of pieces for the slots that can have rows, not for all."""
    few = lib.llmq_lora_grad_workspace_bytes(rows, sequences, 1, inp, out, rank, sequences, BF16)
    for slots in (8, 64, 1024):
        more = lib.llmq_lora_grad_workspace_bytes(rows, sequences, 1, inp, out, rank, slots, BF16)
        assert 0 <= more - few <= (slots - sequences) * (2 * rank * (inp + out) + 8) + 5 * 256
