"""The entry points of learning (vocabulary loss, gradient of a quantized Linear, adapters) refuse what their kernels do not take, before
any device is asked for."""

import pytest

F32, F16, BF16 = 0, 1, 2
DTYPE = [(dict(dtype=3), "dtype code 3"), (dict(dtype=-1), "dtype code -1")]
GIB = 1 << 30


@pytest.fixture(scope="module")
def lib():
    from llmquant.hip.build import CAPI_PATH, build_extension, load_capi

    if not CAPI_PATH.exists():
        build_extension()
    return load_capi()


def text(lib):
    return lib.llmq_last_error().decode()


LOSS = dict(rows=4, vocab=1000, hidden=256, stride=256, group=128, out_group=0, format=8, dtype=BF16, workspace=16, bytes=0)


def loss(lib, **change):
    a = LOSS | change
    p = a.get("pointer", 16)
    return lib.llmq_vocab_loss(a.get("hidden_at", p), a["stride"], p, a.get("scale", p), p, -100, p, p, a["workspace"], a["bytes"], a["rows"],
                               a["vocab"], a["hidden"], a["group"], a["out_group"], a["format"], a["dtype"], None)


def loss_grad(lib, **change):
    a = LOSS | change
    p = a.get("pointer", 16)
    return lib.llmq_vocab_loss_grad(a.get("hidden_at", p), a["stride"], p, a.get("scale", p), p, -100, p, p, p, a.get("grad_weight"),
                                    a["workspace"], a["bytes"], a["rows"], a["vocab"], a["hidden"], a["group"], a["out_group"],
                                    a["format"], a["dtype"], None)


LOSSES = DTYPE + [
    (dict(rows=-1), "bad dimension"), (dict(vocab=-1), "bad dimension"), (dict(hidden=0), "bad dimension"), (dict(format=16), "weight format 16"),
    (dict(format=-8), "weight format -8"), (dict(hidden=260, group=130), "multiple of 8"), (dict(hidden=65544, group=8, stride=65544), "at most 65536"),
    (dict(group=0), "group_size"), (dict(group=12), "group_size"), (dict(group=96), "group_size"), (dict(group=-128), "group_size"),
    (dict(out_group=-1), "out_group"), (dict(stride=248), "row stride"), (dict(stride=260), "row stride"), (dict(rows=(1 << 20) + 1), "at most 2^20"),
    (dict(vocab=(1 << 24) + 1), "at most 2^20"), (dict(vocab=0), "no tokens"), (dict(pointer=None), "null tensor pointer"),
    (dict(scale=None), "null tensor pointer"), (dict(hidden_at=24), "16-byte aligned"), (dict(workspace=None), "workspace"),
    (dict(workspace=24, bytes=GIB), "workspace"), (dict(bytes=64), "workspace")]


@pytest.mark.parametrize("change,what", LOSSES)
@pytest.mark.parametrize("entry", [loss, loss_grad])
def test_the_loss_refuses(lib, entry, change, what):
    assert entry(lib, **change) == 1 and what in text(lib)


def test_codes_do_not_learn(lib):
    assert loss_grad(lib, grad_weight=16) == 1 and "no gradient" in text(lib)
    assert loss_grad(lib, grad_weight=24, format=0, scale=None) == 1 and "16-byte aligned" in text(lib)


def test_the_loss_of_nothing(lib):
    assert loss(lib, rows=0) == 0 and loss_grad(lib, rows=0) == 0 and loss_grad(lib, rows=0, vocab=0, format=0, grad_weight=16) == 0
    for rows, vocab, hidden in ((0, 8, 8), (-1, 8, 8), (8, 0, 8), (8, 8, 0)):
        assert lib.llmq_vocab_loss_workspace_bytes(rows, vocab, hidden, 0, 0, BF16) == 0
        assert lib.llmq_vocab_loss_grad_workspace_bytes(rows, vocab, hidden, 0, 0, BF16, 1) == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,hidden,group,format", [
    (1, 1, 8, 0, 0), (16, 128256, 2048, 0, 0), (64, 1 << 24, 65536, 0, 0), (65, 50257, 768, 128, 8), (1 << 20, 128256, 8192, 128, 4),
    (1 << 20, 1 << 24, 65536, 0, 0), (64, 1 << 20, 4096, 128, 4)])
def test_workspaces_of_the_loss_are_within_reason(lib, rows, vocab, hidden, group, format, dtype):
    """Never the logits: the statistics of 256 (few rows: 64) of them, a piece of the vocabulary, and what the rows themselves take."""
    planes = 3 if dtype == F32 else 1
    row = 2 * planes * (hidden + 64)
    forward = lib.llmq_vocab_loss_workspace_bytes(rows, vocab, hidden, group, format, dtype)
    assert 0 < forward <= (rows + 256) * (row + 8 * (vocab // 64 + 2)) + 256 * row + GIB
    for learned in (0, 1):
        need = lib.llmq_vocab_loss_grad_workspace_bytes(rows, vocab, hidden, group, format, dtype, learned)
        most = (rows + 256) * (row + 4 * 64 * hidden + 64) + 256 * (row + 2 * planes * (rows + 256)) + GIB
        assert 0 < need <= most


GRAD = dict(rows=4, N=512, stride=512, G=4, gs=128, keep=128, out_group=0, format=8, dtype=BF16, workspace=16, bytes=0)


def linear(lib, **change):
    a = GRAD | change
    p = a.get("pointer", 16)
    return lib.llmq_wq_linear_grad(a.get("grad", p), a["stride"], p, p, p, a["workspace"], a["bytes"], a["rows"], a["N"], a["G"], a["gs"], a["keep"],
                                   a["out_group"], a["format"], a["dtype"], None)


@pytest.mark.parametrize("change,what", DTYPE + [
    (dict(rows=-1), "negative"), (dict(N=-8), "negative"), (dict(G=-1), "negative"), (dict(format=0), "weight format 0"), (dict(gs=0), "group_size"),
    (dict(gs=12), "group_size"), (dict(keep=0), "keep_per_group"), (dict(keep=136), "keep_per_group"), (dict(keep=12), "keep_per_group"),
    (dict(out_group=-1), "out_group"), (dict(N=516, stride=520), "rows must be a multiple of 8"), (dict(N=0), "no rows"), (dict(rows=(1 << 20) + 1), "at most 2^20"),
    (dict(stride=504), "row stride"), (dict(stride=516), "row stride"), (dict(stride=1 << 25), "row stride"), (dict(pointer=None), "null tensor pointer"),
    (dict(grad=24), "16-byte aligned"), (dict(workspace=None), "workspace"), (dict(workspace=8, bytes=GIB), "workspace"), (dict(bytes=1000), "workspace")])
def test_the_gradient_of_a_linear_refuses(lib, change, what):
    assert linear(lib, **change) == 1 and what in text(lib)


def test_the_gradient_of_nothing(lib):
    assert linear(lib, rows=0) == 0 and linear(lib, G=0) == 0
    assert lib.llmq_wq_linear_grad_workspace_bytes(0, 512, 4, 128, 8, BF16) == 0


LORA = dict(rows=6, sequences=3, start=16, inp=256, out=512, x_stride=256, base_stride=512, rank=16, slots=2, dtype=BF16, workspace=16, bytes=0)


def lora(lib, **change):
    a = LORA | change
    p = a.get("pointer", 16)
    return lib.llmq_lora_add(a.get("x", p), a["x_stride"], p, a["base_stride"], a.get("bank", p), p, p, p, a["start"], a.get("to", 32),
                             a.get("low"), a["workspace"], a["bytes"], a["rows"], a["sequences"], a["inp"], a["out"], a["rank"], a["slots"],
                             a["dtype"], None)


def lora_grad(lib, **change):
    a = LORA | change
    p = a.get("pointer", 16)
    return lib.llmq_lora_grad(p, a["base_stride"], a.get("x", p), a["x_stride"], a.get("scale"), p, a.get("bank", p), p, p, p, a["start"],
                              a.get("grad_base"), a.get("grad_base_stride", 256), a.get("to", 32), p, p, a["workspace"], a["bytes"], a["rows"],
                              a["sequences"], a["inp"], a["out"], a["rank"], a["slots"], a["dtype"], None)


ADAPTERS = DTYPE + [
    (dict(rows=-1), "bad dimension"), (dict(sequences=-1), "bad dimension"), (dict(slots=-1), "bad dimension"), (dict(rank=0), "rank must be"),
    (dict(rank=12), "rank must be"), (dict(rank=136), "rank must be"), (dict(inp=252, x_stride=256), "multiples of 8"), (dict(out=0), "multiples of 8"),
    (dict(out=(1 << 20) + 8, base_stride=(1 << 20) + 8), "multiples of 8"), (dict(rows=(1 << 20) + 1), "at most 2^20"),
    (dict(sequences=(1 << 20) + 1), "at most 2^20"), (dict(start=None), "one row"),
    (dict(sequences=1 << 20, inp=1 << 20, out=1 << 20, x_stride=1 << 20, base_stride=1 << 20), "too many pieces"), (dict(pointer=None), "null tensor pointer"),
    (dict(x_stride=248), "row stride"), (dict(x_stride=260), "row stride"), (dict(base_stride=504), "row stride"), (dict(x=24), "16-byte aligned"),
    (dict(to=40), "16-byte aligned"), (dict(bank=20), "16-byte aligned"), (dict(workspace=None), "workspace"), (dict(workspace=24, bytes=GIB), "workspace"),
    (dict(bytes=16), "workspace")]


@pytest.mark.parametrize("change,what", ADAPTERS)
@pytest.mark.parametrize("entry", [lora, lora_grad])
def test_adapters_refuse(lib, entry, change, what):
    assert entry(lib, **change) == 1 and what in text(lib)


@pytest.mark.parametrize("entry,change,what", [
    (lora, dict(to=16, base_stride=520), "contiguous rows"), (lora, dict(low=24), "16-byte aligned"), (lora_grad, dict(slots=1025), "at most 1024 slots"),
    (lora_grad, dict(scale=16, inp=264, x_stride=272), "groups of 128"), (lora_grad, dict(scale=16, x_stride=264), "row stride"),
    (lora_grad, dict(grad_base=16, grad_base_stride=248), "row stride"), (lora_grad, dict(grad_base=24), "16-byte aligned")])
def test_adapters_refuse_one_way(lib, entry, change, what):
    assert entry(lib, **change) == 1 and what in text(lib)


def test_adapters_of_nothing(lib):
    for entry in (lora, lora_grad):
        assert entry(lib, rows=0) == 0 and entry(lib, sequences=0) == 0 and entry(lib, rows=0, sequences=0, start=None) == 0
    assert lora_grad(lib, slots=0) == 0
    assert lib.llmq_lora_add_workspace_bytes(0, 3, 1, 256, 16, BF16) == 0 and lib.llmq_lora_grad_workspace_bytes(6, 3, 1, 256, 512, 16, 0, BF16) == 0
