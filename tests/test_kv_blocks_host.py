"""The entry points over a cache in blocks refuse what their kernels do not take, before any device is asked for."""

import pytest

F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    from llmquant.hip.build import CAPI_PATH, build_extension, load_capi

    if not CAPI_PATH.exists():
        build_extension()
    return load_capi()


def text(lib):
    return lib.llmq_last_error().decode()


def norm(lib, **change):
    a = dict(tokens=4, q_heads=8, kv_heads=2, dim=128, rotary=128, rows=64, q_stride=1280, k_stride=1280, eps=1e-6, dtype=BF16, table=BF16,
             position_bytes=4, positions=16) | change
    return lib.llmq_qk_norm_rope(*[a.get("pointer")] * 6, a["positions"], a["position_bytes"], *[a.get("pointer")] * 2, a["tokens"], a["q_heads"],
                                 a["kv_heads"], a["dim"], a["rotary"], a["rows"], a["q_stride"], a["k_stride"], a["eps"], a["dtype"],
                                 a["table"], None)


@pytest.mark.parametrize("change,what", [
    (dict(tokens=-1), "bad dimension"), (dict(dtype=7), "float32, float16 or bfloat16"), (dict(table=F16), "the tables hold"),
    (dict(dim=72), "head_dim must be a multiple of 16"), (dict(dim=512, rotary=64), "up to 256"), (dict(dim=0), "head_dim"),
    (dict(rotary=8), "rotated part"), (dict(rotary=256), "rotated part"), (dict(rotary=0), "rotated part"),
    (dict(q_stride=1281), "row strides"), (dict(k_stride=1284), "row strides"), (dict(position_bytes=2), "4 or 8 bytes"),
    (dict(positions=None, rows=3), "a row for each"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(), "null tensor pointer"), (dict(pointer=24), "16-byte aligned"),
    (dict(pointer=16, tokens=2 ** 31 - 1, rows=1), "too many heads")])
def test_norm_and_rotation_refuses(lib, change, what):
    assert norm(lib, **change) == 1 and what in text(lib)


def test_norm_and_rotation_of_nothing(lib):
    assert norm(lib, tokens=0) == 0 and norm(lib, q_heads=0, kv_heads=0) == 0
    assert norm(lib, dtype=F32, table=F32, dim=72, rotary=8) == 1 and "null tensor pointer" in text(lib)   # packets of four


SHAPE = dict(tokens=4, sequences=4, kv_heads=2, dim=64, block=64, blocks=8, width=3, stride=3, dtype=BF16)
SHAPES = [
    (dict(tokens=-1), "bad dimension"), (dict(sequences=-1), "bad dimension"), (dict(kv_heads=0), "bad dimension"),
    (dict(blocks=-1), "bad dimension"), (dict(width=-1), "bad dimension"), (dict(dim=96), "head_dim must be 64, 128 or 256"),
    (dict(block=48), "block must be"), (dict(block=8), "block must be"), (dict(block=256), "block must be"), (dict(dtype=3), "dtype code 3"),
    (dict(stride=-3), "negative stride"), (dict(tokens=2 ** 31 - 1, sequences=2 ** 31 - 1, kv_heads=64), "too many rows")]


def append(lib, **change):
    a = SHAPE | dict(key_stride=128, value_stride=128) | change
    p = a.get("pointer")
    return lib.llmq_kv_block_append(p, p, a["key_stride"], a["value_stride"], a.get("codes", p), p, p, p, p, a["stride"], p, a.get("start"),
                                    a["tokens"], a["sequences"], a["kv_heads"], a["dim"], a["block"], a["blocks"], a["width"], a["dtype"], None)


@pytest.mark.parametrize("change,what", SHAPES + [
    (dict(sequences=3), "one row"), (dict(key_stride=130), "row strides"), (dict(value_stride=130), "row strides"),
    (dict(dtype=F32, key_stride=130), "row strides"), (dict(), "null tensor pointer"), (dict(pointer=16, codes=None), "null tensor pointer"),
    (dict(pointer=16, codes=24), "codes must be 16-byte aligned"), (dict(pointer=8, codes=16), "16-byte aligned")])
def test_append_refuses(lib, change, what):
    assert append(lib, **change) == 1 and what in text(lib)


def test_append_of_nothing(lib):
    assert append(lib, tokens=0, sequences=0) == 0 and append(lib, blocks=0) == 0 and append(lib, width=0) == 0


def dequant(lib, **change):
    a = SHAPE | change
    p = a.get("pointer")
    return lib.llmq_kv_block_dequant(a.get("codes", p), p, p, p, p, a["stride"], p, None, p, p, a["tokens"], a["sequences"], a["kv_heads"],
                                     a["dim"], a["block"], a["blocks"], a["width"], a["dtype"], None)


@pytest.mark.parametrize("change,what", SHAPES + [
    (dict(), "null tensor pointer"), (dict(pointer=16, codes=24), "codes must be 16-byte aligned"), (dict(pointer=8, codes=16), "16-byte aligned")])
def test_dequant_refuses(lib, change, what):
    assert dequant(lib, **change) == 1 and what in text(lib)


def test_dequant_of_nothing(lib):
    assert dequant(lib, tokens=0) == 0 and dequant(lib, sequences=0) == 0


def attention(lib, **change):
    a = SHAPE | dict(q_stride=512, q_heads=8, scale=0.125, space=2 ** 40) | change
    p = a.get("pointer")
    return lib.llmq_kv_block_attention(p, a["q_stride"], a.get("codes", p), p, p, p, p, a["stride"], p, a.get("start"), p, a.get("workspace", p), a["space"],
                                       a["scale"], a["tokens"], a["sequences"], a["q_heads"], a["kv_heads"], a["dim"], a["block"], a["blocks"],
                                       a["width"], a["dtype"], None)


@pytest.mark.parametrize("change,what", SHAPES + [
    (dict(q_heads=7), "not a multiple"), (dict(q_heads=0), "not a multiple"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(sequences=3), "one row"), (dict(q_stride=513), "row strides"), (dict(), "null tensor pointer"),
    (dict(pointer=16, codes=24), "16-byte aligned"), (dict(pointer=8, codes=16), "16-byte aligned"),
    (dict(tokens=2 ** 27, sequences=2 ** 20, start=16, pointer=16, q_heads=64), "too many rows")])
def test_attention_refuses(lib, change, what):
    assert attention(lib, **change) == 1 and what in text(lib)


def test_attention_of_nothing(lib):
    assert attention(lib, tokens=0, sequences=0) == 0 and attention(lib, sequences=0, tokens=0, start=16) == 0


def test_attention_workspace(lib):
    """(tokens, sequences, q_heads, kv_heads, head_dim, block, table width)"""
    size = lib.llmq_kv_block_attention_workspace_bytes
    assert size(0, 0, 8, 2, 64, 64, 100) == 0 and size(1, 1, 8, 0, 64, 64, 100) == 0 and size(1, 1, 8, 2, 64, 64, 0) == 0
    need = size(1, 1, 32, 8, 128, 128, 1024)
    if need:   # a long sequence of few rows is split, and a workspace that is too small refused
        assert attention(lib, tokens=1, sequences=1, q_heads=32, kv_heads=8, dim=128, block=128, width=1024, q_stride=4096, pointer=16, space=need - 1) == 1
        assert "workspace" in text(lib)


# ---- the batch's bookkeeping ------------------------------------------------------------------------------------------
def make(**change):
    from llmquant.runtime import BlockQuantCache

    return BlockQuantCache(**(dict(num_layers=2, kv_heads=2, head_dim=64, num_blocks=10, max_sequences=3, max_len=100, block=16, device="cpu") | change))


def test_cache_shapes_and_refusals():
    cache = make(block=64, num_blocks=5)
    assert cache.k_codes.shape == (2, 5, 2, 64, 64) and cache.v_codes.shape == (2, 5, 2, 4, 64, 16) and cache.k_scale.shape == (2, 5, 2)
    assert cache.block_table.tolist() == [[-1, -1]] * 3 and cache.cached.tolist() == [-1] * 3
    assert cache.bytes_per_token() == 2 * 2 * 2 * (64 + 4 / 64)
    for bad in (dict(block=48), dict(head_dim=96), dict(num_blocks=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            make(**bad)


def test_sequences_come_grow_and_go():
    cache = make()
    a, b = cache.add(), cache.add()
    assert (a, b) == (0, 1) and cache.cached.tolist() == [0, 0, -1]
    cache.reserve([33, 16, 0])
    assert cache.free_blocks() == 6 and [(r >= 0).sum().item() for r in cache.block_table] == [3, 1, 0]
    cache.advance([33, 16, 0])
    assert cache.cached.tolist() == [33, 16, -1] and cache.get_seq_length(a) == 33
    cache.reserve(1)                      # a token each: only the full block's owner needs another
    assert cache.free_blocks() == 5 and (cache.block_table[1] >= 0).sum() == 2
    cache.advance(1)
    c = cache.add()
    assert c == 2 and cache.cached.tolist() == [34, 17, 0]
    with pytest.raises(RuntimeError, match="places"):
        cache.add()
    used = cache.block_table[cache.block_table >= 0].tolist()
    assert len(set(used)) == len(used) == 5
    cache.truncate(a, 20)
    assert cache.get_seq_length(a) == 20 and cache.cached.tolist() == [20, 17, 0] and cache.free_blocks() == 5
    cache.reserve([20, 0, 0])             # within what it still has
    assert cache.free_blocks() == 5
    cache.release(b)
    assert cache.cached.tolist() == [20, -1, 0] and cache.free_blocks() == 7 and cache.block_table[1].tolist() == [-1] * 7
    cache.advance_device(2)
    assert cache.cached.tolist() == [22, -1, 2]
    cache.advance(2, device=False)
    assert cache.get_seq_length(a) == 22 and cache.get_seq_length(c) == 2


def test_bookkeeping_refuses_and_changes_nothing():
    cache = make()
    a = cache.add()
    for call, error in ((lambda: cache.reserve([101, 0, 0]), ValueError), (lambda: cache.reserve([1, 1, 0]), ValueError),
                        (lambda: cache.reserve([-1, 0, 0]), ValueError), (lambda: cache.reserve([1, 0]), ValueError),
                        (lambda: cache.release(1), ValueError), (lambda: cache.release(3), ValueError), (lambda: cache.truncate(a, 1), ValueError),
                        (lambda: cache.get_seq_length(2), ValueError), (lambda: cache.advance([0, 0, 1]), ValueError)):
        with pytest.raises(error):
            call()
    b = cache.add()
    with pytest.raises(RuntimeError, match="11 more blocks are needed, 10 are free"):
        cache.reserve([100, 50, 0])
    assert cache.free_blocks() == 10 and cache.block_table.eq(-1).all() and cache.get_seq_length(b) == 0


def test_advance_refuses_tokens_without_blocks():
    cache = make()
    a = cache.add()
    cache.reserve([17, 0, 0])             # two blocks
    with pytest.raises(ValueError, match="would hold 33 tokens, blocks for 32 are reserved"):
        cache.advance([33, 0, 0])
    assert cache.get_seq_length(a) == 0 and cache.cached.tolist() == [0, -1, -1]
    cache.advance(32)
    assert cache.get_seq_length(a) == 32


def test_tokens_that_a_captured_step_lost_are_told():
    import warnings

    cache = make()
    a, b = cache.add(), cache.add()
    cache.reserve([16, 16, 0])
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        cache.advance_device(16)
        cache.advance(16, device=False)   # as many as were reserved
    cache.advance_device(1)               # a step that nothing was reserved for
    with pytest.warns(RuntimeWarning, match="place 0 counts 17 tokens, but blocks for 16 are reserved"):
        cache.advance([1, 0, 0], device=False)
    with pytest.raises(ValueError, match="place 0 counts 17 tokens, its blocks hold 16"):
        cache.reserve(1)
    assert cache.free_blocks() == 8 and cache.get_seq_length(a) == 17 and cache.get_seq_length(b) == 16
    cache.truncate(a, 16)
    cache.reserve(1)
    assert cache.free_blocks() == 6


@pytest.mark.parametrize("scale", [3e38, -2.5e38])
def test_attention_refuses_a_scale_that_overflows(lib, scale):
    """sm_scale is finite in fp32, but the factor of the scores' exponent to base 2 is not."""
    assert attention(lib, scale=scale) == 1 and "finite" in text(lib)
    assert attention(lib, scale=scale * 0.7) == 1 and "null tensor pointer" in text(lib)


def test_attention_refuses_a_small_workspace(lib):
    size = lib.llmq_kv_block_attention_workspace_bytes
    for shape, stride in (((1, 1, 32, 8, 128, 128, 1024), 4096), ((73, 16, 28, 4, 128, 16, 200), 3584), ((3, 3, 4, 2, 64, 64, 16), 256)):
        tokens, sequences, q_heads, kv_heads, dim, block, width = shape
        need = size(*shape)   # (long enough to be split)
        assert need > 0
        a = dict(tokens=tokens, sequences=sequences, q_heads=q_heads, kv_heads=kv_heads, dim=dim, block=block, width=width, q_stride=stride,
                 start=16, pointer=16)
        assert attention(lib, space=need - 1, **a) == 1 and f"{need - 1} bytes" in text(lib) and str(need) in text(lib)
        assert attention(lib, space=need, workspace=None, **a) == 1 and "workspace" in text(lib)
        assert attention(lib, space=need, workspace=24, **a) == 1 and "16-byte aligned" in text(lib)
    assert size(1, 1, 32, 8, 128, 64, 15) == 0 and size(4096, 1, 32, 8, 128, 64, 10000) == 0   # a short walk, rows enough
