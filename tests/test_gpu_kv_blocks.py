"""The batch's operators over a cache in blocks (qk_norm_rope, kv_block_append, kv_block_dequant, kv_block_attention)
against their formulas in 64 bits, or, where every rounding is fixed, bit for bit.

Tolerances are bounds by arithmetic: half a step of the output's type, and what the kernels' roundings on the way can
add up to (given at each test)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
TAGS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
U32 = 2.0 ** -24   # half a step of fp32


@pytest.fixture(scope="module")
def ext():
    from llmquant.hip import load_extension

    return load_extension()


def half_step(dtype, want):
    """Half a step of `dtype` at the values `want` (its smallest subnormals included)."""
    info = torch.finfo(dtype)
    return torch.clamp(want.abs() * (info.eps / 2), min=info.tiny * info.eps / 2)


# ---- the norm of heads and the rotation ------------------------------------------------------------------------------
def norm_rope64(x, weight, cos, sin, eps):
    """x [tokens, heads, D] and cos, sin [tokens, R] in 64 bits -> (result, sum of the magnitudes that make an element)."""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight
    half = cos.shape[-1] // 2
    cos, sin = cos[:, None], sin[:, None]
    turned = torch.cat([-y[..., half:2 * half], y[..., :half]], -1)
    out, size = y.clone(), y.abs()
    out[..., :2 * half] = y[..., :2 * half] * cos + turned * sin
    size[..., :2 * half] = (y[..., :2 * half] * cos).abs() + (turned * sin).abs()
    return out, size


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary,wide,kind", [
    (1, 32, 8, 128, 128, False, "int32"), (1, 4, 4, 64, 64, True, "none"), (7, 6, 2, 128, 64, True, "int64"),
    (33, 5, 1, 256, 256, False, "int32"), (3, 7, 0, 96, 96, True, "int32"), (65, 3, 3, 80, 32, False, "int64"),
    (5, 0, 2, 16, 16, True, "none"), (257, 28, 4, 128, 128, True, "int32"), (2, 1, 1, 240, 48, False, "int32")])
def test_norm_and_rotation(ext, dtype, tokens, q_heads, kv_heads, dim, rotary, wide, kind):
    g = torch.Generator().manual_seed(tokens * dim)
    rows, eps = 300, 1e-6
    # queries and keys as column blocks of wider rows; a head of zeros, a very small and a very large one among them
    flat = torch.randn(tokens, (q_heads + kv_heads + 2) * dim, generator=g) * 2
    flat[0, :dim] = 0.0
    flat[-1, dim:2 * dim] *= 1e-4
    flat[-1, -dim * 2:] *= 100.0
    flat = flat.to(dtype).cuda()
    q, k = flat[:, dim:(1 + q_heads) * dim], flat[:, (1 + q_heads) * dim:(1 + q_heads + kv_heads) * dim]
    qw, kw = ((1 + torch.randn(dim, generator=g)).to(dtype).cuda() for _ in range(2))
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * (100.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary))
    # (the two halves of a row need not be alike: the formula takes each element's own)
    table = torch.float32 if wide else dtype
    cos, sin = torch.cat([angle.cos(), angle.cos() * 0.5], -1).to(table).cuda(), torch.cat([angle.sin(), angle.sin() + 0.1], -1).to(table).cuda()
    position = None if kind == "none" else torch.randint(0, rows, (tokens,), generator=g).to(getattr(torch, kind)).cuda()
    got = ext.qk_norm_rope(q, k, qw, kw, cos, sin, eps, position)
    at = torch.arange(tokens, device="cuda") if position is None else position.long()
    for out, x, w, heads in zip(got, (q, k), (qw, kw), (q_heads, kv_heads)):
        assert out.shape == (tokens, heads, dim) and out.dtype == dtype and out.is_contiguous()
        want, size = norm_rope64(x.double().reshape(tokens, heads, dim), w.double(), cos[at].double(), sin[at].double(), eps)
        # fp32 on the way: a sum of squares (at most 16 + 5 roundings in a row, halved by the root), the mean, the root, the
        # reciprocal, two products (5), a product and a multiply-add (2): below 20 half steps of what is added up
        assert torch.all((out.double() - want).abs() <= half_step(dtype, want) + 20 * U32 * size)


def test_norm_of_positions_outside_the_tables(ext):
    q, w = torch.randn(5, 128, device="cuda"), torch.ones(64, device="cuda")
    table = torch.ones(4, 32, device="cuda")
    position = torch.tensor([0, -1, 3, 4, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    for where in (position, position.long() * 2 ** 20):
        known = ((where >= 0) & (where < 4)).cpu()
        for out in ext.qk_norm_rope(q, q, w, w, table, table, 1e-5, where):
            nan = out.isnan().cpu()
            assert torch.equal(nan.all(-1).all(-1), ~known) and torch.equal(nan.any(-1).any(-1), ~known)


def test_norm_takes_odd_layouts(ext):
    """Rows that are not 16-byte aligned, transposed and expanded tensors: copied, same bits."""
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(6, 4 * 64 + 1, generator=g, device="cuda", dtype=torch.float16)
    w, table = torch.ones(64, device="cuda", dtype=torch.float16), torch.rand(6, 64, generator=g, device="cuda")
    plain = ext.qk_norm_rope(base[:, 1:].contiguous(), base[:, 1:129].contiguous(), w, w, table, table, 1e-5)
    odd = ext.qk_norm_rope(base[:, 1:], base[:, 1:129], w, w, table, table, 1e-5)
    turned = ext.qk_norm_rope(base[:, 1:].t().contiguous().t(), base[:, 1:129], w[:1].expand(64), w, table.t().contiguous().t(), table, 1e-5)
    same = ext.qk_norm_rope(base[:1, 1:].expand(6, -1), base[:, 1:129], w, w, table[:1].expand(6, -1), table[:1].expand(6, -1), 1e-5)
    assert all(torch.equal(a, b) for a, b in zip(plain * 2, odd + turned))
    assert torch.equal(same[0], same[0][:1].expand(6, -1, -1))


# ---- a batch's cache ---------------------------------------------------------------------------------------------------
def make_cache(g, blocks, heads, block, dim, outliers=True):
    """Codes and scales of any values, on the CPU; scales far from each other from block to block."""
    k = torch.randint(-127, 128, (blocks, heads, block, dim), generator=g, dtype=torch.int8)
    v = torch.randint(-127, 128, (blocks, heads, block // 16, dim, 16), generator=g, dtype=torch.int8)
    ks, vs = (torch.exp(0.5 * torch.randn(blocks, heads, generator=g)) / 60 for _ in range(2))
    if outliers and blocks > 2:
        vs[1] *= 1e4   # one block's values are far above the others', another's far below
        vs[2] *= 1e-5
    return [k, v, ks, vs]


def make_table(g, counts, blocks, spare=1):
    """Blocks for sequences of `counts` blocks each, in any order; entries behind them name no block."""
    order = torch.randperm(blocks, generator=g, dtype=torch.int64).tolist()
    table = torch.full((len(counts), max(counts) + spare), -1, dtype=torch.int32)
    for b, n in enumerate(counts):
        table[b, :n] = torch.tensor(order[:n], dtype=torch.int32)
        order = order[n:]
    return table


def starts_of(new):
    return torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)


def rows_first(v):
    """Value codes [.., block / 16, D, 16] as [.., block, D]."""
    return np.ascontiguousarray(np.swapaxes(v, -1, -2)).reshape(*v.shape[:-3], -1, v.shape[-2])


def append_oracle(x, codes, scale, table, cached, start, block):
    """fp32 with every rounding in its place; x [tokens, heads, D], codes [blocks, heads, block, D] (changed)."""
    f = np.float32
    for b in range(len(cached)):
        n, c = int(start[b + 1] - start[b]), int(cached[b])
        if c < 0:
            continue
        for logical in range(c // block, (c + n - 1) // block + 1 if n else 0):
            id = table[b, logical] if logical < table.shape[1] else -1
            if not 0 <= id < len(codes):
                continue
            lo, hi = max(c, logical * block), min(c + n, (logical + 1) * block)
            rows = x[start[b] + lo - c:start[b] + hi - c].astype(f)       # [new, heads, D]
            s = np.maximum(np.abs(rows).max((0, 2)) * (f(1) / f(127)), f(1e-8))
            old = lo - logical * block
            if old:
                before = scale[id].copy()
                s = np.maximum(s, before)
                moved = np.clip(np.rint(codes[id, :, :old].astype(f) * before[:, None, None] / s[:, None, None]), -128, 127)
                codes[id, :, :old] = np.where((s > before)[:, None, None], moved, codes[id, :, :old]).astype(np.int8)
            scale[id] = s
            codes[id, :, old:hi - logical * block] = np.clip(np.rint(rows.transpose(1, 0, 2) / s[:, None, None]), -128, 127).astype(np.int8)


APPENDS = [  # block, D, heads, cached, new (None: a row each)
    (64, 64, 2, [0], None), (64, 128, 1, [0, 1, 63, 64, 65, -1, 640], None), (16, 64, 8, [15, 16, 17, 31, 0], None),
    (128, 256, 3, [127, 128, 5], None), (32, 128, 4, [0, 31, 40, -1, 7], [100, 1, 0, 9, 33]), (64, 64, 1, [0], [64]),
    (16, 256, 2, [3, 0, 16], [200, 16, 15]), (128, 64, 5, [100, 0], [27, 300]), (64, 128, 2, [10] * 70, [3] * 70),
    (64, 128, 1, [70] * 130, None), (32, 64, 3, [0, 0, 0], [0, 0, 5]), (128, 128, 2, [130], [1]), (16, 128, 1, [0, -1], [1, 0])]


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
@pytest.mark.parametrize("block,dim,heads,cached,new", APPENDS)
def test_append_bit_for_bit(ext, dtype, block, dim, heads, cached, new):
    """Every code and scale of the cache, those that the call must leave alone too."""
    counts = [(max(c, 0) + n - 1) // block + 1 for c, n in zip(cached, new or [1] * len(cached))]
    g = torch.Generator().manual_seed(sum(counts) + dim)
    blocks = sum(counts) + 3
    cache, table = make_cache(g, blocks, heads, block, dim, outliers=False), make_table(g, counts, blocks)
    start = starts_of(new or [1] * len(cached))
    rows = torch.randn(int(start[-1]), 2, heads, dim, generator=g) * torch.exp(torch.randn(int(start[-1]), 2, heads, 1, generator=g))
    if len(rows) > 1:
        rows[1, :, 0] = 0.0     # a token of zeros
    rows = rows.to(dtype)
    cache[2][table[0, 0], 0] = float("nan") if cached[0] == 0 else 1e-3   # (a new block's old scale does not count)
    want_k, want_ks = cache[0].numpy().copy(), cache[2].numpy().copy()
    want_v, want_vs = rows_first(cache[1].numpy()), cache[3].numpy().copy()
    append_oracle(rows[:, 0].float().numpy(), want_k, want_ks, table.numpy(), cached, start.numpy(), block)
    append_oracle(rows[:, 1].float().numpy(), want_v, want_vs, table.numpy(), cached, start.numpy(), block)
    on_gpu = [t.cuda() for t in cache]
    side = rows.cuda()   # keys and values as slices of one tensor
    args = (side[:, 0], side[:, 1], *on_gpu, table.cuda(), torch.tensor(cached, dtype=torch.int32, device="cuda"),
            None if new is None else start.cuda())
    ext.kv_block_append(*args)
    for _ in range(2):
        k, v, ks, vs = (t.cpu().numpy() for t in on_gpu)
        np.testing.assert_array_equal(ks, want_ks)
        np.testing.assert_array_equal(vs, want_vs)
        np.testing.assert_array_equal(k, want_k)
        np.testing.assert_array_equal(rows_first(v), want_v)
        ext.kv_block_append(*args)   # the same rows at the same places again change nothing


def test_append_token_by_token_stays_within_its_steps(ext):
    """A block that is filled one token at a time: half a step of the last scale for each time that it grew, and half."""
    g = torch.Generator().manual_seed(5)
    block, dim, heads = 64, 128, 2
    cache, table = [t.cuda() for t in make_cache(g, 2, heads, block, dim)], torch.tensor([[1]], dtype=torch.int32, device="cuda")
    rows = (torch.randn(block, heads, dim, generator=g) * torch.exp(torch.randn(block, heads, 1, generator=g))).cuda()
    grew = torch.zeros(heads, dtype=torch.int64)
    for t in range(block):
        before = cache[2][1].cpu()
        ext.kv_block_append(rows[t:t + 1], rows[t:t + 1], *cache, table, torch.tensor([t], dtype=torch.int32, device="cuda"))
        grew += cache[2][1].cpu() > before if t else 1
    largest = rows.abs().amax((0, 2)).cpu()
    assert torch.equal(cache[2][1].cpu(), largest * torch.tensor(np.float32(1) / np.float32(127)))
    for codes in (cache[0][1].cpu().double(), torch.from_numpy(rows_first(cache[1][1].cpu().numpy())).double()):
        off = (codes * cache[2][1].cpu()[:, None, None].double() - rows.cpu().double().transpose(0, 1)).abs().amax((1, 2))
        assert torch.all(off <= 0.5 * grew * cache[2][1].cpu().double() * (1 + 1e-5)) and int(grew.max()) < 12


def test_append_leaves_out_tokens_without_a_block(ext):
    g = torch.Generator().manual_seed(9)
    block, dim, heads = 16, 64, 2
    cache = make_cache(g, 3, heads, block, dim)
    # beyond the table, no block, an id above the cache's, in the first and in the middle sequence
    table = torch.tensor([[0, -1], [3, 1], [2, 2 ** 31 - 1]], dtype=torch.int32)
    cached, start = [10, 0, 20], starts_of([30, 20, 20])
    rows = torch.randn(70, heads, dim, generator=g)
    want_k, want_ks = cache[0].numpy().copy(), cache[2].numpy().copy()
    append_oracle(rows.numpy(), want_k, want_ks, table.numpy(), cached, start.numpy(), block)
    on_gpu = [t.cuda() for t in cache]
    ext.kv_block_append(rows.cuda(), rows.cuda(), *on_gpu, table.cuda(), torch.tensor(cached, dtype=torch.int32, device="cuda"), start.cuda())
    np.testing.assert_array_equal(on_gpu[0].cpu().numpy(), want_k)
    np.testing.assert_array_equal(on_gpu[2].cpu().numpy(), want_ks)
    # positions near the end of 32 bits, more rows than the starts name, fewer sequences than a table's
    far = torch.tensor([2 ** 31 - 1, 2 ** 31 - 8, -2 ** 31], dtype=torch.int32, device="cuda")
    held = [t.clone() for t in on_gpu]
    ext.kv_block_append(rows.cuda(), rows.cuda(), *on_gpu, table.cuda(), far, start.cuda())
    assert all(torch.equal(a, b) for a, b in zip(held, on_gpu))


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
@pytest.mark.parametrize("block,dim,heads,first,count", [
    (64, 64, 2, None, [1]), (64, 128, 1, None, [64, 0, 65, 200]), (16, 64, 3, [5, 16, 0], [1, 40, 16]),
    (32, 256, 2, [31, 0], [2, 33]), (128, 128, 4, [100, 128, 7], [29, 127, 300]), (128, 64, 1, None, [3] * 70)])
def test_dequant_is_the_product_rounded(ext, dtype, block, dim, heads, first, count):
    g = torch.Generator().manual_seed(dim + sum(count))
    begin = first or [0] * len(count)
    counts = [max((f + n - 1) // block + 1, 1) for f, n in zip(begin, count)]
    blocks = sum(counts) + 1
    cache, table = make_cache(g, blocks, heads, block, dim), make_table(g, counts, blocks)
    table[-1, 0] = blocks   # no block: zeros
    tokens = sum(count)
    on_gpu = [t.cuda() for t in cache]
    got = ext.kv_block_dequant(*on_gpu, table.cuda(), starts_of(count).cuda(), tokens, dtype,
                               None if first is None else torch.tensor(first, dtype=torch.int32, device="cuda"))
    flat = [cache[0], torch.from_numpy(rows_first(cache[1].numpy()))]
    for out, codes, scale in zip(got, flat, cache[2:]):
        want = torch.zeros(heads, tokens, dim)
        at = 0
        for b, n in enumerate(count):
            for p in range(begin[b], begin[b] + n):
                id = int(table[b, p // block])
                if 0 <= id < blocks:
                    want[:, at] = codes[id, :, p % block].float() * scale[id][:, None]
                at += 1
        assert out.shape == want.shape and torch.equal(out.cpu(), want.to(dtype))


# ---- attention -----------------------------------------------------------------------------------------------------------
def attention64(q, cache, table, cached, start, block, scale, bias, weight_step):
    """(result, bound of what the kernel's roundings on the way can add), both [tokens, q_heads, D] in 64 bits, NaN in
    rows of no sequence. Roundings: the scores' sums of D products of a query and a code (the code may enter with `bias`, which
    is taken out again); queries as 11-bit pieces below their row's largest; softmax weights as numbers of `weight_step`,
    at the least 2^-25 of the row's largest; and a handful of fp32 operations on each weight and sum."""
    tokens, q_heads, dim = q.shape
    keys, values = cache[0].double() * cache[2].double()[..., None, None], torch.from_numpy(rows_first(cache[1].numpy())).double() * cache[3].double()[..., None, None]
    heads = keys.shape[1]
    out, bound = torch.full(q.shape, float("nan"), dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(cached)):
        for i in range(int(start[b + 1] - start[b])):
            row, limit = int(start[b]) + i, int(cached[b]) + i + 1 if cached[b] >= 0 else 0
            at = [(int(table[b, p // block]), p % block) for p in range(min(limit, table.shape[1] * block)) if 0 <= int(table[b, p // block]) < len(keys)]
            out[row] = 0.0
            if not at:
                continue
            ids, slots = (torch.tensor(t) for t in zip(*at))
            for h in range(q_heads):
                k, v, x = keys[ids, h * heads // q_heads, slots], values[ids, h * heads // q_heads, slots], q[row, h].double()
                step = cache[2][ids, h * heads // q_heads].double()
                t = scale * (k @ x)
                p = torch.softmax(t, 0)
                out[row, h] = p @ v
                x_off = (2.0 ** -22 * x.abs() if weight_step < 2.0 ** -12 else 0.0) + 2.0 ** -25 * x.abs().max()
                off = abs(scale) * (k.abs() @ (x_off + torch.zeros(dim, dtype=torch.float64)) + U32 * (dim + 8) * ((k.abs() + bias * step[:, None]) @ x.abs()))
                off = off + 4 * U32 * (t.abs() + (t.abs().max()) + 24)       # the exponent's own roundings
                rel = weight_step + 2 * float(off.max()) + 40 * U32 + len(at) * U32
                weighted = p * cache[3][ids, h * heads // q_heads].double()
                bound[row, h] = rel * (p @ v.abs()) + len(at) * 2.0 ** -25 * (1 if weight_step > 2.0 ** -12 else 2.0 ** -11) * 127 * weighted.max()
    return out, bound


def check_attention(ext, dtype, block, dim, heads, group, cached, new, seed=0, table=None, out=None, rows=None, scale=None, adjust=None):
    g = torch.Generator().manual_seed(seed + dim * block + sum(cached))
    count = new or [1] * len(cached)
    counts = [max((max(c, 0) + n - 1) // block + 1, 1) for c, n in zip(cached, count)]
    blocks = sum(counts) + 2 if table is None else 9
    cache = make_cache(g, blocks, heads, block, dim)
    table = make_table(g, counts, blocks) if table is None else table
    start = starts_of(count)
    q = (torch.randn(rows or int(start[-1]), heads * group, dim, generator=g) * 1.5).to(dtype)
    if adjust:
        adjust(q, cache, table)
    scale = dim ** -0.5 if scale is None else scale
    on_gpu = [t.cuda() for t in cache]
    args = (q.cuda(), *on_gpu, table.cuda(), torch.tensor(cached, dtype=torch.int32, device="cuda"), scale,
            None if new is None else start.cuda())
    got = ext.kv_block_attention(*args) if out is None else ext.kv_block_attention(*args, out)
    assert got.shape == (len(q), heads * group * dim) and got.dtype == dtype
    narrow = dtype != torch.float32
    want, bound = attention64(q, cache, table, cached, start, block, scale, 1152.0 if narrow else 0.0, 2.0 ** -11 if narrow else 2.0 ** -22)
    covered = int(start[-1])
    off = (got.cpu().double().reshape(want.shape) - want)[:covered].abs()
    tolerance = (half_step(dtype, want) + bound)[:covered]
    assert torch.all(off <= tolerance), f"worst {float((off / tolerance).max()):.3f} of what may be"
    assert torch.equal(got, ext.kv_block_attention(*args) if out is None else ext.kv_block_attention(*args, out))   # the same bits again
    return got, args


STEPS = [  # block, D, kv heads, group, cached, new
    (64, 64, 1, 1, [0], None), (64, 64, 2, 4, [0, 1, 14, 15, 16, 62, 63, 64, 65], None), (16, 128, 2, 4, [300, 0, -1, 15, 31], None),
    (32, 64, 1, 7, [33, 31, 95, 257], None), (128, 128, 1, 8, [127, 128, 500], None), (64, 256, 2, 2, [70, 3], None),
    (128, 256, 1, 3, [200], None), (16, 64, 1, 16, [47, 200], None), (64, 128, 1, 24, [90], None), (16, 256, 1, 1, [17], None),
    (64, 128, 1, 40, [65, 130], None), (64, 64, 1, 100, [66], None), (32, 128, 3, 5, [-1, -1, 40], None)]
DRAFTS = [
    (64, 64, 1, 4, [60, 0, 200], [5, 3, 4]), (16, 128, 1, 7, [100, 31, -1, 0], [4, 5, 2, 1]), (32, 64, 2, 1, [10, 40], [17, 0]),
    (64, 128, 1, 8, [3], [9]), (128, 64, 1, 2, [0, 130], [33, 8]), (64, 256, 1, 4, [20], [6]), (16, 64, 1, 4, [5] * 67, [2] * 67)]
PROMPTS = [
    (64, 64, 1, 4, [0], [130]), (16, 128, 1, 2, [37, 0], [70, 150]), (64, 128, 1, 1, [200], [100]), (32, 256, 1, 2, [0, 9], [75, 40]),
    (128, 64, 1, 3, [0, 3, 100], [1, 200, 40]), (64, 64, 1, 1, [64], [64]), (64, 128, 2, 4, [0], [65])]


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
@pytest.mark.parametrize("block,dim,heads,group,cached,new", STEPS + DRAFTS + PROMPTS)
def test_attention(ext, dtype, block, dim, heads, group, cached, new):
    check_attention(ext, dtype, block, dim, heads, group, cached, new)


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_of_long_sequences(ext, dtype, dim):
    """Long enough for the work to be split over the tokens, short sequences and one of nothing beside them."""
    check_attention(ext, dtype, 64, dim, 1, 4, [5000, 3, -1, 0, 1500], None)
    check_attention(ext, dtype, 16, dim, 2, 2, [2600], [3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=TAGS.get)
def test_attention_without_some_blocks(ext, dtype):
    """Blocks that are none, in the middle, at the end and throughout; a sequence longer than its table."""
    table = torch.tensor([[0, -1, 2, 99], [-1, -1, -1, -1], [3, 4, 5, 6], [2 ** 31 - 1, 7, -2 ** 31, 1]], dtype=torch.int32)
    check_attention(ext, dtype, 16, 64, 2, 2, [60, 60, 300, 40], None, table=table)
    check_attention(ext, dtype, 32, 128, 1, 4, [100, 5, 126, 70], [3, 2, 9, 40], table=table)
    check_attention(ext, dtype, 64, 64, 1, 1, [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 2, 200], None, table=table)


def test_attention_leaves_rows_of_no_sequence(ext):
    for new, cached in (([3, 0, 2], [70, 5, 9]), ([40, 1, 30], [2, 0, 100])):
        out = torch.full((sum(new) + 7, 4 * 64), 7.5, device="cuda", dtype=torch.float16)
        check_attention(ext, torch.float16, 16, 64, 1, 4, cached, new, out=out, rows=sum(new) + 7)
        assert torch.all(out[sum(new):] == 7.5)


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
def test_attention_of_far_apart_values(ext, dtype):
    """Queries whose elements lie far apart, scores that leave one token, scales of zero, negative and large factors."""
    def wide(q, cache, table):
        q[..., 0] *= 300.0
        q[..., 1] *= 1e-4
        q[0, 0] = 0.0
        q[0, 1] *= 1e-3 if dtype == torch.float16 else 1e-30

    def nothing(q, cache, table):
        cache[2][table[0, 0]] = 0.0
        cache[3][table[0, 1]] = 0.0
        cache[3][table[1, 0]] = 1e-8

    check_attention(ext, dtype, 16, 64, 1, 4, [90, 40], None, adjust=wide)
    check_attention(ext, dtype, 16, 64, 1, 4, [90, 40], None, adjust=nothing)
    check_attention(ext, dtype, 64, 128, 1, 2, [90, 200], [2, 3], scale=-0.05)
    check_attention(ext, dtype, 64, 64, 1, 2, [130], None, scale=0.0)


def test_values_behind_the_last_token_do_not_count(ext):
    """Places behind a sequence's last token, and blocks of other sequences, may hold anything."""
    g = torch.Generator().manual_seed(1)
    cache = make_cache(g, 4, 2, 32, 64)
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, generator=g).half().cuda()
    cached = torch.tensor([40, 3], dtype=torch.int32, device="cuda")
    plain = ext.kv_block_attention(q, *[t.cuda() for t in cache], table, cached, 0.125)
    cache[0][0, :, 9:] = -128
    cache[1][0, :, 1, :, :] = -128          # tokens 16 .. 31 of that block: behind the last one
    cache[1][0, :, 0, :, 9:] = -128
    cache[0][3], cache[1][3] = 127, 127
    cache[2][3], cache[3][3] = float("nan"), float("inf")
    assert torch.equal(plain, ext.kv_block_attention(q, *[t.cuda() for t in cache], table, cached, 0.125))


def test_a_query_that_is_not_a_number_stays_in_its_rows(ext):
    g = torch.Generator().manual_seed(2)
    cache = [t.cuda() for t in make_cache(g, 4, 1, 64, 64)]
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 3, 64, generator=g).cuda()
    cached = torch.tensor([70, 90], dtype=torch.int32, device="cuda")
    for dtype in DTYPES:
        clean = ext.kv_block_attention(q.to(dtype), *cache, table, cached, 0.125).reshape(2, 3, 64)
        for bad in (float("nan"), float("inf")):
            x = q.clone()
            x[0, 1, 5] = bad
            got = ext.kv_block_attention(x.to(dtype), *cache, table, cached, 0.125).reshape(2, 3, 64)
            assert got[0, 1].isnan().all()
            got[0, 1] = clean[0, 1]
            assert torch.equal(got, clean)


# ---- together ----------------------------------------------------------------------------------------------------------
def test_refusals(ext):
    cache = [t.cuda() for t in make_cache(torch.Generator().manual_seed(0), 2, 2, 16, 64)]
    table, cached = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    row, q = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 4, 64, device="cuda")

    def refused(what, call, *args):
        with pytest.raises(RuntimeError, match=what):
            call(*args)

    append, attend, back = ext.kv_block_append, ext.kv_block_attention, ext.kv_block_dequant
    refused("one row", append, row.expand(2, -1, -1), row.expand(2, -1, -1), *cache, table, cached)
    refused("of one dtype", append, row, row.half(), *cache, table, cached)
    refused("of one dtype", append, row[..., :32], row[..., :32], *cache, table, cached)
    refused("float32, float16 or bfloat16", append, row.double(), row.double(), *cache, table, cached)
    refused("cached must be int32", append, row, row, *cache, table, cached.long())
    refused("block_table must be int32", append, row, row, *cache, table.long(), cached)
    refused("query_start must be int32", append, row, row, *cache, table, cached, cached)
    refused("v_codes must be", append, row, row, cache[0], cache[0], *cache[2:], table, cached)
    refused("k_codes must be", append, row, row, cache[0].transpose(0, 1), *cache[1:], table, cached)
    refused("scales must be", append, row, row, *cache[:2], cache[2].half(), cache[3], table, cached)
    refused("cache's device", append, row.cpu(), row, *cache, table, cached)
    refused("CUDA", append, row, row, *[t.cpu() for t in cache], table, cached)
    refused("not a multiple of kv_heads", attend, torch.zeros(1, 3, 64, device="cuda"), *cache, table, cached, 1.0)
    refused("query must be", attend, torch.zeros(1, 4, 32, device="cuda"), *cache, table, cached, 1.0)
    refused("finite", attend, q, *cache, table, cached, float("inf"))
    refused("finite", attend, q, *cache, table, cached, float("nan"))
    refused("out must be", attend, q, *cache, table, cached, 1.0, None, torch.zeros(1, 4, 64, device="cuda"))
    refused("n_tokens is out of range", back, *cache, table, torch.zeros(2, dtype=torch.int32, device="cuda"), -1, torch.float16)
    refused("starts must be int32", back, *cache, table, cached, 1, torch.float16)
    narrow = [cache[0][..., :32].contiguous(), cache[1][..., :32, :].contiguous(), *cache[2:]]
    refused("head_dim must be 64", attend, torch.zeros(1, 2, 32, device="cuda"), *narrow, table, cached, 1.0)
    odd = [cache[0][:, :, :8].contiguous(), cache[1][:, :, :0].contiguous(), *cache[2:]]
    refused("v_codes must be", attend, q, *odd, table, cached, 1.0)
    w, t = torch.ones(64, device="cuda"), torch.ones(1, 64, device="cuda")
    flat = torch.zeros(1, 128, device="cuda")
    refused("whole heads", ext.qk_norm_rope, flat[:, :96], flat, w, w, t, t, 1e-5)
    refused("without positions", ext.qk_norm_rope, flat.expand(2, -1), flat.expand(2, -1), w, w, t, t, 1e-5)
    refused("q's dtype", ext.qk_norm_rope, flat, flat, w.half(), w, t, t, 1e-5)
    refused("rotated part", ext.qk_norm_rope, flat, flat, w, w, t[:, :36], t[:, :36], 1e-5)
    refused("rotated part", ext.qk_norm_rope, flat, flat, w, w, flat, flat, 1e-5)
    refused("eps", ext.qk_norm_rope, flat, flat, w, w, t, t, -1.0)
    refused("positions must be", ext.qk_norm_rope, flat, flat, w, w, t, t, 1e-5, torch.zeros(1, device="cuda"))


def test_nothing_to_do(ext):
    for blocks, sequences, width in ((0, 0, 0), (2, 0, 0), (0, 2, 3), (2, 2, 0)):
        cache = [torch.zeros(blocks, 2, 16, 64, dtype=torch.int8, device="cuda"), torch.zeros(blocks, 2, 1, 64, 16, dtype=torch.int8, device="cuda"),
                 torch.zeros(blocks, 2, device="cuda"), torch.zeros(blocks, 2, device="cuda")]
        table = torch.zeros(sequences, width, dtype=torch.int32, device="cuda")
        cached, row = torch.zeros(sequences, dtype=torch.int32, device="cuda"), torch.ones(sequences, 2, 64, device="cuda")
        ext.kv_block_append(row, row, *cache, table, cached)
        got = ext.kv_block_attention(row, *cache, table, cached, 1.0)
        assert got.shape == (sequences, 128) and torch.all(got == 0)
        starts = torch.arange(sequences + 1, dtype=torch.int32, device="cuda")
        for out in ext.kv_block_dequant(*cache, table, starts, sequences, torch.float16):
            assert out.shape == (2, sequences, 64) and torch.all(out == 0)
    w, t = torch.ones(64, device="cuda"), torch.ones(0, 64, device="cuda")
    q, k = ext.qk_norm_rope(torch.zeros(0, 128, device="cuda"), torch.zeros(0, 64, device="cuda"), w, w, t, t, 1e-5)
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)
    q, k = ext.qk_norm_rope(torch.ones(1, 128, device="cuda"), torch.zeros(1, 0, device="cuda"), w, w, t, t, 1e-5,
                            torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert q.isnan().all() and k.shape == (1, 0, 64)   # (a table of no rows knows no position)


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_of_many_rows_over_long_sequences(ext, dtype, dim):
    """Rows enough for waves with a row tile each (three and four of them, the last part of one), over tokens enough to be split."""
    check_attention(ext, dtype, 64, dim, 1, 4, [1990], [29])
    check_attention(ext, dtype, 16, dim, 1, 3, [1200, -1, 40], [33, 2, 35])


def test_attention_of_a_large_batch(ext):
    """More sequences than the places of several waves, most of them short, some long."""
    cached = [700 if b % 97 == 5 else -1 if b % 50 == 3 else b % 40 for b in range(450)]
    check_attention(ext, torch.bfloat16, 16, 64, 1, 2, cached, None)
    check_attention(ext, torch.float32, 32, 64, 1, 1, cached[:330], [b % 3 for b in range(330)])


def test_blocks_far_into_a_large_cache(ext):
    """Codes beyond 2^31 bytes: the same bits as at the front."""
    blocks, heads, block, dim = 17000, 8, 128, 128
    cache = [torch.zeros(blocks, heads, block, dim, dtype=torch.int8, device="cuda"),
             torch.zeros(blocks, heads, block // 16, dim, 16, dtype=torch.int8, device="cuda"),
             torch.zeros(blocks, heads, device="cuda"), torch.zeros(blocks, heads, device="cuda")]
    g = torch.Generator(device="cuda").manual_seed(4)
    rows = torch.randn(300, heads, dim, generator=g, device="cuda", dtype=torch.bfloat16)
    q = torch.randn(300, 2 * heads, dim, generator=g, device="cuda", dtype=torch.bfloat16)
    start = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = []
    for table in ([[0, 1, 2]], [[16999, 16500, 16998]]):
        table = torch.tensor(table, dtype=torch.int32, device="cuda")
        ext.kv_block_append(rows, rows, *cache, table, none, start)
        got.append((ext.kv_block_attention(q, *cache, table, none, 0.1, start),
                    ext.kv_block_attention(q[:1], *cache, table, none + 299, 0.1),
                    *ext.kv_block_dequant(*cache, table, start, 300, torch.float16)))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][0].abs().sum() > 0 and got[0][2].abs().sum() > 0


def fresh(cls, **change):
    return cls(**(dict(num_layers=2, kv_heads=2, head_dim=64, num_blocks=40, max_sequences=3, max_len=400, block=16) | change))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=TAGS.get)
def test_a_batch_as_it_is_served(ext, dtype):
    """Prompts, a prompt's second chunk, single tokens, drafts some of which are taken back, a sequence that ends and one that takes
    its place: norm and rotation, append, attention, reading back, each against its formula on what the others gave."""
    from llmquant.runtime import BlockQuantCache

    cache, heads, group, dim = fresh(BlockQuantCache), 2, 3, 64
    g = torch.Generator().manual_seed(11)
    qw, kw = ((1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).cuda() for _ in range(2))
    angle = torch.arange(400, dtype=torch.float64)[:, None] * (1000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim))
    cos, sin = (torch.cat([t, t], -1).float().cuda() for t in (angle.cos(), angle.sin()))
    narrow = dtype != torch.float32
    codes = [[np.zeros((40, heads, 16, dim), np.int8) for _ in range(2)] for _ in range(2)]
    scales = [[np.zeros((40, heads), np.float32) for _ in range(2)] for _ in range(2)]

    def step(new):
        cache.reserve(new)
        held = [max(cache._lengths[p], 0) if cache._lengths[p] >= 0 else -1 for p in range(3)]
        start = None if all(n == 1 for n in new) else starts_of(new)
        offsets = starts_of(new)
        tokens = int(offsets[-1])
        position = torch.cat([torch.arange(max(h, 0), max(h, 0) + n) for h, n in zip(held, new)]).to(torch.int32)
        table = cache.block_table.cpu()
        for layer in range(2):
            qkv = torch.randn(tokens, (heads * group + 2 * heads) * dim, generator=g).to(dtype).cuda()
            k_at, v_at = heads * group * dim, (heads * group + heads) * dim
            q, k = ext.qk_norm_rope(qkv[:, :k_at], qkv[:, k_at:v_at], qw, kw, cos, sin, 1e-6, position.cuda())
            want_q, size = norm_rope64(qkv[:, :k_at].double().reshape(tokens, -1, dim), qw.double(), cos[position.long().cuda()].double(),
                                       sin[position.long().cuda()].double(), 1e-6)
            assert torch.all((q.double() - want_q).abs() <= half_step(dtype, want_q) + 20 * U32 * size)
            value = qkv[:, v_at:].unflatten(1, (heads, dim))
            cache.append(layer, k, value, None if start is None else start.cuda())
            for x, which in ((k, 0), (value, 1)):
                append_oracle(x.float().cpu().numpy(), codes[layer][which], scales[layer][which], table.numpy(), held, offsets.numpy(), 16)
            np.testing.assert_array_equal(cache.k_codes[layer].cpu().numpy(), codes[layer][0])
            np.testing.assert_array_equal(rows_first(cache.v_codes[layer].cpu().numpy()), codes[layer][1])
            np.testing.assert_array_equal(cache.k_scale[layer].cpu().numpy(), scales[layer][0])
            got = cache.attend(layer, q, 0.125, None if start is None else start.cuda())
            on_cpu = [cache.k_codes[layer].cpu(), cache.v_codes[layer].cpu(), cache.k_scale[layer].cpu(), cache.v_scale[layer].cpu()]
            want, bound = attention64(q.cpu(), on_cpu, table, held, offsets, 16, 0.125, 1152.0 if narrow else 0.0, 2.0 ** -11 if narrow else 2.0 ** -22)
            assert torch.all((got.cpu().double().reshape(want.shape) - want).abs() <= half_step(dtype, want) + bound)
        cache.advance(new)

    cache.add(), cache.add()
    step([50, 17, 0])
    step([70, 1, 0])             # the first prompt's second chunk, the second sequence's next token
    assert cache.add() == 2
    step([1, 1, 33])
    step([1, 1, 1])
    step([5, 4, 1])              # drafts
    cache.truncate(0, cache.get_seq_length(0) - 3)
    cache.truncate(1, cache.get_seq_length(1) - 4)
    step([1, 1, 1])
    cache.release(1)
    step([1, 0, 1])
    assert cache.add() == 1
    step([1, 40, 1])
    for place in range(3):
        k, v = cache.dequantized(1, place, torch.float32)
        for out, which in ((k, 0), (v, 1)):
            ids = cache._blocks[place]
            want = (codes[1][which][ids] * scales[1][which][ids][..., None, None]).transpose(1, 0, 2, 3).reshape(heads, -1, dim)
            np.testing.assert_array_equal(out.cpu().numpy(), want[:, :cache.get_seq_length(place)])


def test_a_captured_step_replays(ext):
    """A step of two layers in a graph, replayed with eager work of the same program in between: outputs and the whole cache are
    the eager step's, bit for bit, while sequences grow through blocks and one place is empty."""
    from llmquant.runtime import BlockQuantCache

    # (max_len: long enough that the tokens are split and merged)
    eager, graphed = (fresh(BlockQuantCache, max_len=2048, num_blocks=300) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.ones(64, device="cuda", dtype=torch.float16)
    angle = torch.arange(2048, device="cuda")[:, None] * (1000.0 ** (-torch.arange(0, 64, 2, device="cuda") / 64))
    cos, sin = (torch.cat([t, t], -1) for t in (angle.cos(), angle.sin()))
    static = torch.zeros(3, 8 * 64, device="cuda", dtype=torch.float16)

    def step(cache, rows):
        outs = []
        for layer in range(2):
            q, k = ext.qk_norm_rope(rows[:, :256], rows[:, 256:384], w, w, cos, sin, 1e-6, cache.cached)
            cache.append(layer, k, rows[:, 384:].unflatten(1, (2, 64)))
            outs.append(cache.attend(layer, q, 0.125))
        cache.advance_device(1)
        return outs

    start = torch.tensor([0, 900, 0 + 900, 1000], dtype=torch.int32, device="cuda")
    prompt = torch.randn(1000, 2, 64, generator=g, device="cuda", dtype=torch.float16)
    for cache in (eager, graphed):
        cache.add(), cache.add(), cache.add(), cache.release(1)
        cache.reserve([900, 0, 100])
        for layer in range(2):
            cache.append(layer, prompt, prompt, start)
        cache.advance([900, 0, 100])
        cache.reserve([40, 0, 40])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # (a warm-up, taken back)
        step(graphed, static)
    torch.cuda.current_stream().wait_stream(side)
    for place in (0, 2):
        graphed.truncate(place, graphed.get_seq_length(place))
    for a, b in zip((eager.k_codes, eager.v_codes, eager.k_scale, eager.v_scale), (graphed.k_codes, graphed.v_codes, graphed.k_scale, graphed.v_scale)):
        b.copy_(a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(graphed, static)
    for turn in range(37):
        rows = torch.randn(3, 8 * 64, generator=g, device="cuda", dtype=torch.float16) * (1 + 0.1 * turn)
        want = step(eager, rows)
        static.copy_(rows)
        graph.replay()
        if turn % 3 == 0:
            torch.cuda.synchronize()
        for a, b in zip(want, captured):
            assert torch.equal(a, b) and torch.all(a[1] == 0) and a[0].abs().sum() > 0
        assert torch.equal(eager.cached, graphed.cached)
    for a, b in ((eager.k_codes, graphed.k_codes), (eager.v_codes, graphed.v_codes), (eager.k_scale, graphed.k_scale), (eager.v_scale, graphed.v_scale)):
        assert torch.equal(a, b)


def test_two_streams_at_once(ext):
    """Calls on two streams, each with its workspace, beside each other: the bits of one after the other."""
    g = torch.Generator().manual_seed(6)
    sets = []
    for seed in range(2):
        cache, table = make_cache(g, 60, 2, 64, 128, outliers=False), make_table(g, [50, 3, 1], 60)
        sets.append((torch.randn(3, 8, 128, generator=g).bfloat16().cuda(), *[t.cuda() for t in cache], table.cuda(),
                     torch.tensor([3150, 150, 9 + seed], dtype=torch.int32, device="cuda"), 0.09))
    want = [ext.kv_block_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(ext.kv_block_attention(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(w, x) for w, xs in zip(want, got) for x in xs)


@pytest.mark.parametrize("block,in_front", [(16, 15), (16, 16), (16, 100), (64, 300), (128, 128)])
def test_rows_in_front_of_the_first_sequence_are_nobodys(ext, block, in_front):
    g = torch.Generator().manual_seed(17)
    dim, heads, cached, new = 64, 2, [3, 40, -1, 0], [20, 1, 5, 33]
    counts = [-(-max(c + n, 1) // block) for c, n in zip(cached, new)]
    cache = make_cache(g, sum(counts) + 2, heads, block, dim, outliers=False)
    table, start = make_table(g, counts, sum(counts) + 2), in_front + starts_of(new)
    rows = torch.randn(in_front + sum(new) + 9, heads, dim, generator=g)
    rows[:in_front] = rows[in_front + sum(new):] = 1e4   # (would raise every scale)
    want, want_scale = cache[0].numpy().copy(), cache[2].numpy().copy()
    append_oracle(rows.numpy(), want, want_scale, table.numpy(), cached, start.numpy(), block)
    want_v, want_v_scale = rows_first(cache[1].numpy()).copy(), cache[3].numpy().copy()
    append_oracle(rows.numpy(), want_v, want_v_scale, table.numpy(), cached, start.numpy(), block)
    on_gpu = [t.cuda() for t in cache]
    lengths = torch.tensor(cached, dtype=torch.int32, device="cuda")
    ext.kv_block_append(rows.cuda(), rows.cuda(), *on_gpu, table.cuda(), lengths, start.cuda())
    np.testing.assert_array_equal(on_gpu[0].cpu().numpy(), want)
    np.testing.assert_array_equal(rows_first(on_gpu[1].cpu().numpy()), want_v)
    np.testing.assert_array_equal(on_gpu[2].cpu().numpy(), want_scale)
    np.testing.assert_array_equal(on_gpu[3].cpu().numpy(), want_v_scale)
    # read back, and attended to: as with the rows from 0 on
    shifted, plain = start.cuda(), starts_of(new).cuda()
    total = in_front + sum(new)
    for a, b in zip(ext.kv_block_dequant(*on_gpu, table.cuda(), shifted, total, torch.float32), ext.kv_block_dequant(*on_gpu, table.cuda(), plain, sum(new), torch.float32)):
        assert torch.equal(a[:, in_front:], b)
    query = torch.randn(total, 4, dim, generator=g).cuda()
    out = torch.full((total, 4 * dim), 7.5, device="cuda")
    ext.kv_block_attention(query, *on_gpu, table.cuda(), lengths, dim ** -0.5, shifted, out)
    assert torch.all(out[:in_front] == 7.5)
    assert torch.equal(out[in_front:], ext.kv_block_attention(query[in_front:], *on_gpu, table.cuda(), lengths, dim ** -0.5, plain))


def test_out_may_not_share_memory(ext):
    cache = [t.cuda() for t in make_cache(torch.Generator().manual_seed(0), 2, 2, 16, 64)]
    table, cached = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    room = torch.zeros(4, 4, 64, device="cuda")
    for out in (room[:2].view(2, 256), room[1:3].view(2, 256)):   # the query's memory, and one row of it
        with pytest.raises(RuntimeError, match="out must not share memory"):
            ext.kv_block_attention(room[:2], *cache, table, cached, 1.0, None, out)
    beside = room[2:].view(2, 256)
    assert ext.kv_block_attention(room[:2], *cache, table, cached, 1.0, None, beside).data_ptr() == beside.data_ptr()


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
def test_blocks_shared_for_reading(ext, dtype):
    g = torch.Generator().manual_seed(23)
    block, dim, heads, n = 32, 128, 2, 40
    cache = [t.cuda() for t in make_cache(g, n, heads, block, dim, outliers=False)]
    query = torch.randn(3, 8, dim, generator=g).to(dtype).cuda()
    lengths = torch.tensor([32 * 36 - 1, 700, 32 * 20], dtype=torch.int32, device="cuda")
    prefix = torch.randperm(n, generator=g)[:36].to(torch.int32)
    prefix[5] = prefix[9]   # the same block twice in a sequence
    one = prefix[None].cuda()
    attend = lambda q, t, c: ext.kv_block_attention(q, *cache, t, c, dim ** -0.5)
    got = attend(query, one.expand(3, -1), lengths)                     # one row of a table for all
    assert torch.equal(got, attend(query, one.repeat(3, 1), lengths))
    # .. and as from copies of the blocks, each sequence its own
    copies = [t[one.repeat(3, 1).flatten().long()].contiguous() for t in cache]
    own = torch.arange(3 * 36, dtype=torch.int32, device="cuda").view(3, 36)
    assert torch.equal(got, ext.kv_block_attention(query, *copies, own, lengths, dim ** -0.5))
    starts = torch.tensor([0, 100, 150, 151], dtype=torch.int32, device="cuda")
    for a, b in zip(ext.kv_block_dequant(*cache, one.expand(3, -1), starts, 151, dtype), ext.kv_block_dequant(*copies, own, starts, 151, dtype)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("cached,new,at", [(0, 30, 7), (0, 30, 25), (5, 30, 3), (5, 30, 29), (5, 1, 0), (0, 1, 0), (15, 2, 1)])
def test_append_of_values_that_are_not_finite(ext, dtype, bad, cached, new, at):
    """They show: the block's scale is not a number, and neither are its tokens in that head, when they are read back and in the
    attention rows that see them. Other blocks and heads do not change, and the block's next first token makes it whole."""
    g = torch.Generator().manual_seed(31 + cached + new)
    block, dim, heads, head = 16, 64, 2, 1
    total, spot = cached + new, (cached + at) // block
    start = torch.tensor([0, new, new + 2], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([cached, 4], dtype=torch.int32, device="cuda")
    table = torch.tensor([[2, 0, 3], [1, -1, -1]], dtype=torch.int32, device="cuda")
    first = make_cache(g, 4, heads, block, dim, outliers=False)
    rows = torch.randn(new + 2, 2, heads, dim, generator=g)
    query = torch.randn(new + 2, 4, dim, generator=g).to(dtype).cuda()
    ends = torch.tensor([0, total, total], dtype=torch.int32, device="cuda")

    def outcome(rows):
        cache = [t.cuda() for t in first]
        on_gpu = rows.to(dtype).cuda()
        ext.kv_block_append(on_gpu[:, 0], on_gpu[:, 1], *cache, table, lengths, start)
        back = ext.kv_block_dequant(*cache, table, ends, total, torch.float32)
        return cache, back, ext.kv_block_attention(query, *cache, table, lengths, 0.125, start).reshape(new + 2, 4, dim)

    clean = outcome(rows)
    for which in range(2):   # a key, a value
        spoilt = rows.clone()
        spoilt[at, which, head, 33] = bad
        cache, back, out = outcome(spoilt)
        unit = (int(table[0, spot]), head)
        assert cache[2 + which][unit].isnan()
        lo, hi = spot * block, min((spot + 1) * block, total)
        assert back[which][head, lo:hi].isnan().all()
        back[which][head, lo:hi] = clean[1][which][head, lo:hi]
        assert all(torch.equal(a, b) for a, b in zip(back, clean[1]))
        for got, want in zip(cache, clean[0]):
            got[unit] = want[unit]
            assert torch.equal(got, want)
        see = torch.arange(new + 2, device="cuda").lt(new) & (cached + torch.arange(new + 2, device="cuda") >= lo)   # the block's first token
        assert out[see][:, 2 * head:2 * head + 2].isnan().all()
        out[see, 2 * head:2 * head + 2] = clean[2][see, 2 * head:2 * head + 2]
        assert torch.equal(out, clean[2])
    # a block whose scale is not a number, from its first token on again
    cache = [t.cuda() for t in first]
    for values in (rows.clone().fill_(bad), rows):
        on_gpu = values[:1].to(dtype).cuda()
        ext.kv_block_append(on_gpu[:, 0], on_gpu[:, 1], *cache, table[:1], torch.zeros(1, dtype=torch.int32, device="cuda"))
    want = [t.numpy().copy() for t in first]
    append_oracle(rows[:1, 0].to(dtype).float().numpy(), want[0], want[2], table[:1].cpu().numpy(), [0], np.array([0, 1]), block)
    np.testing.assert_array_equal(cache[2].cpu().numpy(), want[2])
    np.testing.assert_array_equal(cache[0][:, :, 0].cpu().numpy(), want[0][:, :, 0])


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary,wide", [
    (2049, 28, 4, 128, 128, True), (13200, 7, 3, 64, 32, False), (3300, 4, 1, 256, 256, False), (9500, 5, 2, 96, 96, True),
    (33000, 3, 1, 64, 64, False), (33000, 0, 4, 64, 64, True), (9000, 1, 7, 80, 48, False), (4200, 32, 8, 128, 128, False)])
def test_norm_of_many_heads(ext, dtype, tokens, q_heads, kv_heads, dim, rotary, wide):
    """Calls of more lanes than the chip holds, where a lane takes several heads of a token (heads that are no multiple of four, lanes with
    query and key heads among them): the formula, and the bits of calls of a few tokens."""
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    flat = (torch.randn(tokens, (q_heads + kv_heads) * dim, generator=g, device="cuda") * 2).to(dtype)
    q, k = flat[:, :q_heads * dim], flat[:, q_heads * dim:]
    qw, kw = ((1 + 0.5 * torch.randn(dim, generator=g, device="cuda")).to(dtype) for _ in range(2))
    angle = torch.rand(500, rotary, generator=g, device="cuda") * 6.28
    cos, sin = (t.to(torch.float32 if wide else dtype) for t in (angle.cos(), angle.sin()))
    position = torch.randint(0, 500, (tokens,), generator=g, device="cuda")
    got = ext.qk_norm_rope(q, k, qw, kw, cos, sin, 1e-6, position)
    for out, x, w, heads in zip(got, (q, k), (qw, kw), (q_heads, kv_heads)):
        want, size = norm_rope64(x.double().reshape(tokens, heads, dim), w.double(), cos[position].double(), sin[position].double(), 1e-6)
        # (as in test_norm_and_rotation)
        assert torch.all((out.double() - want).abs() <= half_step(dtype, want) + 20 * U32 * size)
    few = [ext.qk_norm_rope(q[at:at + 600], k[at:at + 600], qw, kw, cos, sin, 1e-6, position[at:at + 600]) for at in range(0, tokens, 600)]
    assert all(torch.equal(a, torch.cat(parts)) for a, parts in zip(got, zip(*few)))


PAST = [  # block, D, kv heads, group, cached, new, rows of the table (-1, 99: no block)
    (128, 64, 1, 4, [700, 90, -1, 0, 200], None, [[0, 1, 2, 3, 4, 5], [6], [7], [8], [3, 0]]),
    (128, 128, 2, 4, [1100], None, [[8, 7, 6, 5, 4, 3, 2, 1, 0]]),
    (16, 64, 2, 2, [100, 140], None, [[0, -1, 2, 99, 4, 5, 6], [8, 7, 1, 3, 5, 0, 2, -1, 6]]),
    (64, 128, 1, 8, [300, -1, 5, 63], None, [[4, 3, 99, 1, 0], [2], [8], [7]]),
    (32, 128, 1, 4, [200, 7], [4, 3], [[0, 1, 2, 3, 4, 5, 6], [7]]),
    (64, 64, 1, 7, [0, 250, 64], [1, 2, 3], [[7], [0, 2, 4, 6], [1, 3]]),
    (16, 128, 4, 1, [127], [16], [[0, 1, 2, 3, 4, 5, 6, 7, 8]])]


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
@pytest.mark.parametrize("block,dim,heads,group,cached,new,entries", PAST)
def test_attention_past_the_caches(ext, dtype, block, dim, heads, group, cached, new, entries):
    """Tables so wide that codes are read past the caches (as long as their bound says 512 MB and more, or 128 MB a sequence; heads of 64:
    128 MB together): the formula, and the bits of a table one entry narrower, whose codes are read through them."""
    limit = 128e6 if dim == 64 else min(128e6 * len(cached), 512e6)
    width = int(limit // (2 * len(cached) * block * heads * dim)) + 1
    table = torch.full((len(cached), width), -1, dtype=torch.int32)
    for b, row in enumerate(entries):
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    got, args = check_attention(ext, dtype, block, dim, heads, group, cached, new, table=table)
    assert torch.equal(got, ext.kv_block_attention(*args[:5], args[5][:, :-1], *args[6:]))


def test_a_captured_step_past_the_caches(ext):
    """A graph of append and attention under a table of a long max_len, replayed with eager work in between: the eager step's bits."""
    from llmquant.runtime import BlockQuantCache

    eager, graphed = (fresh(BlockQuantCache, max_len=400000, block=128, num_blocks=30, kv_heads=2) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(8)
    static = torch.zeros(3, 8 * 64, device="cuda", dtype=torch.bfloat16)

    def step(cache, rows):
        outs = []
        for layer in range(2):
            cache.append(layer, rows[:, 256:384].unflatten(1, (2, 64)), rows[:, 384:].unflatten(1, (2, 64)))
            outs.append(cache.attend(layer, rows[:, :256].unflatten(1, (4, 64)), 0.125))
        cache.advance_device(1)
        return outs

    start = torch.tensor([0, 1500, 1500, 1600], dtype=torch.int32, device="cuda")
    prompt = torch.randn(1600, 2, 64, generator=g, device="cuda", dtype=torch.bfloat16)
    for cache in (eager, graphed):
        cache.add(), cache.add(), cache.add(), cache.release(1)
        cache.reserve([1600, 0, 200])
        for layer in range(2):
            cache.append(layer, prompt, prompt, start)
        cache.advance([1500, 0, 100])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # (a warm-up, taken back)
        step(graphed, static)
    torch.cuda.current_stream().wait_stream(side)
    for place in (0, 2):
        graphed.truncate(place, graphed.get_seq_length(place))
    for a, b in zip((eager.k_codes, eager.v_codes, eager.k_scale, eager.v_scale), (graphed.k_codes, graphed.v_codes, graphed.k_scale, graphed.v_scale)):
        b.copy_(a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(graphed, static)
    for turn in range(12):
        rows = torch.randn(3, 8 * 64, generator=g, device="cuda", dtype=torch.bfloat16)
        want = step(eager, rows)
        static.copy_(rows)
        graph.replay()
        if turn % 3 == 0:
            torch.cuda.synchronize()
        for a, b in zip(want, captured):
            assert torch.equal(a, b) and torch.all(a[1] == 0) and a[0].abs().sum() > 0
    for a, b in ((eager.k_codes, graphed.k_codes), (eager.v_codes, graphed.v_codes), (eager.cached, graphed.cached)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=TAGS.get)
def test_out_may_not_share_memory_with_rows_that_stand_apart(ext, dtype):
    """Queries as slices of q|k|v rows: refused where out has a byte of one, of the scales or of the batch's vectors; taken between and behind them."""
    g = torch.Generator().manual_seed(41)
    cache = [t.cuda() for t in make_cache(g, 2, 2, 16, 64)]
    table, cached = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.tensor([3, 9, 15], dtype=torch.int32, device="cuda")
    heads, wide, tokens, row = 2, 2048, 3, 128
    room = torch.randn(6, wide, generator=g).to(dtype).cuda()
    query = room[:tokens, 512:512 + row].unflatten(1, (heads, 64))
    want, flat, size = ext.kv_block_attention(query, *cache, table, cached, 1.0), room.view(-1), tokens * row

    def attend(at):
        return ext.kv_block_attention(query, *cache, table, cached, 1.0, None, flat[at:at + size].view(tokens, row))

    # rows 0, 1 and 2: from the start, the last packet, the first one
    for at in (512, 512 + row - 8, 512 - size + 8, wide + 512 + row - 8, wide + 512 - size + 8, 2 * wide + 512 - size + 8, 2 * wide + 512 + row - 8):
        with pytest.raises(RuntimeError, match="out must not share memory"):
            attend(at)
    for at in (0, 512 - size, 512 + row, wide + 512 - size, wide + 512 + row, 2 * wide + 512 - size, 2 * wide + 512 + row, 3 * wide):
        kept = room.clone()
        assert torch.equal(attend(at), want)
        room.copy_(kept)
    # the codes, the scales, a table whose rows stand apart and the vectors
    out = torch.zeros(tokens, row, device="cuda")
    q, words, inside = query.float(), out.view(-1).view(torch.int32), out.view(-1)[8:12].view(2, 2)
    apart = words.as_strided((tokens, 1), (row, 1), 3)
    for args in ((q, *cache[:2], inside, cache[3], table, cached, 1.0, None), (q, *cache[:3], inside, table, cached, 1.0, None),
                 (q, *cache, apart, cached, 1.0, None), (q, *cache, table, words[9:12], 1.0, None), (q, *cache, table, cached, 1.0, words[9:13])):
        with pytest.raises(RuntimeError, match="out must not share memory"):
            ext.kv_block_attention(*args, out)
    for codes in cache[:2]:
        with pytest.raises(RuntimeError, match="out must not share memory"):
            ext.kv_block_attention(q, *cache, table, cached, 1.0, None, codes.view(-1)[:4 * size].view(torch.float32).view(tokens, row))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=TAGS.get)
def test_attention_of_value_scales_far_apart(ext, dtype):
    """Blocks of the least value scale beside one of 2^50: the least one's tokens count in the softmax's sum."""
    def far(q, cache, table):
        q[:] *= 0.1                            # (scores near each other)
        cache[3][:] = 1e-8
        cache[3][table[0, 1]] = 2.0 ** 50
        cache[3][table[1, 0]] = 2.0 ** 50

    check_attention(ext, dtype, 16, 64, 1, 4, [90, 40], None, adjust=far)
    check_attention(ext, dtype, 16, 64, 1, 2, [1500, 1100], [1, 3], adjust=far)
    check_attention(ext, dtype, 16, 128, 1, 4, [60, 20], [40, 33], adjust=far)
