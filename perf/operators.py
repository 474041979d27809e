"""Serving a batch of sequences from an 8-bit key/value cache in blocks, as cases that can be timed: the norm and the
rotation of queries and keys (`qk_norm_rope`), quantizing new tokens into the cache (`kv_block_append`), reading it back
(`kv_block_dequant`) and attention over it (`kv_block_attention`), each as a plain form in elementary tensor
operations and as the package's call.

The cache of a layer: a block holds `block` consecutive tokens of one sequence; `k_codes` [blocks, kv_heads, block, dim]
and `v_codes` [blocks, kv_heads, block / 16, dim, 16] (16 tokens innermost) int8, `k_scale` and `v_scale`
[blocks, kv_heads] float32, one scale for a block and head. `block_table` [sequences, width] int32 names a sequence's
blocks in order, `cached` [sequences] int32 how many of its tokens lie in the cache before the call (-1: the sequence
takes no part), and the call's own tokens are rows query_start[b] .. query_start[b + 1] - 1 (without it: one row each).
"""

from __future__ import annotations

import functools
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
SCALE_FLOOR = 1e-8   # the smallest scale of the package's quantizers

#: query and key/value heads: those of the models that the benchmark and the tests use, and other group sizes
HEADS = [(32, 8), (32, 8), (16, 16), (28, 4), (8, 1), (12, 4), (64, 8)]

#: no drawn case does more than the largest listed ones
MOST_FLOPS, MOST_BYTES, MOST_SCORES = 2.4e11, 4.0e8, 6.0e8


def listed():
    return [
        # queries and keys of one token: what every layer of a single chat calls
        dict(name="norm_1", kind="norm", tokens=1, q_heads=32, kv_heads=8, dim=128, rotary=128, far=32768, dtype="bf16",
             table="same"),
        # a batch in fp16, its sequences at far positions, half of each head rotated by a table in 32 bits
        dict(name="norm_77_half", kind="norm", tokens=77, q_heads=28, kv_heads=4, dim=128, rotary=64, far=131072,
             dtype="f16", table="f32"),
        # a long prompt
        dict(name="norm_4100", kind="norm", tokens=4100, q_heads=32, kv_heads=8, dim=128, rotary=128, far=8192,
             dtype="bf16", table="f32"),
        # one token for each of a batch of chats, written into their last blocks, and those blocks read back
        dict(name="write_step_64", kind="write", seqs=64, new=64, cached=60000, kv_heads=8, dim=128, block=64,
             dtype="bf16", absent=0),
        # prompts of several users in one call, two of them with something cached already
        dict(name="write_prompts", kind="write", seqs=7, new=6011, cached=900, kv_heads=8, dim=64, block=16,
             dtype="f16", absent=0),
        # the cached part of one chat, as a prompt's next chunk reads it
        dict(name="read_600", kind="read", seqs=1, cached=600, kv_heads=8, dim=64, block=64, dtype="bf16"),
        # a batch of ragged documents, ahead of an attention that wants plain keys and values
        dict(name="read_40000", kind="read", seqs=24, cached=40000, kv_heads=8, dim=128, block=32, dtype="bf16"),
        # the next token of one chat at an ordinary length
        dict(name="attend_1_600", kind="attend", seqs=1, new=1, cached=600, q_heads=32, kv_heads=8, dim=64, block=64,
             dtype="bf16", absent=0),
        # the next token after a long document
        dict(name="attend_1_131000", kind="attend", seqs=1, new=1, cached=131000, q_heads=32, kv_heads=8, dim=128,
             block=128, dtype="bf16", absent=0),
        # a ragged batch of chats at their next token: what a serving loop calls most
        dict(name="attend_48", kind="attend", seqs=48, new=48, cached=150001, q_heads=32, kv_heads=8, dim=128, block=64,
             dtype="bf16", absent=0),
        # a batch in fp16 with drafted tokens to verify, four or five rows each, in small blocks
        dict(name="attend_drafts", kind="attend", seqs=16, new=73, cached=30000, q_heads=28, kv_heads=4, dim=128,
             block=16, dtype="f16", absent=1),
        # the second chunk of a long prompt
        dict(name="attend_chunk", kind="attend", seqs=1, new=2000, cached=6000, q_heads=32, kv_heads=8, dim=128,
             block=64, dtype="bf16", absent=0),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    while True:
        kind = rng.choice(["norm", "write", "read", "attend", "attend", "attend"])
        q_heads, kv_heads = rng.choice(HEADS)
        case = dict(kind=kind, kv_heads=kv_heads, dim=rng.choice([64, 64, 128, 128, 128, 256]),
                    dtype=rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"]))
        if kind == "norm":
            rotary = case["dim"] // rng.choice([1, 1, 1, 2])
            case |= dict(tokens=_spread(rng, 1, 8192), q_heads=q_heads, rotary=rotary, far=rng.choice([4096, 32768, 131072]),
                         table=rng.choice(["same", "f32"]))
        else:
            case |= dict(block=rng.choice([16, 32, 64, 64, 128]), seqs=_spread(rng, 1, 96))
        if kind == "write":
            step = rng.random() < 0.5
            case |= dict(new=case["seqs"] if step else _spread(rng, case["seqs"], 8192),
                         cached=_spread(rng, 1, 1000 * case["seqs"]), absent=rng.choice([0, 0, 1]) if case["seqs"] > 1 else 0)
        elif kind == "read":
            case |= dict(cached=_spread(rng, 16, 100000))
        elif kind == "attend":
            form = rng.choice(["step", "step", "drafts", "prompt"])
            new = {"step": case["seqs"], "drafts": case["seqs"] * rng.randint(2, 9) + rng.randint(0, case["seqs"] - 1),
                   "prompt": _spread(rng, case["seqs"], 2048)}[form]
            case |= dict(q_heads=q_heads, new=new, cached=_spread(rng, 1, 150000), absent=rng.choice([0, 0, 1]) if case["seqs"] > 1 else 0)
        need = work(case)
        if need["flops"] <= MOST_FLOPS and need["bytes"] <= MOST_BYTES and _padded(case) <= MOST_SCORES:
            return case


# ---- sizes of the sequences, from the case alone ------------------------------------------------------------------
def _ragged(total, parts, salt):
    """`total` in `parts` unequal whole numbers."""
    rng = random.Random("%s %d %d" % (salt, total, parts))
    weights = [rng.uniform(0.2, 1.8) for _ in range(parts)]
    got = [int(total * w / sum(weights)) for w in weights]
    for i in range(total - sum(got)):
        got[i % parts] += 1
    return got


def _lengths(case):
    """(cached tokens, new rows) of every sequence; the last `absent` ones take no part, though they have rows."""
    seqs, absent = case["seqs"], case.get("absent", 0)
    cached = _ragged(case["cached"], seqs, "cached")
    if case["kind"] == "read":
        return cached, [0] * seqs
    new = [1 + n for n in _ragged(case["new"] - seqs, seqs, "new")]   # (a row at least, so that new == seqs is a step)
    if case["kind"] == "write" and case["new"] > 8 * seqs:   # prompts: most of them begin at nothing
        cached = [c if b % 3 == 1 or seqs == 1 else 0 for b, c in enumerate(cached)]
    for b in range(seqs - absent, seqs):
        cached[b] = -1
    return cached, new


def _padded(case):
    """Scores of the plain form, whose sequences are padded to the longest."""
    if case["kind"] != "attend":
        return 0
    cached, new = _lengths(case)
    return len(new) * max(new) * case["q_heads"] * max(c + n for c, n in zip(cached, new))


def work(case):
    size, dim, kind = SIZES[case["dtype"]], case["dim"], case["kind"]
    if kind == "norm":
        vectors = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        table = 4 if case["table"] == "f32" else size
        return {"bytes": 2 * vectors * dim * size + 2 * case["tokens"] * case["rotary"] * table + 2 * dim * size,
                "flops": 8.0 * vectors * dim}
    cached, new = _lengths(case)
    part = [(c, n) for c, n in zip(cached, new) if c >= 0]
    row = 2 * case["kv_heads"] * dim   # elements of a token, keys and values
    if kind == "read":
        tokens = sum(cached)
        blocks = sum(-(-c // case["block"]) for c in cached)
        return {"bytes": tokens * row * (1 + size) + 8 * blocks * case["kv_heads"], "flops": tokens * row}
    if kind == "write":   # new rows read, their codes written; the touched blocks' tokens read as codes and written as values
        back = sum(c % case["block"] + n for c, n in part)
        return {"bytes": sum(n for _, n in part) * row * (size + 1) + back * row * (1 + size), "flops": 4.0 * back * row}
    seen = sum(n * c + n * (n + 1) // 2 for c, n in part)   # pairs of a query and a key
    blocks = sum(-(-(c + n) // case["block"]) for c, n in part)
    return {"bytes": sum(c + n for c, n in part) * row + 8 * blocks * case["kv_heads"]
            + 2 * sum(new) * case["q_heads"] * dim * size,
            "flops": 4.0 * dim * case["q_heads"] * seen}


# ---- what a user's program has in hand before the call ------------------------------------------------------------
def _normal(generator, *shape):
    return torch.randn(*shape, generator=generator, device="cuda")


def _cache(case, seed, generator):
    """A cache that holds the sequences, their blocks in any order."""
    cached, new = _lengths(case)
    block, heads, dim = case["block"], case["kv_heads"], case["dim"]
    counts = [-(-(max(c, 0) + n) // block) for c, n in zip(cached, new)]
    blocks, width = sum(counts) + 2, max(counts)
    order = list(range(blocks))
    random.Random(seed).shuffle(order)
    table = torch.full((len(counts), width), -1, dtype=torch.int32)
    at = 0
    for b, count in enumerate(counts):
        table[b, :count] = torch.tensor(order[at:at + count], dtype=torch.int32)
        at += count
    # codes as a normal distribution leaves them; scales that differ from block to block and head to head
    def codes(*shape):
        part = torch.randint(-128, 128, shape, generator=generator, device="cuda", dtype=torch.int8)
        return part // 2 + torch.randint(-63, 64, shape, generator=generator, device="cuda", dtype=torch.int8)

    def scales():
        return torch.exp(0.4 * _normal(generator, blocks, heads)) / 45

    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(kind=case["kind"], block=block, dim=dim, kv_heads=heads, dtype=DTYPES[case["dtype"]],
                k_codes=codes(blocks, heads, block, dim), v_codes=codes(blocks, heads, block // 16, dim, 16),
                k_scale=scales(), v_scale=scales(), block_table=table.cuda(),
                cached=torch.tensor(cached, dtype=torch.int32, device="cuda"),
                query_start=None if all(n == 1 for n in new) else torch.tensor(starts, dtype=torch.int32, device="cuda"),
                rows=sum(new), most_new=max(new), longest=max(max(c, 0) + n for c, n in zip(cached, new)))


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype, dim = DTYPES[case["dtype"]], case["dim"]
    if case["kind"] == "norm":
        tokens, q_heads, kv_heads, rotary = case["tokens"], case["q_heads"], case["kv_heads"], case["rotary"]
        # queries and keys as a projection leaves them, side by side in a row
        rows = (3.0 * _normal(generator, tokens, (q_heads + kv_heads) * dim)).to(dtype)
        positions = torch.randint(0, case["far"], (tokens,), generator=generator, device="cuda", dtype=torch.int32)
        frequency = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
        angle = torch.arange(case["far"], dtype=torch.float64, device="cuda")[:, None] * frequency
        angle = torch.cat([angle, angle], -1)
        table = torch.float32 if case["table"] == "f32" else dtype
        return dict(kind="norm", q=rows[:, :q_heads * dim], k=rows[:, q_heads * dim:], dim=dim,
                    q_weight=(1 + 0.3 * _normal(generator, dim)).to(dtype), k_weight=(1 + 0.3 * _normal(generator, dim)).to(dtype),
                    cos=angle.cos().to(table), sin=angle.sin().to(table), positions=positions)
    state = _cache(case, seed, generator)
    if case["kind"] == "write":
        heads = case["kv_heads"]
        rows = _normal(generator, state["rows"], 2 * heads * dim).to(dtype)   # keys and values side by side
        state["key"] = rows[:, :heads * dim].unflatten(1, (heads, dim))
        state["value"] = rows[:, heads * dim:].unflatten(1, (heads, dim))
        # the touched blocks, read back from their first token on
        cached, new = _lengths(case)
        first = [c - c % case["block"] if c >= 0 else 0 for c in cached]
        read = [c + n - f if c >= 0 else 0 for c, n, f in zip(cached, new, first)]
    elif case["kind"] == "read":
        first, read = None, _lengths(case)[0]
    else:
        state["query"] = (1.5 * _normal(generator, state["rows"], case["q_heads"], dim)).to(dtype)
        state["sm_scale"] = dim ** -0.5
        return state
    state["first"] = None if first is None else torch.tensor(first, dtype=torch.int32, device="cuda")
    state["starts"] = torch.tensor([sum(read[:b]) for b in range(len(read) + 1)], dtype=torch.int32, device="cuda")
    state["n_tokens"], state["most_read"] = sum(read), max(read)
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _calls(state)
    return {"norm": _plain_norm, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}[state["kind"]](state)


@functools.lru_cache(maxsize=1)
def _ext():
    package = os.path.join(os.getcwd(), "llm-quant_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from llmquant.hip import load_extension

    return load_extension()


def _calls(s):
    ext = _ext()
    if s["kind"] == "norm":
        return ext.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], EPS, s["positions"])
    cache = (s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], s["block_table"])
    if s["kind"] == "attend":
        return ext.kv_block_attention(s["query"], *cache, s["cached"], s["sm_scale"], s["query_start"])
    if s["kind"] == "write":
        ext.kv_block_append(s["key"], s["value"], *cache, s["cached"], s["query_start"])
    k, v = ext.kv_block_dequant(*cache, s["starts"], s["n_tokens"], s["dtype"], s["first"])
    return (k, v) if s["kind"] == "read" else (k, v, s["k_scale"], s["v_scale"])


def _plain_norm(s):
    position = s["positions"].long()
    cos, sin = s["cos"][position].float()[:, None], s["sin"][position].float()[:, None]
    rotary = cos.shape[-1]

    def one(x, weight):
        wide = x.unflatten(1, (-1, s["dim"])).float()
        wide = wide * torch.rsqrt(wide.square().mean(-1, keepdim=True) + EPS) * weight.float()
        turned, rest = wide[..., :rotary], wide[..., rotary:]
        half = torch.cat([-turned[..., rotary // 2:], turned[..., :rotary // 2]], -1)
        return torch.cat([turned * cos + half * sin, rest], -1).to(x.dtype)

    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


def _starts(s):
    if s["query_start"] is not None:
        return s["query_start"].long()
    return torch.arange(s["cached"].numel() + 1, device="cuda")


def _tokens_innermost(codes):
    """Value codes [.., block / 16, dim, 16] as [.., block, dim], and back."""
    return codes.transpose(-1, -2).flatten(-3, -2)


def _strips(codes):
    return codes.unflatten(-2, (-1, 16)).transpose(-1, -2)


def _plain_write(s):
    block, starts, cached = s["block"], _starts(s), s["cached"].long()
    part = cached >= 0
    count = torch.where(part, starts[1:] - starts[:-1], 0)
    first_block = torch.where(part, cached, 0) // block
    last_block = torch.where(count > 0, (cached + count - 1) // block, first_block)
    touched = (s["most_new"] - 1) // block + 2
    # block j of those a sequence touches (beyond its last one: the last one again); sequences that take no part
    # repeat a block of nobody's, which is left as it is
    logical = torch.minimum(first_block[:, None] + torch.arange(touched, device="cuda"), last_block[:, None])
    physical = s["block_table"].long().gather(1, logical).clamp_min(0)
    position = logical[..., None] * block + torch.arange(block, device="cuda")   # [sequences, touched, block]
    is_new = part[:, None, None] & (position >= cached[:, None, None]) & (position < (cached + count)[:, None, None])
    row = torch.where(is_new, starts[:-1, None, None] + position - cached[:, None, None], 0)
    fresh = (logical * block >= cached[:, None]) & (count > 0)[:, None]
    old = part[:, None, None] & (position < cached[:, None, None])
    write = (part & (count > 0))[:, None].expand_as(physical)
    for new, codes, scale, values in ((s["key"], s["k_codes"], s["k_scale"], False), (s["value"], s["v_codes"], s["v_scale"], True)):
        tokens = new.float()[row].transpose(2, 3)                    # [sequences, touched, heads, block, dim]
        tokens = torch.where(is_new[:, :, None, :, None], tokens, 0)
        largest = (tokens.abs().amax((-1, -2)) / 127.0).clamp_min(SCALE_FLOOR)
        before = scale[physical]
        after = torch.where(fresh[..., None], largest, torch.maximum(before, largest))
        held = _tokens_innermost(codes[physical]) if values else codes[physical]
        moved = ((held.float() * before[..., None, None]) / after[..., None, None]).round().clamp(-128, 127)
        moved = torch.where(old[:, :, None, :, None], moved, held.float())
        fresh_codes = (tokens / after[..., None, None]).round().clamp(-128, 127)
        got = torch.where(is_new[:, :, None, :, None], fresh_codes, moved).to(torch.int8)
        got = torch.where(write[..., None, None, None], got, held)
        codes[physical] = _strips(got) if values else got
        scale[physical] = torch.where(write[..., None], after, before)
    return (*_plain_read(s), s["k_scale"], s["v_scale"])


def _plain_read(s):
    starts, block = s["starts"].long(), s["block"]
    token = torch.arange(s["n_tokens"], device="cuda")
    sequence = torch.searchsorted(starts, token, right=True) - 1
    position = token - starts[sequence] + (0 if s["first"] is None else s["first"].long()[sequence])
    physical, slot = s["block_table"].long()[sequence, position // block], position % block
    keys = s["k_codes"][physical, :, slot].float() * s["k_scale"][physical][..., None]
    values = s["v_codes"][physical, :, slot // 16, :, slot % 16].float() * s["v_scale"][physical][..., None]
    return keys.transpose(0, 1).to(s["dtype"]).contiguous(), values.transpose(0, 1).to(s["dtype"]).contiguous()


def _plain_attend(s):
    query, starts, cached, heads, dim = s["query"], _starts(s), s["cached"].long(), s["kv_heads"], s["dim"]
    rows, q_heads = query.shape[:2]
    group = q_heads // heads
    count = starts[1:] - starts[:-1]
    table = s["block_table"].long().clamp_min(0)
    keys = (s["k_codes"][table].float() * s["k_scale"][table][..., None, None]).transpose(1, 2).flatten(2, 3)
    values = (_tokens_innermost(s["v_codes"][table]).float() * s["v_scale"][table][..., None, None]).transpose(1, 2).flatten(2, 3)
    keys, values = keys[:, :, :s["longest"]], values[:, :, :s["longest"]]          # [sequences, heads, longest, dim]
    place = torch.arange(s["most_new"], device="cuda")
    row = (starts[:-1, None] + place).clamp_max(rows - 1)
    wide = query.float()[row].unflatten(2, (heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = torch.matmul(wide, keys.transpose(2, 3).contiguous()) * s["sm_scale"]  # [sequences, heads, rows x group, longest]
    limit = torch.where(cached[:, None] >= 0, cached[:, None] + place, -1).repeat_interleave(group, 1)
    hidden = torch.arange(s["longest"], device="cuda") > limit[..., None]
    scores = scores.masked_fill_(hidden[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores.sub_(torch.where(top == -math.inf, 0, top)))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, values) / torch.where(total == 0, 1, total)
    out = out.unflatten(2, (s["most_new"], group)).permute(0, 2, 1, 3, 4).flatten(2, 3)   # [sequences, place, q_heads, dim]
    at = torch.arange(rows, device="cuda")
    sequence = torch.searchsorted(starts, at, right=True) - 1
    return out[sequence, at - starts[sequence]].flatten(1).to(query.dtype)


# ---- the definitions in 64 bits, a sequence and a head at a time --------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(case, s)
    cached, new = _lengths(case)
    if case["kind"] == "write":
        if case["seqs"] > 400:
            return None
        return _exact_write(case, s, cached, new)
    if case["kind"] == "read":
        return _exact_read(s, [range(c) for c in cached])
    return _exact_attend(case, s, cached, new)


def _exact_norm(case, s):
    angle = s["positions"].long()
    cos, sin = s["cos"].double()[angle], s["sin"].double()[angle]
    half = case["rotary"] // 2
    results = []
    for x, weight, heads in ((s["q"], s["q_weight"], case["q_heads"]), (s["k"], s["k_weight"], case["kv_heads"])):
        x = x.double().reshape(case["tokens"], heads, case["dim"])
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS) * weight.double()
        y = x.clone()
        for low in range(half):
            a, b = x[..., low], x[..., low + half]
            y[..., low] = a * cos[:, None, low] - b * sin[:, None, low]
            y[..., low + half] = b * cos[:, None, low + half] + a * sin[:, None, low + half]
        results.append(y)
    return tuple(results)


def _sequence(codes, scale, ids, values):
    """The blocks `ids` of one sequence as numbers, [heads, tokens, dim] in 64 bits."""
    part = codes[ids].double()
    if values:
        part = part.permute(0, 1, 2, 4, 3).reshape(part.shape[0], part.shape[1], -1, part.shape[3])
    part = part * scale[ids].double()[:, :, None, None]
    return part.permute(1, 0, 2, 3).reshape(part.shape[1], -1, part.shape[3])


def _exact_read(s, tokens):
    results = []
    for codes, scale, values in ((s["k_codes"], s["k_scale"], False), (s["v_codes"], s["v_scale"], True)):
        parts = []
        for b, span in enumerate(tokens):
            if len(span):
                ids = s["block_table"][b, : -(-span[-1] // s["block"]) + 1]
                parts.append(_sequence(codes, scale, ids[ids >= 0].long(), values)[:, span[0]:span[-1] + 1])
        results.append(torch.cat(parts, 1))
    return tuple(results)


def _exact_write(case, s, cached, new):
    block, heads, dim = case["block"], case["kv_heads"], case["dim"]
    results, scales = [], []
    for new_rows, codes, scale, values in ((s["key"], s["k_codes"], s["k_scale"], False), (s["value"], s["v_codes"], s["v_scale"], True)):
        scale, parts, row = scale.double(), [], 0
        for b, (c, n) in enumerate(zip(cached, new)):
            if c < 0:
                row += n
                continue
            low = c // block
            ids = s["block_table"][b, low:(c + n - 1) // block + 1].long()
            ones = torch.ones_like(scale)
            held = _sequence(codes, ones, ids, values).reshape(heads, len(ids), block, dim)[:, 0, :c - low * block]
            wide = torch.zeros(heads, len(ids) * block, dim, dtype=torch.float64, device="cuda")
            wide[:, c - low * block:c - low * block + n] = new_rows[row:row + n].double().transpose(0, 1)
            row += n
            wide = wide.reshape(heads, len(ids), block, dim)
            after = (wide.abs().flatten(2).max(-1).values / 127).clamp(min=SCALE_FLOOR)   # [heads, blocks]
            before = scale[ids[0]].clone()
            if c % block:
                after[:, 0] = torch.maximum(after[:, 0], before)
            got = torch.round(wide / after[..., None, None]).clamp(-128, 127)
            got[:, 0, :c - low * block] = torch.round(held * (before / after[:, 0])[:, None, None]).clamp(-128, 127)
            scale[ids] = after.transpose(0, 1)
            parts.append((got * after[..., None, None]).reshape(heads, -1, dim)[:, :c - low * block + n])
        results.append(torch.cat(parts, 1))
        scales.append(scale)
    return (*results, *scales)


def _exact_attend(case, s, cached, new):
    if work(case)["flops"] > 1e13:
        return None
    heads, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        if c >= 0:
            ids = s["block_table"][b, : -(-(c + n) // case["block"])].long()
            keys = _sequence(s["k_codes"], s["k_scale"], ids, False)[:, :c + n]
            values = _sequence(s["v_codes"], s["v_scale"], ids, True)[:, :c + n]
            above = torch.ones(n, c + n, dtype=torch.bool, device="cuda").triu(c + 1)
            for h in range(heads * group):
                scores = s["query"][row:row + n, h].double() @ keys[h // group].T * s["sm_scale"]
                scores[above] = -math.inf
                out[row:row + n, h] = torch.softmax(scores, -1) @ values[h // group]
        row += n
    return out.flatten(1)
