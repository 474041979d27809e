"""The quantized KV cache as real integers in HBM.

FakeQuantCache (llmquant/quantizers/fake.py:39-55) quantizes K and V on write and then stores
the dequantized bf16 values; the accounting the reference reports for it (17 KB per cached
token at int8 instead of 32 KB) is for a cache that keeps the codes. This is that cache:
static-shaped per layer ([kv_heads, t_max, head_dim] codes + [kv_heads, t_max] fp32 scales),
written by the append kernel at a position that lives on the device and read back inside the
decode-attention kernel. Nothing about it changes shape or address from step to step, so a
decode step that uses it can be captured in a HIP graph -- which the reference's
quantized cache cannot (llmquant/runtime/graph_decode.py:40-43).

BlockQuantCache is the same for a batch of sequences, whose tokens lie in blocks (no counterpart in the reference, which
runs one sequence at a time).
"""

from __future__ import annotations

import warnings

import torch

from llmquant.hip.build import load_extension


class KernelQuantCache:
    """K/V codes and scales for every layer of one sequence (batch 1).

    num_bits   8 (int8 codes) or 4 (nibble-packed); 16: an unquantized cache of `dtype` values (the 16-bit
               baseline run through the same decode step; only the fused step's attention launch reads it)
    position   device int32 [1]: where the next token is written
    length     device int32 [1]: tokens valid for attention (position + tokens being added)
    """

    def __init__(self, num_layers: int, kv_heads: int, head_dim: int, max_len: int, num_bits: int = 8,
                 q_heads: int | None = None, device="cuda", dtype=torch.bfloat16):
        if num_bits not in (4, 8, 16):
            raise ValueError(f"KV cache bits must be 4 or 8 (or 16 for an unquantized cache), got {num_bits}")
        if num_bits == 16 and dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("an unquantized cache holds bfloat16 or float16 values")
        self.num_bits, self.num_layers = num_bits, num_layers
        self.kv_heads, self.head_dim, self.max_len = kv_heads, head_dim, max_len
        self._ext = load_extension()
        width = head_dim // 2 if num_bits == 4 else head_dim
        code_dtype = {8: torch.int8, 4: torch.uint8, 16: dtype}[num_bits]
        shape = (num_layers, kv_heads, max_len, width)
        self.k_codes = torch.zeros(shape, dtype=code_dtype, device=device)
        self.v_codes = torch.zeros(shape, dtype=code_dtype, device=device)
        fill = torch.ones if num_bits == 16 else torch.zeros
        self.k_scale = fill(num_layers, kv_heads, max_len, dtype=torch.float32, device=device)
        self.v_scale = fill(num_layers, kv_heads, max_len, dtype=torch.float32, device=device)
        self.position = torch.zeros(1, dtype=torch.int32, device=device)
        self.length = torch.zeros(1, dtype=torch.int32, device=device)
        q_heads = q_heads or kv_heads
        # one workspace per layer: launches that share one must not overlap, and layers of a
        # captured step could in principle be reordered onto other streams by a caller
        floats = self._ext.kv_decode_workspace_floats(q_heads, head_dim, max_len)
        self.workspace = torch.zeros(num_layers, floats, dtype=torch.float32, device=device)
        self._host_length = 0  # mirror for prefill bookkeeping only; decode never reads it

    # ---- bookkeeping ------------------------------------------------------------------------------
    def get_seq_length(self) -> int:
        return self._host_length

    def set_position(self, position: int) -> None:
        """Next write position (host call; inside a graph the tensors are advanced instead)."""
        self.set_counters(position, position)

    def set_counters(self, position: int, length: int) -> None:
        """Write position and valid length, one launch on the GPU."""
        self._host_length = position
        if self.position.is_cuda:
            self._ext.seed_step(None, None, None, self.position, self.length, position, length, None, None)
        else:
            self.position.fill_(position)
            self.length.fill_(length)

    def advance(self, tokens: int = 1) -> None:
        """Move the write position forward on the device (capturable)."""
        self.position.add_(tokens)
        self._host_length += tokens

    def bytes_per_token(self) -> int:
        """Codes + scales stored per cached token over all layers, K and V."""
        if self.num_bits == 16:
            return 2 * self.num_layers * self.kv_heads * self.head_dim * 2
        width = self.head_dim if self.num_bits == 8 else self.head_dim // 2
        return 2 * self.num_layers * self.kv_heads * (width + 4)

    # ---- per-layer operations ------------------------------------------------------------------------
    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, return_dequantized: bool = False):
        """key / value: [kv_heads, n_new, head_dim] (any strides with a contiguous last axis).
        Writes at position .. position + n_new - 1. With return_dequantized, hands back what
        FakeQuantCache.update would have returned for these tokens."""
        if self.num_bits == 16:
            # the unquantized cache: a copy at the host-side position (prompt passes only; the fused decode step
            # appends inside its attention launch)
            start, stop = self._host_length, self._host_length + key.shape[1]
            self.k_codes[layer][:, start:stop] = key
            self.v_codes[layer][:, start:stop] = value
            return (key.contiguous(), value.contiguous()) if return_dequantized else (None, None)
        return self._ext.kv_append(key, value, self.k_codes[layer], self.v_codes[layer], self.k_scale[layer],
                                   self.v_scale[layer], self.position, return_dequantized)

    def attend(self, layer: int, query: torch.Tensor, scaling: float) -> torch.Tensor:
        """query [q_heads, head_dim] -> [q_heads, head_dim], over tokens 0 .. length - 1."""
        return self._ext.kv_decode_attention(query, self.k_codes[layer], self.v_codes[layer], self.k_scale[layer],
                                             self.v_scale[layer], self.workspace[layer], self.length, scaling)

    def dequantized(self, layer: int, n_tokens: int, dtype=torch.bfloat16):
        """(keys, values) [kv_heads, n_tokens, head_dim] as the fake-quant cache would hold them."""
        k = self._ext.kv_dequant(self.k_codes[layer], self.k_scale[layer], n_tokens, dtype)
        v = self._ext.kv_dequant(self.v_codes[layer], self.v_scale[layer], n_tokens, dtype)
        return k, v


class BlockQuantCache:
    """K/V codes and scales for every layer of a batch of sequences that come and go, in blocks.

    A block holds `block` consecutive tokens of one sequence under one scale per head (8 bytes a block and head, where
    KernelQuantCache keeps 8 a token); sequences take blocks as they grow and give them back when they end, so that memory
    goes by what is cached and not by the longest sequence that might come. The batch has `max_sequences` places. What the
    kernels read of it lies on the device and keeps its address (a step can be captured in a HIP graph):

    block_table  int32 [max_sequences, blocks of max_len]: a place's blocks in order, -1 where there is none
    cached       int32 [max_sequences]: tokens a place holds; -1: nobody is in it, and it takes no part

    The attention's launches go by the table's width, and so by `max_len`, not by what is cached: no more than is needed.

    A step: reserve() the blocks for its tokens, append() and attend() in every layer, advance() (a copy to the device that waits
    for its stream, as reserve() where it takes a block; a captured step has advance_device()). The rows of a call are one
    for each place, or, with `query_start` (int32 [max_sequences + 1]), rows query_start[b] .. query_start[b + 1] - 1 for
    place b: drafted tokens, prompts, a prompt's next chunk, single tokens, mixed as they come.
    """

    def __init__(self, num_layers: int, kv_heads: int, head_dim: int, num_blocks: int, max_sequences: int, max_len: int,
                 block: int = 64, device="cuda"):
        if block not in (16, 32, 64, 128):
            raise ValueError(f"a block holds 16, 32, 64 or 128 tokens, got {block}")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if min(num_layers, kv_heads, num_blocks, max_sequences, max_len) < 1:
            raise ValueError("layers, heads, blocks, sequences and max_len must be positive")
        self.num_layers, self.kv_heads, self.head_dim, self.block = num_layers, kv_heads, head_dim, block
        self.num_blocks, self.max_sequences, self.max_len = num_blocks, max_sequences, max_len
        width = -(-max_len // block)
        self.k_codes = torch.zeros(num_layers, num_blocks, kv_heads, block, head_dim, dtype=torch.int8, device=device)
        self.v_codes = torch.zeros(num_layers, num_blocks, kv_heads, block // 16, head_dim, 16, dtype=torch.int8, device=device)
        self.k_scale = torch.zeros(num_layers, num_blocks, kv_heads, dtype=torch.float32, device=device)
        self.v_scale = torch.zeros(num_layers, num_blocks, kv_heads, dtype=torch.float32, device=device)
        self.block_table = torch.full((max_sequences, width), -1, dtype=torch.int32, device=device)
        self.cached = torch.full((max_sequences,), -1, dtype=torch.int32, device=device)
        self._ext = load_extension() if self.cached.is_cuda else None
        self._free = list(range(num_blocks - 1, -1, -1))
        self._blocks: list[list[int]] = [[] for _ in range(max_sequences)]
        self._lengths = [-1] * max_sequences   # as `cached`, on the host

    # ---- bookkeeping (host calls, outside of a captured step) ------------------------------------------
    def get_seq_length(self, place: int) -> int:
        """Tokens cached for the sequence in a place."""
        self._taken(place)
        return self._lengths[place]

    def free_blocks(self) -> int:
        return len(self._free)

    def add(self) -> int:
        """A place for a new sequence, which holds nothing yet."""
        place = next((i for i, n in enumerate(self._lengths) if n < 0), None)
        if place is None:
            raise RuntimeError(f"all {self.max_sequences} places of the batch are taken")
        self._set_length(place, 0)
        return place

    def release(self, place: int) -> None:
        """The sequence in a place ends; its blocks are free again."""
        self._taken(place)
        self._free.extend(reversed(self._blocks[place]))
        self._blocks[place] = []
        self.block_table[place].fill_(-1)
        self._set_length(place, -1)

    def truncate(self, place: int, length: int) -> None:
        """Take back what was cached behind the first `length` tokens (drafted tokens that were not accepted). Blocks stay
        reserved. A partly kept block keeps the scale and the codes that the tokens taken back left: where one of them was larger than
        all before, the kept ones have that step, and where one was not finite they are lost."""
        self._taken(place)
        if not 0 <= length <= self._lengths[place]:
            raise ValueError(f"place {place} holds {self._lengths[place]} tokens, cannot be cut to {length}")
        self._set_length(place, length)

    def reserve(self, new) -> None:
        """Blocks for `new` more tokens of every sequence: a number, or one for each place (0 for an empty one). Nothing
        changes if there are not enough. A sequence that counts more tokens than its blocks hold is refused: a new block would
        pass for tokens that were never stored."""
        new = self._per_place(new)
        for place, (n, have) in enumerate(zip(self._lengths, self._blocks)):
            if n > len(have) * self.block:
                raise ValueError(f"place {place} counts {n} tokens, its blocks hold {len(have) * self.block}: truncate() it first")
        wanted = [0 if n < 0 else max(0, -(-(n + more) // self.block) - len(have))
                  for n, more, have in zip(self._lengths, new, self._blocks)]
        for place, (n, more) in enumerate(zip(self._lengths, new)):
            if n >= 0 and n + more > self.max_len:
                raise ValueError(f"place {place} would hold {n + more} tokens, at most {self.max_len} fit")
        if sum(wanted) > len(self._free):
            raise RuntimeError(f"{sum(wanted)} more blocks are needed, {len(self._free)} are free")
        at: list[tuple[int, int]] = []
        ids: list[int] = []
        for place, count in enumerate(wanted):
            for _ in range(count):
                at.append((place, len(self._blocks[place])))
                ids.append(self._free.pop())
                self._blocks[place].append(ids[-1])
        if ids:
            rows, columns = (torch.tensor(i, device=self.block_table.device) for i in zip(*at))
            self.block_table[rows, columns] = torch.tensor(ids, dtype=torch.int32, device=self.block_table.device)

    def advance(self, new, device: bool = True) -> None:
        """Count `new` tokens (as for reserve) as cached, behind the last layer of a step. device=False: the host's counts
        alone, for a step whose captured graph has advanced `cached` itself (advance_device). Tokens that no block was reserved
        for are refused, or, where the device has counted them already, warned of: append() has left them out."""
        new = self._per_place(new)
        for place, (n, more, have) in enumerate(zip(self._lengths, new, self._blocks)):
            if n + more <= len(have) * self.block or n < 0:
                continue
            if device:
                raise ValueError(f"place {place} would hold {n + more} tokens, blocks for {len(have) * self.block} are reserved")
            warnings.warn(f"place {place} counts {n + more} tokens, but blocks for {len(have) * self.block} are reserved: those behind "
                          "were not stored (reserve() before the step; truncate() to go on)", RuntimeWarning, stacklevel=2)
        self._lengths = [n if n < 0 else n + more for n, more in zip(self._lengths, new)]
        if device:
            self.cached.copy_(torch.tensor(self._lengths, dtype=torch.int32))

    def advance_device(self, new) -> None:
        """The device's counts alone, by a number or an int32 tensor [max_sequences]; empty places stay (capturable)."""
        torch.where(self.cached >= 0, self.cached + new, self.cached, out=self.cached)

    def bytes_per_token(self) -> float:
        """Codes and scales stored per cached token of full blocks over all layers, K and V."""
        return 2 * self.num_layers * self.kv_heads * (self.head_dim + 4 / self.block)

    def _taken(self, place: int) -> None:
        if not 0 <= place < self.max_sequences or self._lengths[place] < 0:
            raise ValueError(f"nobody is in place {place}")

    def _set_length(self, place: int, length: int) -> None:
        self._lengths[place] = length
        self.cached[place] = length

    def _per_place(self, new) -> list[int]:
        if isinstance(new, int):
            new = [new if n >= 0 else 0 for n in self._lengths]
        new = [int(n) for n in new]
        if len(new) != self.max_sequences or min(new) < 0:
            raise ValueError(f"one number for each of {self.max_sequences} places, none negative, got {new}")
        if any(more and n < 0 for n, more in zip(self._lengths, new)):
            raise ValueError("tokens for a place that nobody is in")
        return new

    # ---- per-layer operations -----------------------------------------------------------------------
    def _layer(self, layer: int):
        return self.k_codes[layer], self.v_codes[layer], self.k_scale[layer], self.v_scale[layer], self.block_table

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, query_start: torch.Tensor | None = None) -> None:
        """key / value: [tokens, kv_heads, head_dim] (rows may be slices of wider ones), written behind what is cached."""
        self._ext.kv_block_append(key, value, *self._layer(layer), self.cached, query_start)

    def attend(self, layer: int, query: torch.Tensor, scaling: float, query_start: torch.Tensor | None = None) -> torch.Tensor:
        """query [tokens, q_heads, head_dim] -> [tokens, q_heads * head_dim], causal, over what is cached and the call's own
        tokens, which append() has written. Rows of empty places are zero."""
        return self._ext.kv_block_attention(query, *self._layer(layer), self.cached, scaling, query_start)

    def dequantized(self, layer: int, place: int, dtype=torch.bfloat16):
        """(keys, values) [kv_heads, tokens, head_dim] of the sequence in a place."""
        tokens = self.get_seq_length(place)
        starts = torch.zeros(self.max_sequences + 1, dtype=torch.int32, device=self.cached.device)
        starts[place + 1:] = tokens
        return self._ext.kv_block_dequant(*self._layer(layer), starts, tokens, dtype)


def make_kernel_cache_factory(num_bits, model, max_len: int):
    """Counterpart of make_cache_factory (llmquant/quantizers/fake.py:58-62) for the kernel
    path: a zero-argument factory of KernelQuantCache sized for `model`, or None for bf16."""
    if num_bits is None:
        return None
    cfg = model.config
    head_dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
    device = next(model.parameters()).device
    return lambda: KernelQuantCache(cfg.num_hidden_layers, cfg.num_key_value_heads, head_dim, max_len, num_bits,
                                    q_heads=cfg.num_attention_heads, device=device)
