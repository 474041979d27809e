"""Low-rank adapters beside kernel-mode Linears: out = codes x + scaling * B (A x), learned on top of frozen codes and
served for many requests at once, each with an adapter of its own or none.

No counterpart in the reference, whose quantized modules are for inference. add_adapters() puts a bank of `slots` adapters
beside every chosen KernelQuantLinear; use_adapters() says which adapter the requests of the next calls have. Requests are
sequences of rows, as the batch of BlockQuantCache has them: a call's rows are one a request, or query_start[b] ..
query_start[b + 1] - 1 of request b.
"""

from __future__ import annotations

import re

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from llmquant.hip.build import load_extension
from llmquant.hip.ops import keep, kept
from llmquant.quantizers.kernel import KernelQuantLinear


_copies: dict[torch.device, torch.cuda.Stream] = {}


def _settled(values: list[int], device: torch.device) -> torch.Tensor:
    """int32 values on the device, there when this returns, so that any stream may read them: a copy on a stream of its own, which alone is waited for. An ordinary
    tensor in inference mode, too: a training step may read it later."""
    with torch.inference_mode(False):
        host = torch.tensor(values, dtype=torch.int32)
        if device.type != "cuda":
            return host.to(device)
        stream = _copies.get(device)
        if stream is None:
            stream = _copies[device] = torch.cuda.Stream(device)
        with torch.cuda.stream(stream):
            return host.to(device)


def _version(tensor: torch.Tensor) -> int | None:
    """How often it was written in place; None: not known."""
    return None if tensor.is_inference() else tensor._version


class AdapterBatch:
    """Which adapter each request has; shared by all banks of a model.

    What the kernels read lies on the device, one tensor for each number of requests, which keeps its address: a captured step
    that ran with n requests reads what select() last said for n. Until then, and after clear(), nobody has an adapter. select() and
    clear() write on the current stream: calls on others come behind them in the way that any other tensor's readers do. A model has one
    batch: threads that call it by turns select and call under a lock of theirs.
    """

    STARTS = 256   # starts of requests of equal length that are kept for the next calls

    def __init__(self, device):
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._adapters: dict[int, torch.Tensor] = {}
        self._starts: dict[tuple[int, int], torch.Tensor] = {}
        self._query_start: torch.Tensor | None = None
        self._selected: tuple[int, int | None] | None = None   # (rows that query_start gave the requests, its version then)
        self._requests = 1
        self._captured: list[torch.Tensor] = []   # what captured steps read
        self._held(1)   # (so that a step captured before anything was selected has it)

    def select(self, adapter, query_start=None) -> None:
        """adapter: a slot for each request (a list, or a tensor on any device; negative: none). query_start: int32 [requests + 1] on the device,
        for calls whose requests have unlike numbers of rows (None: as many rows each). It is kept, not copied: a captured
        step reads the tensor it was captured with, which lives as long as the batch. Calls of fewer rows than it gives the requests are refused
        (a prompt's starts are no step's), unless adapter lies on the device, where nothing is waited for, or the starts were written since."""
        adapter = torch.as_tensor(adapter, dtype=torch.int32).reshape(-1)
        if adapter.numel() == 0:
            raise ValueError("adapters for no request")
        if query_start is not None and (query_start.dtype != torch.int32 or query_start.shape != (adapter.numel() + 1,)
                                        or query_start.device.type != self.device.type):
            raise ValueError(f"query_start must be int32 [{adapter.numel() + 1}] on the model's device")
        selected = None
        if query_start is not None and not adapter.is_cuda and not self._capturing():
            selected = int(query_start[-1]), _version(query_start)
        self._held(adapter.numel()).copy_(adapter)
        self._requests, self._query_start, self._selected = adapter.numel(), query_start, selected

    def clear(self) -> None:
        """Nobody has an adapter, whatever the number of requests."""
        for held in self._adapters.values():
            held.fill_(-1)
        self._requests, self._query_start, self._selected = 1, None, None

    def _capturing(self) -> bool:
        return self.device.type == "cuda" and torch.cuda.is_current_stream_capturing()

    def _held(self, requests: int) -> torch.Tensor:
        held = self._adapters.get(requests)
        if held is None:
            # (made in a capture it would lie in the graph's memory, and every replay would set it to nobody again)
            if self._capturing():
                raise RuntimeError(f"{requests} requests are selected for the first time while a step is captured: select as many before")
            held = self._adapters[requests] = _settled([-1] * requests, self.device)
        return held

    def rows(self, x: torch.Tensor):
        """(adapter, query_start) for a call on x [..., in]."""
        count = x.numel() // x.shape[-1] if x.shape[-1] else 0
        requests, start, selected = self._requests, self._query_start, self._selected
        if selected is not None and count < selected[0] and selected[1] == _version(start):
            raise ValueError(f"{count} rows are fewer than the {selected[0]} of the requests that were selected: select() for this call")
        if start is None and count != requests:
            if count % requests:
                raise ValueError(f"{count} rows are no whole number for each of {requests} requests: select(..., query_start)")
            start = self._starts.get((count, requests))
            if start is None and self._capturing():   # (in the graph's memory)
                return self._held(requests), torch.arange(requests + 1, dtype=torch.int32, device=self.device) * (count // requests)
            if start is None:
                if len(self._starts) >= self.STARTS:   # nobody reads them any more, but for captured steps
                    if self.device.type == "cuda":
                        torch.cuda.synchronize(self.device)
                    self._starts = {k: t for k, t in self._starts.items() if any(t is c for c in self._captured)}
                start = self._starts[count, requests] = _settled([b * (count // requests) for b in range(requests + 1)], self.device)
        if start is not None and self._capturing() and not any(t is start for t in self._captured):
            self._captured.append(start)
        return self._held(requests), start

    # (a copy of the model has a batch of its own; captured steps do not come along)
    def __deepcopy__(self, memo):
        new = AdapterBatch(self.device)
        new._adapters = {n: t.clone() for n, t in self._adapters.items()}
        new._query_start = None if self._query_start is None else self._query_start.clone()
        if self._selected is not None and self._selected[1] == _version(self._query_start):
            new._selected = self._selected[0], _version(new._query_start)
        new._requests = self._requests
        memo[id(self)] = new
        return new


class _LoraAdd(torch.autograd.Function):
    """base + scaling * (x A^T) B^T. Kept for the backward pass: x (or its 8-bit codes, a scale for 128 of them) and the
    rank's numbers of each row."""

    @staticmethod
    def forward(ctx, x, base, lora_a, lora_b, scaling, adapter, query_start, save_bits):
        ext = load_extension()
        low = torch.empty(x.shape[0], lora_a.shape[1], dtype=torch.float32, device=x.device)
        out = ext.lora_add(x, base, lora_a, lora_b, scaling, adapter, query_start, low=low)
        held, scale = (x, None) if save_bits == 16 else ext.quant_group_codes(x, 8, 128, False)
        # (the rows' adapters as they are now: select() writes the batch's in place)
        keep(ctx, held, scale, low, lora_a, lora_b, scaling, adapter.clone(), query_start)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, scale, low, lora_a, lora_b, scaling, adapter, query_start = kept(ctx)
        of_x, of_a, of_b = load_extension().lora_grad(grad, x, low, lora_a, lora_b, scaling, adapter, query_start, x_scale=scale)
        return of_x, grad, of_a, of_b, None, None, None, None


class LoraAdapters(nn.Module):
    """The bank of one Linear: lora_a [slots, rank, in], lora_b [slots, out, rank], scaling float32 [slots]. A learns from a random
    start and B from zeros, so that a new adapter changes nothing. save_bits 8 keeps the activation in 8 bits between the
    passes (a scale for 128 values, as the package's activation quantizer writes them); the result does not depend on it, the
    gradient of lora_a does."""

    def __init__(self, in_features: int, out_features: int, rank: int, slots: int, alpha: float, dtype, device, batch: AdapterBatch,
                 save_bits: int = 16):
        super().__init__()
        if rank % 8 or not 8 <= rank <= 128:
            raise ValueError(f"rank must be a multiple of 8 from 8 to 128, got {rank}")
        if in_features % 8 or out_features % 8:
            raise ValueError(f"adapters take Linears of multiples of 8, got {in_features} x {out_features}")
        if save_bits not in (8, 16) or (save_bits == 8 and in_features % 128):
            raise ValueError(f"save_bits must be 16, or 8 for rows of whole groups of 128, got {save_bits} for {in_features}")
        if not 1 <= slots <= 1024:
            raise ValueError(f"a bank has 1 to 1024 slots, got {slots}")
        self.save_bits, self.batch = save_bits, batch
        self.lora_a = nn.Parameter(torch.randn(slots, rank, in_features, device=device).mul_(in_features ** -0.5).to(dtype))
        self.lora_b = nn.Parameter(torch.zeros(slots, out_features, rank, dtype=dtype, device=device))
        self.register_buffer("scaling", torch.full((slots,), alpha / rank, dtype=torch.float32, device=device))

    def forward(self, x, base):
        """base, the Linear's own result [..., out], with the adapters of the batch's requests added."""
        if x.numel() == 0:
            return base
        adapter, query_start = self.batch.rows(x)
        rows, flat = x.reshape(-1, x.shape[-1]), base.reshape(-1, base.shape[-1])
        if torch.is_grad_enabled() and (x.requires_grad or base.requires_grad or self.lora_a.requires_grad or self.lora_b.requires_grad):
            out = _LoraAdd.apply(rows, flat, self.lora_a, self.lora_b, self.scaling, adapter, query_start, self.save_bits)
        else:   # (the Linear's result is nobody else's yet)
            flat = flat.contiguous()
            out = load_extension().lora_add(rows, flat, self.lora_a, self.lora_b, self.scaling, adapter, query_start, out=flat)
        return out.reshape(base.shape)


def _kernel_linears(model, targets):
    for name, module in model.named_modules():
        if isinstance(module, KernelQuantLinear) and (re.search(targets, name) if targets is not None else name.split(".")[-1] != "lm_head"):
            yield name, module


def _forget_captured(model) -> None:
    from llmquant.runtime import drop_kept   # (runtimes kept on the model have steps without the change)

    drop_kept(model)


def add_adapters(model, rank: int = 16, slots: int = 1, alpha: float | None = None, targets: str | None = None,
                 save_bits: int = 16, dtype=None) -> list[str]:
    """A bank of adapters beside every kernel-mode Linear whose name `targets` (a regular expression) finds; without it, beside all but
    lm_head. alpha: scaling is alpha / rank (None: 2). Everything else of the model stops learning. Steps that a program of its own captured before run on
    without the adapters: capture them again. Returns the names."""
    chosen = [(name, module) for name, module in _kernel_linears(model, targets)]
    if not chosen:
        raise ValueError("the model has no kernel-mode Linear of that name")
    if any(module._adapted for _, module in chosen):
        raise ValueError("there are adapters already: remove_adapters() first")
    device = chosen[0][1].qdata.device
    if any(module.qdata.device != device for _, module in chosen):
        raise ValueError("adapters take a model on one device")
    batch = getattr(model, "_llmq_adapter_batch", None)
    if batch is None:
        batch = AdapterBatch(device)
    floating = dtype or next((p.dtype for p in model.parameters() if p.is_floating_point()), torch.bfloat16)
    banks = [LoraAdapters(module.in_features, module.out_features, rank, slots, 2.0 * rank if alpha is None else alpha, floating, device,
                          batch, save_bits) for _, module in chosen]
    for parameter in model.parameters():
        parameter.requires_grad_(False)
    for (_, module), bank in zip(chosen, banks):
        module.adapters = bank
        module._adapted = True
    for bank in _banks(model):
        bank.requires_grad_(True)
    model.__dict__["_llmq_adapter_batch"] = batch
    _forget_captured(model)
    return [name for name, _ in chosen]


def _banks(model):
    return [m for m in model.modules() if isinstance(m, LoraAdapters)]


def use_adapters(model, adapter, query_start=None) -> None:
    """The adapter of each request of the calls that follow (AdapterBatch.select); None: nobody has one."""
    banks = _banks(model)
    if not banks:
        raise ValueError("the model has no adapters: add_adapters() first")
    for batch in {id(b.batch): b.batch for b in banks}.values():
        batch.clear() if adapter is None else batch.select(adapter, query_start)


def remove_adapters(model) -> None:
    """The model as it was before add_adapters() (its parameters stay frozen)."""
    for module in model.modules():
        if isinstance(module, KernelQuantLinear) and module._adapted:
            del module.adapters
            module._adapted = False
    model.__dict__.pop("_llmq_adapter_batch", None)
    _forget_captured(model)


def adapter_parameters(model):
    """What an optimizer of the adapters takes."""
    return [p for bank in _banks(model) for p in bank.parameters()]
