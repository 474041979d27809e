"""Python-level ops over the extension (counterpart of llmquant/cuda/ops.py)."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from llmquant.core.observers import pad_to_group
from llmquant.core.scheme import QuantizationArgs
from llmquant.hip.build import load_extension


def _group_size_for(x: torch.Tensor, args: QuantizationArgs) -> int:
    if args.strategy == "group":
        return args.group_size
    if args.strategy in ("channel", "token"):
        return x.shape[-1]  # a single group spanning the row
    raise ValueError(f"unsupported strategy {args.strategy!r}")


def _rows_in_place(numel: int, width: int, element_size: int, group_size: int) -> bool:
    """Whether ragged rows go to the kernel that takes them as they lie: groups of a power of two 16-byte packets that
    one wave holds, rows of a packet or more, and fewer than 2^31 packets counting each row's zeros up to whole groups
    (narrow rows under wide groups are mostly zeros)."""
    if numel == 0 or width < 8 or width % group_size == 0 or element_size > 4:
        return False
    packets, rest = divmod(group_size * element_size, 16)
    padded_packets = numel // width * -(-width // group_size) * packets
    return rest == 0 and packets <= 64 and packets & (packets - 1) == 0 and padded_packets < 1 << 31


def fake_quantize_hip(x: torch.Tensor, args: QuantizationArgs, return_scale: bool = False):
    """Quant-dequant on the GPU, bit-exact with llmquant.core.quant_ops.fake_quantize.

    Groups run along the last axis. A last axis that is not a whole number of groups gives
    what the PyTorch form's zero padding and trimming give: for groups of a power of two 16-byte
    packets the kernel reads and writes the rows as they lie, others are padded and trimmed.
    """
    group_size = _group_size_for(x, args)
    width = x.shape[-1]
    if x.is_cuda and _rows_in_place(x.numel(), width, x.element_size(), group_size):
        out, scale = load_extension().fake_quant_rows(x, args.num_bits, group_size, return_scale)
        return (out, scale) if return_scale else out
    padded = pad_to_group(x, group_size)
    out, scale = load_extension().fake_quant_group(padded, args.num_bits, group_size, return_scale)
    if padded.shape[-1] != width:
        out = out[..., :width]
    return (out, scale) if return_scale else out


def quantize_activation(x: torch.Tensor, args: QuantizationArgs):
    """(int8 codes [..., K], fp32 scales [..., K / group]) for an activation whose last axis
    is already a whole number of groups -- the dynamic A8 quantizer as one kernel."""
    group_size = _group_size_for(x, args)
    return load_extension().quant_group_codes(x, args.num_bits, group_size, False)


# the reference's name for the same op
fake_quantize_cuda = fake_quantize_hip


def keep(ctx, *tensors) -> None:
    """Tensors (or None) for the backward pass, where a change in place since then is an error; those of inference mode, which autograd does not save, as they are."""
    ctx.plain = [t if t is not None and t.is_inference() else None for t in tensors]
    ctx.save_for_backward(*(t if p is None else None for t, p in zip(tensors, ctx.plain)))


def kept(ctx) -> list:
    return [saved if p is None else p for saved, p in zip(ctx.saved_tensors, ctx.plain)]


class _VocabLoss(torch.autograd.Function):
    """Losses of rows over a vocabulary; the logits are made again in the backward pass, a piece at a time."""

    @staticmethod
    def forward(ctx, hidden, weight, wscale, out_group, targets, ignore_index):
        losses, lse = load_extension().vocab_loss(hidden, weight, targets, ignore_index, wscale, out_group)
        keep(ctx, hidden, weight, wscale, targets, lse)
        ctx.out_group, ctx.ignore_index = out_group, ignore_index
        return losses

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, weight, wscale, targets, lse = kept(ctx)
        of_hidden, of_weight = load_extension().vocab_loss_grad(hidden, weight, targets, lse, grad, ctx.ignore_index, wscale,
                                                                ctx.out_group, ctx.needs_input_grad[1])
        return of_hidden, of_weight, None, None, None, None


def _head_weight(head):
    """(weight or codes, scales or None, out_group) of an lm_head: a tensor, a Linear without bias, a kernel-mode Linear."""
    if isinstance(head, torch.Tensor):
        return head, None, 0
    if getattr(head, "bias", None) is not None:
        raise ValueError("a head with a bias has no fused loss")
    if getattr(head, "adapters", None) is not None:
        raise ValueError("a head with adapters has no fused loss")
    if hasattr(head, "qdata"):
        if head._needs_padding or head._int8_act:
            raise ValueError("a fused loss takes a weight-only head of whole groups")
        return head.qdata, head.wscale, head.out_group
    scheme = getattr(head, "scheme", None)
    weight = getattr(head, "weight", None)
    if weight is None or weight.dim() != 2 or (scheme is not None and scheme.input_activations is not None):
        raise TypeError(f"{type(head).__name__} is no head that a fused loss takes")
    return weight, None, 0


def vocab_cross_entropy(hidden, head, targets, ignore_index: int = -100, reduction: str = "mean"):
    """F.cross_entropy(head(hidden), targets) without the logits, in float32, differentiable by hidden and by a dense weight.

    hidden [..., hidden size]; head: an nn.Linear without bias, a kernel-mode Linear (its codes are frozen), or a weight [vocab, hidden size];
    targets int64 [...]. reduction "none", "sum", or "mean" over the rows whose target is not ignore_index (NaN if there is none,
    as F.cross_entropy has it). A target outside the vocabulary makes its loss NaN.
    """
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    weight, wscale, out_group = _head_weight(head)
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} do not go with hidden {tuple(hidden.shape)}")
    rows = hidden.reshape(-1, hidden.shape[-1])
    losses = _VocabLoss.apply(rows, weight, wscale, out_group, targets.reshape(-1), ignore_index)
    if reduction == "none":
        return losses.reshape(targets.shape)
    total = losses.sum()
    return total if reduction == "sum" else total / (targets != ignore_index).sum()
