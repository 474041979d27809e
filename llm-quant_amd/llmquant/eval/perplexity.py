"""Perplexity of a model over token ids, without its logits (the reference's evaluation is described by its pipeline of
llmquant/eval/evaluate.py, which hands the logits of every position to a loss): the accuracy beside the timings of a result row.
"""

from __future__ import annotations

import inspect
import math

import torch

from llmquant.hip.ops import vocab_cross_entropy


@torch.no_grad()
def token_losses(model, input_ids: torch.Tensor) -> torch.Tensor:
    """-log p of every token but the first given those before it: float32 [batch, length - 1]. The model's decoder runs as it
    is; its lm_head (an nn.Linear, or a kernel-mode Linear: its codes) goes into the loss, and no logits are made but each sequence's last, from which it is
    seen that they are the head's product and nothing else: a model that scales or caps its logits is refused."""
    if input_ids.dim() != 2 or input_ids.shape[1] < 2:
        raise ValueError(f"token ids must be [batch, length of 2 or more], got {tuple(input_ids.shape)}")
    return _losses(model, input_ids, _decoded(model, input_ids))


def _losses(model, input_ids: torch.Tensor, hidden: torch.Tensor) -> torch.Tensor:
    hidden = hidden[:, :-1]
    return vocab_cross_entropy(hidden, model.get_output_embeddings(), input_ids[:, 1:], reduction="none")


def _decoded(model, input_ids: torch.Tensor) -> torch.Tensor:
    """The decoder's hidden states [batch, length, hidden size], of a model whose logits are its head's product with them (not asked in a capture, which can
    wait for no answer)."""
    if input_ids.is_cuda and torch.cuda.is_current_stream_capturing():
        return model.get_decoder()(input_ids=input_ids, use_cache=False).last_hidden_state
    if "logits_to_keep" not in inspect.signature(model.forward).parameters:   # (all logits or none: a token tells)
        _check_logits(model, model.get_decoder()(input_ids=input_ids[:1, :1], use_cache=False).last_hidden_state,
                      model(input_ids=input_ids[:1, :1], use_cache=False).logits)
        return model.get_decoder()(input_ids=input_ids, use_cache=False).last_hidden_state
    states = []
    hook = model.get_decoder().register_forward_hook(lambda module, args, out: states.append(out.last_hidden_state))
    try:
        logits = model(input_ids=input_ids, use_cache=False, logits_to_keep=1).logits
    finally:
        hook.remove()
    _check_logits(model, states[-1][:, -1:], logits[:, -1:])
    return states[-1]


def _check_logits(model, hidden: torch.Tensor, logits: torch.Tensor) -> None:
    """(The same product of as many rows: equal to the bit, but for sums whose order may change.)"""
    own = model.get_output_embeddings()(hidden).float()
    if own.shape != logits.shape or (own - logits.float()).norm() > 1e-4 * own.norm():   # (NaN stays NaN)
        raise ValueError(f"{type(model).__name__} makes more of its logits than its head's product with the hidden states (it scales or caps them): "
                         "their loss is not that of the head")


@torch.no_grad()
def measure_perplexity(model, input_ids: torch.Tensor, context: int = 2048) -> dict:
    """exp of the mean loss over a text [1, length] (or [length]) cut into windows of `context` tokens, each by itself: {"ppl",
    "nll", "ppl_tokens"}, columns for latency_row(..., accuracy=...)."""
    ids = input_ids.reshape(1, -1)
    if context < 2:
        raise ValueError(f"a window has 2 tokens or more, got {context}")
    device = next(model.parameters()).device
    total, count = torch.zeros((), dtype=torch.float64, device=device), 0
    for at in range(0, ids.shape[1], context):
        window = ids[:, at:at + context].to(device)
        if window.shape[1] > 1:
            if count == 0:   # (what the model makes of its logits it makes of all windows')
                hidden = _decoded(model, window)
            else:
                hidden = model.get_decoder()(input_ids=window, use_cache=False).last_hidden_state
            total += _losses(model, window, hidden).double().sum()
            count += window.shape[1] - 1
    if count == 0:
        raise ValueError("a text of fewer than two tokens has no perplexity")
    nll = total.item() / count
    return {"ppl": math.exp(nll) if nll < 700 else math.inf, "nll": nll, "ppl_tokens": count}
