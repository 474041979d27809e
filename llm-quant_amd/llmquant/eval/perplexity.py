"""Perplexity of a model over token ids, without its logits (the reference's evaluation is described by its pipeline of
llmquant/eval/evaluate.py, which hands the logits of every position to a loss): the accuracy beside the timings of a result row.
"""

from __future__ import annotations

import math

import torch

from llmquant.hip.ops import vocab_cross_entropy


@torch.no_grad()
def token_losses(model, input_ids: torch.Tensor) -> torch.Tensor:
    """-log p of every token but the first given those before it: float32 [batch, length - 1]. The model's decoder runs as it
    is; its lm_head (an nn.Linear, or a kernel-mode Linear: its codes) goes into the loss, and no logits are made."""
    if input_ids.dim() != 2 or input_ids.shape[1] < 2:
        raise ValueError(f"token ids must be [batch, length of 2 or more], got {tuple(input_ids.shape)}")
    hidden = model.get_decoder()(input_ids=input_ids, use_cache=False).last_hidden_state[:, :-1]
    return vocab_cross_entropy(hidden, model.get_output_embeddings(), input_ids[:, 1:], reduction="none")


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
            total += token_losses(model, window).double().sum()
            count += window.shape[1] - 1
    if count == 0:
        raise ValueError("a text of fewer than two tokens has no perplexity")
    nll = total.item() / count
    return {"ppl": math.exp(nll) if nll < 700 else math.inf, "nll": nll, "ppl_tokens": count}
