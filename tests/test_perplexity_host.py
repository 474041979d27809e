"""Losses without logits are of models whose logits are the head's product; others are refused before the loss is asked for. On the CPU."""

import pytest
import torch
from transformers import LlamaConfig, LlamaForCausalLM

from llmquant.eval.perplexity import _decoded


def small(kind=LlamaForCausalLM):
    torch.manual_seed(0)
    return kind(LlamaConfig(hidden_size=64, intermediate_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=16,
                            vocab_size=100, tie_word_embeddings=False, attn_implementation="eager", initializer_range=0.2)).eval()


class Scaled(LlamaForCausalLM):
    """Logits times a factor, in place."""

    def forward(self, *args, **kwargs):
        out = super().forward(*args, **kwargs)
        out.logits.mul_(0.125)
        return out


class Capped(LlamaForCausalLM):
    def forward(self, *args, **kwargs):
        out = super().forward(*args, **kwargs)
        out.logits = torch.tanh(out.logits / 30) * 30
        return out


class AllLogits(LlamaForCausalLM):
    """Without a way to ask for the last logits alone."""

    factor = 1.0

    def forward(self, input_ids, use_cache=False):
        assert input_ids.shape == (1, 1)   # (not all of them)
        out = super().forward(input_ids=input_ids, use_cache=use_cache)
        out.logits = out.logits * self.factor
        return out


class Moved(LlamaForCausalLM):
    """The head takes something else than the decoder's states."""

    def __init__(self, config):
        super().__init__(config)
        self.lm_head.register_forward_pre_hook(lambda module, args: (args[0] + 1,) if self.moved else None)
        self.moved = True

    def get_output_embeddings(self):
        return torch.nn.Linear(64, 100, bias=False)


IDS = torch.randint(0, 100, (3, 9), generator=torch.Generator().manual_seed(1))


@pytest.mark.parametrize("kind", [LlamaForCausalLM, AllLogits])
@torch.no_grad()
def test_the_decoders_states(kind):
    model = small(kind)
    for ids in (IDS, IDS[:1]):
        states = _decoded(model, ids)
        want = model.get_decoder()(input_ids=ids, use_cache=False).last_hidden_state
        assert torch.equal(states, want) and not model.get_decoder()._forward_hooks


@pytest.mark.parametrize("kind", [Scaled, Capped, Moved, "all"])
@torch.no_grad()
def test_logits_that_are_more_than_the_heads_product_are_refused(kind):
    model = small(AllLogits if kind == "all" else kind)
    if kind == "all":
        model.factor = 2.0
    with pytest.raises(ValueError, match="makes more of its logits"):
        _decoded(model, IDS)
    assert not model.get_decoder()._forward_hooks


@torch.no_grad()
def test_a_broken_model_is_not_taken_for_another():
    model = small()
    model.model.norm.weight.fill_(float("nan"))
    assert _decoded(model, IDS).isnan().all()
