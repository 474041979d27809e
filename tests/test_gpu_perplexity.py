"""Losses without logits on the device: captured, and of a model that makes more of its logits than its head's product."""

import types

import pytest
import torch

pytestmark = pytest.mark.gpu


class Decoder(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.embed = torch.nn.Embedding(1000, 256)

    def forward(self, input_ids, use_cache=False):
        return types.SimpleNamespace(last_hidden_state=torch.tanh(self.embed(input_ids)))


class Model(torch.nn.Module):
    """Embeddings and a head."""

    def __init__(self):
        super().__init__()
        self.decoder, self.head = Decoder(), torch.nn.Linear(256, 1000, bias=False)

    def get_decoder(self):
        return self.decoder

    def get_output_embeddings(self):
        return self.head

    def forward(self, input_ids, use_cache=False, logits_to_keep=0):
        return types.SimpleNamespace(logits=self.head(self.decoder(input_ids).last_hidden_state[:, -logits_to_keep:]))


def test_captured_losses():
    """Seen eagerly to be the head's, then replayed: a capture waits for no answer."""
    from llmquant.eval import token_losses

    torch.manual_seed(0)
    model = Model().cuda()
    ids = torch.randint(0, 1000, (2, 40), generator=torch.Generator().manual_seed(5)).cuda()
    held = ids.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        token_losses(model, held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_losses(model, held)
    for turn in range(3):
        held.copy_(ids.roll(turn, 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, token_losses(model, held))


@pytest.mark.parametrize("which", ["dense", "kernel"])
def test_capped_logits_are_refused(which):
    from llmquant.eval import measure_perplexity, token_losses
    from test_gpu_adapters import build

    model = build(torch.bfloat16)[which == "kernel"]
    ids = torch.randint(0, 1000, (1, 40), generator=torch.Generator().manual_seed(5)).cuda()
    assert measure_perplexity(model, ids, 16)["ppl_tokens"] == 37
    plain = model.forward

    def capped(input_ids=None, use_cache=None, logits_to_keep=0):
        out = plain(input_ids=input_ids, use_cache=use_cache, logits_to_keep=logits_to_keep)
        out.logits = torch.tanh(out.logits / 2) * 2
        return out

    model.forward = capped
    for call in (lambda: measure_perplexity(model, ids, 16), lambda: token_losses(model, ids)):
        with pytest.raises(ValueError, match="makes more of its logits"):
            call()
