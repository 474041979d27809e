"""Adapters beside a kernel-mode model as they are learned and served: the quantized Linears' gradients, banks of adapters, the loss over
the quantized head and perplexity, together on small Llama-architecture models.

The whole-model comparisons run in float32 against the same architecture in 64 bits with the dequantized weights; their bar is the one that the
package's whole-model float32 logits have, a relative L2 distance of 1e-3. Single operators have their bounds in test_gpu_lora.py and
test_gpu_vocab_loss.py."""

import copy
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def build(dtype, hidden=256, inter=512, heads=4, kv_heads=2, head_dim=64, vocab=1000, layers=2, recipe=None):
    from llmquant import QuantConfig, oneshot
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(hidden_size=hidden, intermediate_size=inter, num_hidden_layers=layers, num_attention_heads=heads,
                      num_key_value_heads=kv_heads, head_dim=head_dim, vocab_size=vocab, rms_norm_eps=1e-5,
                      rope_parameters={"rope_type": "default", "rope_theta": 500000.0}, tie_word_embeddings=False,
                      max_position_embeddings=2048, attn_implementation="eager")
    model = LlamaForCausalLM(cfg)
    for p in model.parameters():
        if p.dim() > 1:
            nn.init.normal_(p, 0, 0.05)
    model = model.to(dtype).cuda().eval()
    recipe = recipe or QuantConfig(attn_weight="int8", mlp_weight="int4", head_weight="int8", kv_cache="int8")
    return model, oneshot(copy.deepcopy(model), recipe.to_modifier("kernel"))


class Wide(nn.Module):
    """A Linear of the quantized weight in 64 bits, with its adapters, rows of each request by turns."""

    def __init__(self, module, adapters):
        super().__init__()
        weight = module._dequantized_weight(torch.float32, real_width=True)
        if weight.shape[1] != module.in_features:
            head_dim = module._weight_args.head_dim
            weight = (weight.unflatten(1, (module.in_features // head_dim, -1))[..., :head_dim].flatten(1) if head_dim
                      else weight[:, :module.in_features])
        self.weight = weight.double()
        bank = getattr(module, "adapters", None)
        self.adapters = adapters
        if bank is not None:
            self.a, self.b = (nn.Parameter(p.detach().double()) for p in (bank.lora_a, bank.lora_b))
            self.s = bank.scaling.double()
        else:
            self.a = None

    def forward(self, x):
        out = x @ self.weight.T
        if self.a is None:
            return out
        parts = []
        for row, a in zip(x, self.adapters):
            parts.append((row @ self.a[a].T) @ self.b[a].T * self.s[a] if a >= 0 else torch.zeros(row.shape[0], out.shape[-1], dtype=out.dtype, device=out.device))
        return out + torch.stack(parts)


def widened(kernel, adapters):
    from llmquant.quantizers import KernelQuantLinear

    wide = copy.deepcopy(kernel)
    for name, module in list(wide.named_modules()):
        if isinstance(module, KernelQuantLinear):
            parent = wide.get_submodule(name.rpartition(".")[0]) if "." in name else wide
            setattr(parent, name.rpartition(".")[2], Wide(module, adapters))
    return wide.double()


def rel(got, want):
    return ((got.double() - want.double()).norm() / want.double().norm().clamp_min(1e-300)).item()


def stir(model, seed=1):
    """B of every adapter away from zero."""
    from llmquant.quantizers import LoraAdapters

    gen = torch.Generator(device="cuda").manual_seed(seed)
    for bank in model.modules():
        if isinstance(bank, LoraAdapters):
            with torch.no_grad():
                bank.lora_b.copy_(0.1 * torch.randn(bank.lora_b.shape, generator=gen, device="cuda"))


@pytest.mark.parametrize("recipe", ["mixed", "int4 with a bf16 head"])
@pytest.mark.parametrize("save_bits", [16, 8])
def test_a_training_step_on_frozen_codes(save_bits, recipe):
    from llmquant import QuantConfig
    from llmquant.hip import vocab_cross_entropy
    from llmquant.quantizers import adapter_parameters, add_adapters, use_adapters

    config = None if recipe == "mixed" else QuantConfig(attn_weight="int4", mlp_weight="int4", head_weight="bf16")
    _, kernel = build(torch.float32, recipe=config)
    names = add_adapters(kernel, rank=8, slots=3, save_bits=save_bits)
    assert len(names) == 14 and not any("lm_head" in n for n in names)
    stir(kernel)
    adapters = [2, -1, 0]
    use_adapters(kernel, adapters)
    ids = torch.randint(0, 1000, (3, 37), generator=torch.Generator().manual_seed(2)).cuda()
    targets = ids.roll(-1, 1).clone()
    targets[:, -1] = -100
    targets[0, :9] = -100
    learned = adapter_parameters(kernel)
    assert {id(p) for p in kernel.parameters() if p.requires_grad} == {id(p) for p in learned}
    hidden = kernel.model(input_ids=ids, use_cache=False).last_hidden_state
    loss = vocab_cross_entropy(hidden, kernel.lm_head, targets)
    loss.backward()

    wide = widened(kernel, adapters)
    want = F.cross_entropy(wide(input_ids=ids, use_cache=False).logits.flatten(0, 1), targets.flatten())
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-3 * want.item()
    linears = [m for m in wide.modules() if isinstance(m, Wide) and m.a is not None]
    assert len(linears) * 2 == len(learned)
    for bank_a, bank_b, ref in zip(learned[::2], learned[1::2], linears):
        assert rel(bank_b.grad, ref.b.grad) < 1e-3
        # (8 bits: each value of x off by at most half a step of 127 of its group's largest, a norm of 1 / 254 of largest over root mean square, below 4 for 128
        # values of these)
        assert rel(bank_a.grad, ref.a.grad) < (1e-3 if save_bits == 16 else 4 / 254 + 1e-3)
        assert (bank_a.grad[1] == 0).all() and (bank_b.grad[1] == 0).all()


def test_served_together_and_one_by_one():
    """Requests with their own adapters in one batch, ragged and as single rows, each as when it is alone."""
    from llmquant.quantizers import add_adapters, remove_adapters, use_adapters

    _, kernel = build(torch.float32)
    ids = torch.randint(0, 1000, (4, 9), generator=torch.Generator().manual_seed(3)).cuda()
    with torch.no_grad():
        before = kernel(input_ids=ids, use_cache=False).logits
        add_adapters(kernel, rank=16, slots=2)
        assert torch.equal(kernel(input_ids=ids, use_cache=False).logits, before)   # nobody has one
        use_adapters(kernel, [0, 1, 1, 0])
        assert torch.equal(kernel(input_ids=ids, use_cache=False).logits, before)   # B is zero: x + 0
        stir(kernel)
        use_adapters(kernel, [0, -1, 1, 7])
        together = kernel(input_ids=ids, use_cache=False).logits
        for b, a in enumerate([0, -1, 1, 7]):
            use_adapters(kernel, [a])
            alone = kernel(input_ids=ids[b:b + 1], use_cache=False).logits[0]
            assert rel(together[b], alone) < 1e-3
        assert rel(together[0], before[0]) > 1e-2 and rel(together[1], before[1]) < 1e-3 and rel(together[3], before[3]) < 1e-3
        linear = kernel.model.layers[0].mlp.up_proj
        x = torch.randn(6, 256, device="cuda")
        start = torch.tensor([0, 4, 4, 6], dtype=torch.int32, device="cuda")
        use_adapters(kernel, [1, 0, -1], start)
        got = linear(x)
        use_adapters(kernel, [1, 1, 1, 1, -1, -1])
        assert torch.allclose(got, linear(x), rtol=1e-4, atol=1e-5)
        with pytest.raises(ValueError, match="no whole number"):
            linear(x[:4])
        use_adapters(kernel, None)
        assert torch.equal(linear(x), linear._frozen(x))
        remove_adapters(kernel)
        assert torch.equal(kernel(input_ids=ids, use_cache=False).logits, before)


def test_generation_with_adapters_and_a_captured_step():
    """The runtime that walks the modules takes the adapters along; a captured step reads what was selected last."""
    from llmquant.quantizers import add_adapters, remove_adapters, use_adapters
    from llmquant.runtime import graphed_generate, kernel_runtime
    from llmquant.runtime.llama_fused import LlamaFusedRuntime

    _, kernel = build(torch.float32, hidden=512, inter=1024, heads=8, vocab=512)   # (four groups a row: what the fused step takes)
    ids = torch.randint(0, 512, (1, 12), generator=torch.Generator().manual_seed(4)).cuda()
    plain = graphed_generate(kernel, ids, 12, kv_bits=8)
    assert isinstance(kernel_runtime(kernel, 32), LlamaFusedRuntime)
    add_adapters(kernel, rank=8, slots=2)
    stir(kernel)
    assert not isinstance(kernel_runtime(kernel, 32), LlamaFusedRuntime)

    def eager(a):
        use_adapters(kernel, [a])
        runtime = kernel_runtime(kernel, 32)
        return runtime.generate(ids, 12, use_graph=False)

    streams = {a: eager(a) for a in (-1, 0, 1)}
    assert not torch.equal(streams[0], streams[1])
    for a in (0, 1, -1, 1, 0):   # (one captured step, replayed with each)
        use_adapters(kernel, [a])
        assert torch.equal(graphed_generate(kernel, ids, 12, kv_bits=8), streams[a]), a
    remove_adapters(kernel)
    assert torch.equal(graphed_generate(kernel, ids, 12, kv_bits=8), plain)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_perplexity_without_logits(dtype):
    from llmquant.eval import latency_row, measure_perplexity, token_losses

    dense, kernel = build(dtype)
    ids = torch.randint(0, 1000, (1, 301), generator=torch.Generator().manual_seed(5)).cuda()
    for model in (dense, kernel):
        with torch.no_grad():
            losses = token_losses(model, ids[:, :120])
            hidden = model.model(input_ids=ids[:, :120], use_cache=False).last_hidden_state[0, :-1]
            weight = model.lm_head.weight if model is dense else model.lm_head._dequantized_weight(dtype)
            want = F.cross_entropy(hidden.double() @ weight.double().T, ids[0, 1:120], reduction="none")
        assert (losses[0].double() - want).abs().max() < 1e-4
        row = measure_perplexity(model, ids, context=100)
        assert row["ppl_tokens"] == 3 * 99 and math.isclose(row["ppl"], math.exp(row["nll"]))
        with torch.no_grad():
            parts = torch.cat([token_losses(model, ids[:, at:at + 100]) for at in (0, 100, 200)], 1)
        assert math.isclose(row["nll"], parts.double().mean().item(), rel_tol=1e-6)
        assert latency_row(None, "kernel", {"ttft_ms": 1.0}, accuracy=row)["ppl"] == row["ppl"]
    with pytest.raises(ValueError, match="fewer than two"):
        measure_perplexity(dense, ids[:, :1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 3, 70, 300])
@pytest.mark.parametrize("geometry", ["plain", "heads", "ragged", "bias", "int8 activations"])
def test_gradient_of_a_kernel_linear(geometry, rows, dtype):
    """Forward as without a gradient, backward the product with the weight that the codes stand for, rounded to the type."""
    from llmquant import QuantConfig
    from llmquant.core.scheme import QuantizationArgs, QuantizationScheme
    from llmquant.quantizers import KernelQuantLinear

    torch.manual_seed(rows)
    heads = 64 if geometry == "heads" else None
    inp = {"ragged": 200, "heads": 192}.get(geometry, 256)
    linear = nn.Linear(inp, 136, bias=geometry == "bias", dtype=dtype, device="cuda")
    weights = QuantizationArgs(num_bits=4, strategy="group", group_size=128, head_dim=heads)
    act = QuantizationArgs(num_bits=8, strategy="group", group_size=128) if geometry == "int8 activations" else None
    module = KernelQuantLinear.from_linear(linear, QuantizationScheme(weights=weights, input_activations=act))
    x = torch.randn(2, rows, inp, device="cuda").to(dtype).requires_grad_()
    out = module(x)
    with torch.no_grad():
        assert torch.equal(out, module(x))
    grad = torch.randn_like(out)
    out.backward(grad)
    weight = Wide(module, []).weight if dtype == torch.float32 else None
    if weight is None:
        full = module._dequantized_weight(dtype)
        weight = (full.unflatten(1, (inp // heads, -1))[..., :heads].flatten(1) if heads else full[:, :inp]).double()
    want = grad.double() @ weight
    size = grad.double().abs() @ weight.abs()
    u = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    tol = (6 * 136 + 72) * 2.0 ** -24 * size + 2.0 ** -22 * size
    assert ((x.grad.double() - want).abs() <= tol + u * (want.abs() + tol)).all()
    if geometry == "bias":
        assert rel(module.bias.grad, grad.double().sum((0, 1))) < 4 * u


def test_refusals_of_the_host_side():
    from llmquant.hip import vocab_cross_entropy
    from llmquant.quantizers import add_adapters, use_adapters

    dense, kernel = build(torch.float32, layers=1)
    with pytest.raises(ValueError, match="no adapters"):
        use_adapters(kernel, [0])
    with pytest.raises(ValueError, match="no kernel-mode Linear"):
        add_adapters(dense)
    with pytest.raises(ValueError, match="rank"):
        add_adapters(kernel, rank=12)
    add_adapters(kernel, rank=8, targets="q_proj|lm_head")
    with pytest.raises(ValueError, match="already"):
        add_adapters(kernel, rank=8, targets="q_proj")
    with pytest.raises(ValueError, match="no request"):
        use_adapters(kernel, [])
    with pytest.raises(ValueError, match="query_start"):
        use_adapters(kernel, [0], torch.zeros(3, dtype=torch.int32, device="cuda"))
    hidden = torch.zeros(2, 256, device="cuda")
    targets = torch.zeros(2, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError, match="adapters"):
        vocab_cross_entropy(hidden, kernel.lm_head, targets)
    with pytest.raises(ValueError, match="bias"):
        vocab_cross_entropy(hidden, nn.Linear(256, 10, device="cuda"), targets)
    with pytest.raises(ValueError, match="reduction"):
        vocab_cross_entropy(hidden, dense.lm_head, targets, reduction="max")
    with pytest.raises(ValueError, match="do not go with"):
        vocab_cross_entropy(hidden, dense.lm_head, targets[:1])
    assert vocab_cross_entropy(hidden, dense.lm_head, torch.full_like(targets, -100)).isnan()
