"""Engine.score on the GPU: the bf16 kernels track the fp32 CPU oracle on the same random weights, with and without
alternatives, for grouped heads, sinks with a sliding window, experts and latent attention."""
import pytest
import torch

from sglang_neuron_b200.configs import model_config as mc
from sglang_neuron_b200.engine import Engine
from sglang_neuron_b200.parallel.state import destroy_parallel
from sglang_neuron_b200.server_args import ServerArgs

pytestmark = pytest.mark.gpu

DENSE = ("qwen3-8b", dict(num_hidden_layers=2, vocab_size=2048, hidden_size=512, intermediate_size=1024,
                          num_attention_heads=8, num_key_value_heads=4, head_dim=128))
SINKS = ("gpt-oss-120b", dict(num_hidden_layers=2, vocab_size=2048, hidden_size=512, intermediate_size=256,
                              num_local_experts=8, num_attention_heads=8, num_key_value_heads=2, head_dim=64,
                              sliding_window=16))
LATENT = ("deepseek-v2-lite", dict(num_hidden_layers=2, vocab_size=2048, hidden_size=512, intermediate_size=1024,
                                   moe_intermediate_size=128, n_routed_experts=8, num_experts_per_tok=2,
                                   num_attention_heads=4))


def _engine(base, over, device):
    destroy_parallel()
    mc.PRESETS[base + "-score"] = dict(mc.PRESETS[base], **over)
    return Engine(ServerArgs(model=base + "-score", device=device, dtype="bfloat16" if device == "cuda" else "float32",
                             page_size=16, context_length=512, max_running_requests=8, disable_cuda_graph=True,
                             random_weight_std=0.05, random_gen_device="cpu", max_total_tokens=4096))


def _prompts():
    g = torch.Generator().manual_seed(3)
    return [torch.randint(0, 2048, (n,), generator=g).tolist() for n in (5, 1, 140, 300, 2, 17)]


def _flat(scores, key="input_token_logprobs"):
    return torch.tensor([v[0] if isinstance(v, list) else v for d in scores for v in d[key][1:]])


@pytest.mark.parametrize("model,rel", [(DENSE, 0.05), (SINKS, 0.2), (LATENT, 0.2)], ids=["dense", "sinks", "latent"])
def test_score_tracks_the_cpu_oracle(model, rel):
    """`rel`: what the engine's own logits tests allow against the oracle (experts run on MXFP8 activations), of
    logits with a standard deviation of 0.05 sqrt(512)."""
    base, over = model
    tol = rel * 0.05 * 512 ** 0.5
    prompts = _prompts()
    want = _engine(base, over, "cpu").score(prompts)
    eng = _engine(base, over, "cuda")
    got = eng.score(prompts)
    top = eng.score(prompts, top_logprobs_num=5)
    for d, p in zip(got, prompts):
        assert [t for _, t in d["input_token_logprobs"]] == p
    w, g, t = _flat(want), _flat(got), _flat(top)
    assert len(g) == sum(len(p) - 1 for p in prompts) and bool(torch.isfinite(g).all())
    assert (g - w).abs().mean().item() < tol and (t - w).abs().mean().item() < tol
    e = (_flat(got, "input_entropies") - _flat(want, "input_entropies")).abs()
    assert e.mean().item() < tol
    # the logits are rounded to bf16 on the way with alternatives (half a unit in 2^8 of a few units), not without
    assert (g - t).abs().max().item() < 0.1
    for d in top:
        for (lp, tok), row in zip(d["input_token_logprobs"][1:], d["input_top_logprobs"][1:]):
            vals = [v for v, _ in row]
            assert len(row) == 5 and vals == sorted(vals, reverse=True) and lp <= vals[0] + 1e-6
            assert all(abs(v - lp) < 1e-6 for v, i in row if i == tok)


def test_score_between_generations():
    """Scoring leaves the serving state alone."""
    eng = _engine(*DENSE, "cuda")
    prompts = [p for p in _prompts() if len(p) > 2]
    before = [o["output_ids"] for o in eng.generate(prompts, {"max_new_tokens": 6})]
    first = eng.score(prompts, top_logprobs_num=2)
    after = [o["output_ids"] for o in eng.generate(prompts, {"max_new_tokens": 6})]
    assert before == after
    assert eng.score(prompts, top_logprobs_num=2) == first
