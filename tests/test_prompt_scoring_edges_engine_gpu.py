"""Engine.score on the GPU: what asking for alternatives, and how the head's weight is kept, must not change."""
import pytest

from sglang_neuron_b200.ops.gemm import TiledWeight
from test_prompt_scoring_engine_gpu import DENSE, LATENT, SINKS, _engine, _flat, _prompts

pytestmark = pytest.mark.gpu

# A logit is a sum of 512 products added up in fp32 16 at a time: 36 roundings of at most 2^-23 of sum |h||w|, here about
# 512 * 0.8 * 0.04 = 16: 7e-5. A log-probability has two of them and the statistics' own 3e-4, on either side.
TOL = 2 * (2 * 7e-5 + 3e-4)


@pytest.mark.parametrize("model", [DENSE, SINKS, LATENT], ids=["dense", "sinks", "latent"])
def test_scores_do_not_change_with_alternatives(model):
    eng = _engine(*model, "cuda")
    prompts = _prompts()
    plain, top = eng.score(prompts), eng.score(prompts, top_logprobs_num=5)
    assert (_flat(plain) - _flat(top)).abs().max().item() <= TOL
    # an entropy's error is at most the log-probabilities' times the mean distance from the best, a few units here
    assert (_flat(plain, "input_entropies") - _flat(top, "input_entropies")).abs().max().item() <= 8 * TOL
    # the tiled weight alone, without the library's copy of it
    head = eng.runner.model.lm_head
    w = head.gemm_weight
    head._packed = TiledWeight(w.rowmajor if isinstance(w, TiledWeight) and w.rowmajor is not None else head.weight)
    tiled, tiled_top = eng.score(prompts), eng.score(prompts, top_logprobs_num=5)
    assert (_flat(tiled) - _flat(plain)).abs().max().item() <= TOL
    assert (_flat(tiled_top) - _flat(plain)).abs().max().item() <= TOL
