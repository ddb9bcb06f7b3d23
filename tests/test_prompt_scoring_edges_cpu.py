"""Edge cases of the prompt-scoring operators' PyTorch forms."""
import math

import pytest
import torch

from sglang_neuron_b200.ops.logprobs import head_logprobs, token_logprobs
from sglang_neuron_b200.ops.prompt import prompt_attention


def test_prompt_attention_leaves_rows_outside_every_prompt():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(12, 8, generator=g) for _ in range(3))
    ip = torch.tensor([3, 7, 7, 10], dtype=torch.int32)
    mark = torch.full((12, 8), 7.0)
    out = prompt_attention(q, k, v, ip, 2, 2, 4, out=mark)
    assert out is mark and bool((out[:3] == 7).all()) and bool((out[10:] == 7).all())
    want = prompt_attention(q[3:10], k[3:10], v[3:10], ip - 3, 2, 2, 4)
    assert torch.equal(out[3:10], want)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("window", [0, 4])
def test_prompt_attention_masked_places_hold_anything(bad, where, window):
    """As on CUDA: a NaN or infinity reaches only the rows that see it."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(20, w, generator=g) for w in (16, 8, 8))
    ip = torch.tensor([0, 12, 20], dtype=torch.int32)
    clean = prompt_attention(q, k, v, ip, 4, 2, 4, window=window)
    (k if where == "k" else v)[5, :4] = bad  # the first KV head: query heads 0 and 1
    out = prompt_attention(q, k, v, ip, 4, 2, 4, window=window)
    hit = torch.zeros(20, 16, dtype=torch.bool)
    hit[5:9 if window else 12, :8] = True
    assert torch.equal(out[~hit], clean[~hit])
    if where == "v":
        assert torch.equal(out[hit], torch.full_like(out[hit], bad)) or bool(torch.isnan(out[hit]).all())


def test_operators_are_forward_only():
    """The CUDA kernels have no backward pass, so the PyTorch forms carry no gradient either."""
    q = torch.randn(4, 8, requires_grad=True)
    ip = torch.tensor([0, 4], dtype=torch.int32)
    w, ids = torch.randn(9, 8, requires_grad=True), torch.zeros(4, dtype=torch.long)
    outs = [prompt_attention(q, q, q, ip, 2, 2, 4), prompt_attention(q, q, q, ip, 2, 2, 4, out=torch.zeros(4, 8))]
    outs += list(head_logprobs(q, w, ids)[:3]) + list(token_logprobs(q, ids, top_k=2)[:4])
    assert not any(t.requires_grad for t in outs)
