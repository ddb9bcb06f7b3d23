"""Edge cases of the prompt-scoring operators' PyTorch forms."""
import math

import pytest
import torch

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
