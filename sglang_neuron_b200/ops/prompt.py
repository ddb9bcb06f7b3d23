"""Causal attention of packed whole prompts: keys and values straight from the projections, no paged cache.

For passes that keep nothing (scoring prompts). Forward only: results carry no gradient, on CUDA or CPU. GQA, sliding
window and learned per-head sinks as in the paged ops (ops/attention.py); the value width may differ from the key width
(decompressed latent attention: 192 / 128).
"""
from typing import Optional

import torch

from .._ext import checked
from .attention import _attend_ref
from .gemm import _status_buf


@torch.no_grad()
def prompt_attention_ref(q, k, v, qo_indptr, num_q_heads, num_kv_heads, head_dim, v_head_dim=None, window=0,
                         sm_scale=None, sinks=None):
    v_head_dim = head_dim if v_head_dim is None else v_head_dim
    sm_scale = head_dim ** -0.5 if sm_scale is None else sm_scale
    T = q.shape[0]
    out = torch.zeros(T, num_q_heads, v_head_dim, dtype=torch.float32, device=q.device)
    bounds = qo_indptr.tolist()
    for a, b in zip(bounds[:-1], bounds[1:]):
        if b <= a:
            continue
        pos = torch.arange(b - a, device=q.device)
        out[a:b] = _attend_ref(q[a:b].reshape(b - a, num_q_heads, head_dim),
                               k[a:b].reshape(b - a, num_kv_heads, head_dim).float(),
                               v[a:b].reshape(b - a, num_kv_heads, v_head_dim).float(), pos, pos, sm_scale, window,
                               sinks)
    return out.reshape(T, num_q_heads * v_head_dim)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, qo_indptr: torch.Tensor, num_q_heads: int,
                     num_kv_heads: int, head_dim: int, v_head_dim: Optional[int] = None, window: int = 0,
                     sm_scale: Optional[float] = None, sinks: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Tokens [qo_indptr[b], qo_indptr[b + 1]) are prompt b; every token attends to itself and the tokens before it
    in its prompt (the last `window` of them where window > 0). q [T, num_q_heads * head_dim], k and v [T,
    num_kv_heads * width]: bf16 or fp16 and widths of 64, 128 or 192 (values 128) on CUDA; views with a row stride
    (columns of a fused projection) are read in place, rows off 16-byte boundaries are copied first.
    Returns [T, num_q_heads * v_head_dim]; rows outside every prompt are left as they are."""
    v_head_dim = head_dim if v_head_dim is None else v_head_dim
    sm_scale = head_dim ** -0.5 if sm_scale is None else sm_scale
    if q.is_cuda:  # the kernel's entry checks its arguments (ValueError)
        return checked("prompt_attention", "prompt_attention", q, k, v, qo_indptr, num_q_heads, num_kv_heads, head_dim,
                       v_head_dim, window, sm_scale, sinks, out, _status_buf(q.device))
    if num_kv_heads <= 0 or num_q_heads % num_kv_heads:
        raise ValueError(f"{num_q_heads} heads do not divide over {num_kv_heads} KV heads")
    T = q.shape[0]
    for name, x, width in (("q", q, num_q_heads * head_dim), ("k", k, num_kv_heads * head_dim),
                           ("v", v, num_kv_heads * v_head_dim)):
        if tuple(x.shape) != (T, width) or x.dtype != q.dtype:
            raise ValueError(f"{name} is {tuple(x.shape)} {x.dtype}, expected {(T, width)} {q.dtype}")
    if qo_indptr.dim() != 1 or qo_indptr.numel() < 1 or qo_indptr.dtype != torch.int32:
        raise ValueError("qo_indptr must be an int32 vector of prompt bounds")
    if window < 0 or not sm_scale > 0:
        raise ValueError(f"window {window} and sm_scale {sm_scale}: a window of 0 (off) or more, a positive scale")
    if sinks is not None and sinks.numel() != num_q_heads:
        raise ValueError(f"{sinks.numel()} sinks for {num_q_heads} heads")
    if out is not None and tuple(out.shape) != (T, num_q_heads * v_head_dim):
        raise ValueError(f"out is {tuple(out.shape)}, expected {(T, num_q_heads * v_head_dim)}")
    r = prompt_attention_ref(q, k, v, qo_indptr, num_q_heads, num_kv_heads, head_dim, v_head_dim, window, sm_scale,
                             sinks).to(q.dtype)
    if out is not None:
        for a, b in zip(qo_indptr[:-1].tolist(), qo_indptr[1:].tolist()):
            out[a:b] = r[a:b]
        return out
    return r
