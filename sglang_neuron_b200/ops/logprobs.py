"""Log-probabilities of given tokens with entropy, log-sum-exp and top alternatives: from a head's logits
(`token_logprobs`) or straight from the hidden rows and the head's weight (`head_logprobs`, which never stores the
logits).

Both describe the distribution at temperature 1 over the first `valid_vocab` columns; what later (padding) columns
hold does not matter. Forward only: results carry no gradient, on CUDA or CPU. With a vocabulary-sharded head every
rank calls them on its own shard with its first token id as `vocab_offset` and `merge_shards` joins the ranks' results.
Parity: the reference sampler's per-shard logsumexp and exact top-logprobs (sglang_neuron/sampling.py:212-470).
"""
from typing import NamedTuple

import torch

from .._ext import checked
from .gemm import TiledWeight, _status_buf

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """Per row: log-probability of the given id (-inf for an id outside this shard), entropy in nats, log-sum-exp
    of the logits, and the `top_k` best (log-probability, id) pairs, descending, ties to the lower id. A row whose
    logits are all -inf has log-probabilities of -inf and entropy 0; a row with a NaN or +inf logit has NaN."""
    logprobs: torch.Tensor       # [N] fp32
    entropy: torch.Tensor        # [N] fp32
    lse: torch.Tensor            # [N] fp32
    top_logprobs: torch.Tensor   # [N, top_k] fp32
    top_ids: torch.Tensor        # [N, top_k] int64


@torch.no_grad()
def token_logprobs_ref(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0, vocab_offset: int = 0,
                       valid_vocab: int = 0) -> TokenLogprobs:
    V = valid_vocab or logits.shape[1]
    x = logits[:, :V].to(torch.float64 if logits.dtype == torch.float64 else torch.float32)
    m = x.amax(-1, keepdim=True)
    none = (m == float("-inf"))[:, 0]
    y = x - torch.where(none[:, None], torch.zeros_like(m), m)
    e = torch.exp(y)
    s = e.sum(-1)
    log_s = torch.log(s)
    ey = torch.where(e == 0, torch.zeros_like(e), e * y)
    lse = torch.where(none, m[:, 0], m[:, 0] + log_s)
    entropy = torch.where(none, torch.zeros_like(s), log_s - ey.sum(-1) / s)
    local = ids.long() - vocab_offset
    own = (local >= 0) & (local < V) & ~none
    lp = y.gather(1, local.clamp(0, V - 1)[:, None])[:, 0] - log_s
    ninf = torch.full_like(lse, float("-inf"))
    tv, ti = torch.sort(x, dim=-1, descending=True, stable=True)
    tl = torch.where(none[:, None], ninf[:, None], (tv[:, :top_k] - m) - log_s[:, None])
    return TokenLogprobs(torch.where(own, lp, ninf), entropy, lse, tl, ti[:, :top_k] + vocab_offset)


def _check(rows: int, cols: int, ids: torch.Tensor, top_k: int, valid_vocab: int) -> int:
    V = valid_vocab or cols
    if not 0 < V <= cols:
        raise ValueError(f"valid_vocab {valid_vocab} outside the {cols} columns")
    if ids.dim() != 1 or ids.shape[0] != rows:
        raise ValueError(f"one id per row: {tuple(ids.shape)} ids for {rows} rows")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"ids must be int64 or int32, got {ids.dtype}")
    if not 0 <= top_k <= min(MAX_TOP, V):
        raise ValueError(f"top_k {top_k} outside [0, {min(MAX_TOP, V)}]")
    return V


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0, vocab_offset: int = 0,
                   valid_vocab: int = 0) -> TokenLogprobs:
    """`logits` [N, C] (bf16, fp16 or fp32 on CUDA; any row stride), `ids` [N]; see TokenLogprobs."""
    if logits.is_cuda:  # the kernel's entry checks its arguments (ValueError)
        return TokenLogprobs(*checked("token_logprobs", "logits_stats", logits, valid_vocab, ids, vocab_offset, top_k,
                                      _status_buf(logits.device)))
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, vocabulary], got {tuple(logits.shape)}")
    V = _check(logits.shape[0], logits.shape[1], ids, top_k, valid_vocab)
    return token_logprobs_ref(logits, ids, top_k, vocab_offset, V)


def head_logprobs(hidden: torch.Tensor, weight, ids: torch.Tensor, vocab_offset: int = 0,
                  valid_vocab: int = 0) -> TokenLogprobs:
    """The same of the logits `hidden @ weight.T`, which are kept in fp32 (never rounded, never stored). `hidden`
    [N, H] bf16 or fp16 on CUDA, `weight` [V, H] of the same type (a tensor or a TiledWeight), H a multiple of 8. Gives
    no alternatives: those need the logits (`token_logprobs`)."""
    tiled, F = False, 0
    if isinstance(weight, TiledWeight):
        if hidden.dim() != 2 or hidden.shape[1] != weight.K:
            raise ValueError(f"hidden {tuple(hidden.shape)} does not fit the weight {tuple(weight.shape)}")
        tiled, F = weight.rowmajor is None and hidden.is_cuda, weight.F
        weight = weight.data if tiled else weight.rowmajor if weight.rowmajor is not None else weight.untiled()
    if hidden.is_cuda:  # the kernel's entry checks its arguments (ValueError)
        lp, ent, lse = checked("head_logprobs", "head_stats", hidden, weight, F, tiled, valid_vocab, ids, vocab_offset,
                               _status_buf(hidden.device))
        return TokenLogprobs(lp, ent, lse, lp.new_empty(lp.shape[0], 0),
                             ids.new_empty(lp.shape[0], 0, dtype=torch.int64))
    if hidden.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} does not fit the weight {tuple(weight.shape)}")
    if hidden.dtype != weight.dtype:
        raise ValueError(f"hidden is {hidden.dtype}, the weight {weight.dtype}")
    V = _check(hidden.shape[0], weight.shape[0], ids, 0, valid_vocab)
    wide = torch.float64 if hidden.dtype == torch.float64 else torch.float32
    return token_logprobs_ref(hidden.to(wide) @ weight[:V].to(wide).t(), ids, 0, vocab_offset, V)


def merge_shards(shards) -> TokenLogprobs:
    """Joins the results of a vocabulary's shards (one TokenLogprobs per shard, in shard order)."""
    lse_i = torch.stack([s.lse for s in shards])                        # [S, N]
    lse = torch.logsumexp(lse_i, dim=0)
    none = lse == float("-inf")
    w = torch.exp(lse_i - torch.where(none, torch.zeros_like(lse), lse))  # a shard's share of the probability
    ninf = torch.full_like(lse, float("-inf"))
    # entropy of a mixture of disjoint shards: each shard's entropy plus what choosing the shard adds
    pick = torch.where(w > 0, w * (torch.stack([s.entropy for s in shards]) - (lse_i - lse)), torch.zeros_like(w))
    chosen = torch.stack([torch.where(s.lse == float("-inf"), ninf, s.logprobs + s.lse) for s in shards])
    k = shards[0].top_ids.shape[1]
    tv = torch.cat([s.top_logprobs + torch.where(s.lse == float("-inf"), torch.zeros_like(s.lse), s.lse)[:, None]
                    for s in shards], dim=1)
    ti = torch.cat([s.top_ids for s in shards], dim=1)
    # shards come in id order, so a stable sort keeps ties at the lower id
    order = torch.sort(tv, dim=1, descending=True, stable=True).indices[:, :k]
    tl = tv.gather(1, order) - torch.where(none, torch.zeros_like(lse), lse)[:, None]
    nan = lse != lse
    return TokenLogprobs(torch.where(none, ninf, torch.where(nan, lse, chosen.amax(0) - lse)),
                         torch.where(nan, lse, pick.sum(0)), lse, tl, ti.gather(1, order))
