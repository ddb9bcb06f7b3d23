"""Edge cases of the prompt-scoring kernels against plain implementations in 64 bits; the tolerances are those that
test_prompt_scoring_gpu.py derives."""
import math

import pytest
import torch

from test_prompt_scoring_gpu import (DEV, U, _attend64, _check_attention, _check_head, _check_stats, _head, _indptr,
                                     _near, _qkv, _stats64)

pytestmark = pytest.mark.gpu


# ---- attention ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", [(2, 1, 128, 128), (3, 1, 64, 64), (2, 2, 192, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("jump", [12.0, 40.0, 90.0])
def test_prompt_attention_scores_jump_in_the_last_block(layout, dtype, jump):
    """The scores rise by 2^jump in weight in the last block of keys only: the output is rescaled right before it is
    read."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    Hq, Hkv, D, Dv = layout
    lens = [129, 256, 200, 300, 384, 100]
    q, k, v = (x.clone() for x in _qkv(sum(lens), Hq, Hkv, D, Dv, dtype, seed=int(jump)))
    q[:] = 1.0
    # scores in units of log 2: 0 before the last block, `jump` in it, a few units of noise
    k.mul_(0.25)
    at = 0
    for n in lens:
        last = at + (n - 1) // 128 * 128
        k[last:at + n] += jump * math.log(2.0) / math.sqrt(D)
        at += n
    out = prompt_attention(q, k, v, _indptr(lens), Hq, Hkv, D, v_head_dim=Dv)
    _check_attention(out, q, k, v, lens, Hq, Hkv, D, Dv)


def test_prompt_attention_scores_jump_beside_rows_without_a_score():
    """Rows of one warp whose first block holds only scores of -inf beside rows that are rescaled."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    n, Hq, Hkv, D = 384, 2, 1, 64
    q, k, v = (x.clone() for x in _qkv(n, Hq, Hkv, D, D, torch.bfloat16, seed=31))
    q[::2] = 1.0  # the first block's scores leave fp32's range
    q[1::2] = 2.0 ** -126  # -16 there, 0 elsewhere
    k[:128] = -(2.0 ** 127)
    k[128:] = k[128:] * 0.25
    k[256:] += 20 * math.log(2.0) / math.sqrt(D)
    out = prompt_attention(q, k, v, _indptr([n]), Hq, Hkv, D)
    want, A = _attend64(q, k, v, [n], Hq, Hkv, D, D, 0, D ** -0.5, None)
    tol = (2 * U[q.dtype] + 4e-4) * A + n * 2.0 ** -24 * v.float().abs().max().item()
    # in 64 bits the first block's scores stay finite: rows that see later keys compare
    assert ((out.double() - want).abs() <= tol)[128:].all()


@pytest.mark.parametrize("layout", [(4, 2, 64, 64), (3, 1, 128, 128), (2, 2, 192, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("huge", [1e4, 1e30, 3e38])
def test_prompt_attention_masked_values_weigh_nothing(layout, dtype, window, huge):
    """Huge finite values, which no recomputing of infinite results catches: rows that do not see them keep their
    bits, and so do rows beside tokens of no prompt."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    if dtype == torch.float16:
        huge = min(huge, 6e4)
    Hq, Hkv, D, Dv = layout
    lens = [100, 190, 150]
    T = sum(lens) + 40  # the last 40 tokens belong to no prompt
    q, k, v = (x.clone() for x in _qkv(T, Hq, Hkv, D, Dv, dtype, seed=9))
    ip = _indptr(lens)
    clean = prompt_attention(q, k, v, ip, Hq, Hkv, D, v_head_dim=Dv, window=window)[:sum(lens)]
    hit = torch.zeros(sum(lens), dtype=torch.bool, device=DEV)
    for t, end in ((30, 100), (100 + 77, 290), (290 + 149, 440)):
        v[t] = huge
        hit[t:min(end, t + window) if window else end] = True
    v[sum(lens):] = -huge
    out = prompt_attention(q, k, v, ip, Hq, Hkv, D, v_head_dim=Dv, window=window)[:sum(lens)]
    assert torch.equal(out[~hit], clean[~hit])


def test_prompt_attention_seen_scores_of_minus_infinity_weigh_nothing():
    """A key that scores -inf has weight 0 also where the row sees it, whatever finite value it holds."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    n, Hq, Hkv, D = 300, 2, 1, 64
    q, k, v = (x.clone() for x in _qkv(n, Hq, Hkv, D, D, torch.bfloat16, seed=12))
    q = q.abs() + 0.1
    clean_k, clean_v = k.clone(), v.clone()
    k[2::5], v[2::5] = -math.inf, 3e38
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    keep[2::5] = False
    out = prompt_attention(q, k, v, _indptr([n]), Hq, Hkv, D)
    # in 64 bits: the prompt without those keys, a row of it at every kept token
    s = torch.einsum("qhd,kd->hqk", q.double().view(n, Hq, D), clean_k.double()) * D ** -0.5
    t = torch.arange(n, device=DEV)
    s.masked_fill_((t[None, :] > t[:, None]) | ~keep[None, :], -math.inf)
    p = torch.softmax(s, -1)
    want = torch.einsum("hqk,kd->qhd", p, clean_v.double()).reshape(n, -1)
    A = torch.einsum("hqk,kd->qhd", p, clean_v.double().abs()).reshape(n, -1)
    assert ((out.double() - want).abs() <= (2 * U[q.dtype] + 4e-4) * A + 1e-6).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", [(2, 1, 64, 64), (1, 1, 128, 128), (2, 2, 192, 128)])
def test_prompt_attention_one_key_far_above_the_blocks_before_and_after(dtype, layout):
    """A key whose weight is up to 2^300 of the first block's, at every step around fp32's range, with lesser keys in
    the blocks behind it."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    Hq, Hkv, D, Dv = layout
    n = 420
    _, _, v = _qkv(n, Hq, Hkv, D, Dv, dtype, seed=41)
    q = torch.zeros(n, Hq * D, device=DEV, dtype=dtype)
    q.view(n, Hq, D)[..., :2] = 1.0
    jumps = [8.0, 17.0, 100.0, 300.0] + [120.0 + 0.25 * i for i in range(44)]
    for jump in jumps:
        t = torch.zeros(n, device=DEV, dtype=torch.float64)
        t[200], t[300] = jump, jump - 60.0
        t *= math.log(2.0) * math.sqrt(D)
        k = torch.zeros(n, Hkv, D, device=DEV, dtype=dtype)
        k[..., 0] = t.to(dtype)[:, None]
        k[..., 1] = (t - t.to(dtype).double()).to(dtype)[:, None]
        k = k.view(n, Hkv * D)
        out = prompt_attention(q, k, v, _indptr([n]), Hq, Hkv, D, v_head_dim=Dv)
        _check_attention(out, q, k, v, [n], Hq, Hkv, D, Dv)


def _odd_views(x):
    """The values of x in forms that tensor maps do not take as they are."""
    n, w = x.shape
    flat = torch.empty(n * w + 1, device=DEV, dtype=x.dtype)
    flat[1:] = x.reshape(-1)
    yield "contiguous, off the 16-byte boundaries", flat[1:].view(n, w)
    wide = torch.empty(n, w + 3, device=DEV, dtype=x.dtype)
    wide[:, :w] = x
    yield "a row stride of its own", wide[:, :w]
    yield "columns first", x.t().contiguous().t()


@pytest.mark.parametrize("T", [1, 37])
def test_prompt_attention_takes_any_rows(T):
    from sglang_neuron_b200.ops.prompt import prompt_attention
    Hq, Hkv, D = 4, 2, 64
    qkv = [x.contiguous() for x in _qkv(T, Hq, Hkv, D, D, torch.bfloat16)]
    ip = _indptr([T])
    want = prompt_attention(*qkv, ip, Hq, Hkv, D)
    for i in range(3):
        for what, view in _odd_views(qkv[i]):
            args = qkv[:i] + [view] + qkv[i + 1:]
            assert torch.equal(prompt_attention(*args, ip, Hq, Hkv, D), want), (i, what)
    # one row for all tokens
    k1, v1 = (x[:1].expand(T, -1) for x in qkv[1:])
    want = prompt_attention(qkv[0], k1.contiguous(), v1.contiguous(), ip, Hq, Hkv, D)
    assert torch.equal(prompt_attention(qkv[0], k1, v1, ip, Hq, Hkv, D), want)


def test_prompt_attention_output_rows():
    from sglang_neuron_b200.ops.prompt import prompt_attention
    Hq, Hkv, D = 4, 2, 64
    q, k, v = (x.contiguous() for x in _qkv(3, Hq, Hkv, D, D, torch.bfloat16))
    ip1, ip3 = _indptr([1]), _indptr([3])
    want = prompt_attention(q[:1], k[:1], v[:1], ip1, Hq, Hkv, D)
    # a single row's stride means nothing
    one = torch.zeros(1, Hq * D + 3, device=DEV, dtype=q.dtype)[:, :Hq * D]
    assert torch.equal(prompt_attention(q[:1], k[:1], v[:1], ip1, Hq, Hkv, D, out=one), want)
    flat = torch.zeros(3 * Hq * D + 1, device=DEV, dtype=q.dtype)
    for bad in (flat[1:].view(3, -1), flat[:Hq * D].expand(3, -1),
                torch.zeros(3, Hq * D + 3, device=DEV, dtype=q.dtype)[:, :Hq * D]):
        with pytest.raises(ValueError):
            prompt_attention(q, k, v, ip3, Hq, Hkv, D, out=bad)


# ---- log-probabilities from logits --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [1, 700])
@pytest.mark.parametrize("big", [1e6, 3e7, 1e9, 1e10, 1e15, 1e20, 1e30, 1e34])
def test_token_logprobs_large_finite_logits(dtype, N, big):
    """Masks of finite values between the ordinary and the type's lowest, and rows at such a level."""
    from sglang_neuron_b200.ops.logprobs import token_logprobs
    V = 30011
    g = torch.Generator(device=DEV).manual_seed(N)
    x = (torch.randn(N, V, device=DEV, generator=g) * 3).to(dtype)
    ids = torch.randint(0, V, (N,), device=DEV, generator=g)
    # long masked stretches before, between and after the ordinary logits; a lone ordinary logit at the end
    y = x.clone()
    y[:, :20000] = -big
    y[:, 20100:29000] = -big
    z = torch.full_like(x, -big)
    z[:, -1] = 1.5
    up = x.clone()
    up[:, 5000:5003] = big  # far above the rest
    for t, i in ((y, ids.clamp(29000, V - 1)), (y, ids), (z, ids), (up, torch.full_like(ids, 5001)), (up, ids)):
        _check_stats(token_logprobs(t, i, top_k=5), t, i, 5)
    for c in (big, -big):
        t = torch.full_like(x, c)
        _check_stats(token_logprobs(t, ids, top_k=32), t, ids, 32)
        t[:, 77] = c * 1.25
        _check_stats(token_logprobs(t, ids, top_k=3), t, ids, 3)


# ---- log-probabilities from hidden rows ---------------------------------------------------------------------
@pytest.mark.parametrize("N", [70, 300])
def test_head_logprobs_logits_of_minus_infinity_in_some_rows(N):
    """Columns whose logits are -inf for some rows of a warp and ordinary for the others."""
    from sglang_neuron_b200.ops.logprobs import head_logprobs
    H, V = 128, 1000
    h, w, ids = _head(N, H, V, torch.bfloat16, seed=N)
    low = torch.zeros(N, dtype=torch.bool, device=DEV)
    low[3::5] = True
    dark = torch.zeros(V, dtype=torch.bool, device=DEV)
    dark[32:64] = dark[100:420] = dark[999:] = True
    h[:, 0] = w[:, 0] = 0
    z = h.double() @ w.double().t()
    tol = 3e-4 + (H / 16 + 4) * 2.0 ** -23 * (h.double().abs() @ w.double().abs().t()).max().item()
    z[low[:, None] & dark[None, :]] = -math.inf
    h[low, 0], w[dark, 0] = -3e38, 3e38  # their product leaves fp32's range
    r = head_logprobs(h, w, ids)
    lp, ent, lse, _, _ = _stats64(z, ids, 0)
    assert _near(r.logprobs, lp, 2 * tol) and _near(r.lse, lse, tol)
    assert _near(r.entropy, ent, 3e-4 + 3e-6 * 128 + 8 * tol)


@pytest.mark.parametrize("N", [1, 50, 200])
@pytest.mark.parametrize("V", [1, 300])
def test_head_logprobs_takes_any_rows(N, V):
    from sglang_neuron_b200.ops.logprobs import head_logprobs
    h, w, ids = _head(N, 136, V, torch.bfloat16)
    want = head_logprobs(h, w, ids)
    cases = [(what, view, w) for what, view in _odd_views(h)] + [(what, h, view) for what, view in _odd_views(w)]
    cases += [("one row", h[:1].expand(N, -1), w)]
    for what, hh, ww in cases:
        ref = head_logprobs(hh.contiguous().clone(), w, ids) if what == "one row" else want
        for a, b in zip(head_logprobs(hh, ww, ids)[:3], ref[:3]):
            assert torch.equal(a, b), what


@pytest.mark.parametrize("N", [70, 129, 300, 1000])
@pytest.mark.parametrize("V", [1003, 8000, 9000, 10003, 12000, 15000])
def test_head_logprobs_forms_of_the_weight(N, V):
    """Both kernels (up to 128 rows, and more) at several tile widths: a vocabulary below the weight's rows with NaN
    behind it, tiles, strided rows, int32 ids, a shard's offset, a row of NaN."""
    from sglang_neuron_b200.ops.gemm import TiledWeight
    from sglang_neuron_b200.ops.logprobs import head_logprobs
    H = 200  # not a multiple of the 64 that a step of the contraction takes
    h, w, ids = _head(N, H, V + 97, torch.bfloat16, seed=V)
    ids = ids % V
    ids[0], ids[-1] = 0, V - 1
    w[V:] = math.nan
    want = head_logprobs(h, w[:V], ids)
    _check_head(want, h, w[:V], ids)
    wide_h = torch.zeros(N, H + 8, device=DEV, dtype=h.dtype)
    wide_h[:, 8:] = h
    wide_w = torch.zeros(V + 97, H + 24, device=DEV, dtype=w.dtype)
    wide_w[:, 16:16 + H] = w
    for hh, ww in ((h, w), (wide_h[:, 8:], w), (h, wide_w[:, 16:16 + H]), (h, TiledWeight(w)),
                   (wide_h[:, 8:], TiledWeight(w)), (h, TiledWeight(w, keep_rowmajor=True))):
        r = head_logprobs(hh, ww, ids.int(), valid_vocab=V)
        for a, b in zip(r[:3], want[:3]):
            assert torch.equal(a, b)
    for weight in (w, TiledWeight(w)):
        r = head_logprobs(h, weight, ids + 5000, vocab_offset=5000, valid_vocab=V)
        assert all(torch.equal(a, b) for a, b in zip(r[:3], want[:3]))
        for off in (5000 + V, -V):  # every id before or behind the shard
            r = head_logprobs(h, weight, ids, vocab_offset=off, valid_vocab=V)
            assert bool((r.logprobs == -math.inf).all()) and torch.equal(r.lse, want.lse)
            assert torch.equal(r.entropy, want.entropy)
        h2 = h.clone()
        h2[N // 2] = math.nan
        r = head_logprobs(h2, weight, ids, valid_vocab=V)
        keep = torch.arange(N, device=DEV) != N // 2
        for a, b in zip(r[:3], want[:3]):
            assert torch.equal(a[keep], b[keep]) and bool(torch.isnan(a[~keep]).all())
