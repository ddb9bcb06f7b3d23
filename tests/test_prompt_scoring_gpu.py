"""The prompt-scoring kernels against plain implementations in 64 bits.

Attention: an output is sum p v / sum p with p and the result each rounded once to the operand type (unit roundoff u:
2^-8 for bf16, 2^-11 for fp16) and everything else in fp32, exponentials within 2e-4; so its error is at most
(2 u + 4e-4) A + L 2^-24 max|v| with A = sum p |v| / sum p >= |out| and L the number of keys (the last term: weights
below the smallest fp16). Statistics: exponents carry an error of 2^-23 of their magnitude (at most 2^7 here), sums
at most 2^11 additions in a row: 3e-4 relative in a sum, so 3e-4 absolute in a log-sum-exp, and 2^-22 of the value.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


# ---- attention ---------------------------------------------------------------------------------------------
def _attend64(q, k, v, lens, Hq, Hkv, D, Dv, window, scale, sinks):
    """(out, A) in 64 bits, prompt by prompt; A is the same sum with |v|."""
    T = q.shape[0]
    out = torch.zeros(T, Hq, Dv, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    at = 0
    for n in lens:
        if n == 0:
            continue
        G = Hq // Hkv
        qs = q[at:at + n].double().reshape(n, Hq, D)
        ks = k[at:at + n].double().reshape(n, Hkv, D).repeat_interleave(G, 1)
        vs = v[at:at + n].double().reshape(n, Hkv, Dv).repeat_interleave(G, 1)
        s = torch.einsum("qhd,khd->hqk", qs, ks) * scale
        t = torch.arange(n, device=q.device)
        dark = t[None, :] > t[:, None]
        if window > 0:
            dark |= t[:, None] - t[None, :] >= window
        s.masked_fill_(dark, -math.inf)
        if sinks is not None:
            s = torch.cat([s, sinks.double()[:, None, None].expand(Hq, n, 1)], -1)
        p = torch.softmax(s, -1)[..., :n]
        out[at:at + n] = torch.einsum("hqk,khd->qhd", p, vs)
        bound[at:at + n] = torch.einsum("hqk,khd->qhd", p, vs.abs())
        at += n
    return out.reshape(T, -1), bound.reshape(T, -1)


def _qkv(T, Hq, Hkv, D, Dv, dtype, seed=0, mult=1.0, pad=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(T, Hq * D + Hkv * (D + Dv) + pad, device=DEV, generator=g) * mult).to(dtype)
    return x.split([Hq * D, Hkv * D, Hkv * Dv] + ([pad] if pad else []), dim=1)[:3]


def _indptr(lens, extra=0):
    t = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)
    return t.to(DEV)


def _check_attention(got, q, k, v, lens, Hq, Hkv, D, Dv, window=0, scale=None, sinks=None):
    scale = D ** -0.5 if scale is None else scale
    want, A = _attend64(q, k, v, lens, Hq, Hkv, D, Dv, window, scale, sinks)
    vmax = v.float().abs().max().item() if v.numel() else 0.0
    tol = (2 * U[q.dtype] + 4e-4) * A + max(lens) * 2.0 ** -24 * vmax + 1e-30
    n = sum(lens)
    worst = ((got.double() - want).abs() / tol)[:n].max().item()
    assert worst <= 1.0, f"error is {worst:.2f} of its bound"


LAYOUTS = [(16, 8, 128, 128), (8, 1, 64, 64), (4, 4, 192, 128), (6, 2, 128, 128), (5, 5, 64, 64), (3, 1, 192, 128)]
LENS = [[1], [2, 1, 3], [127, 128, 129], [256, 1, 255, 257], [300], [64] * 9, [0, 17, 0, 0, 130, 0]]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("lens", LENS, ids=lambda v: "-".join(map(str, v)))
def test_prompt_attention_layouts(layout, lens):
    from sglang_neuron_b200.ops.prompt import prompt_attention
    Hq, Hkv, D, Dv = layout
    q, k, v = _qkv(sum(lens), Hq, Hkv, D, Dv, torch.bfloat16, seed=len(lens))
    out = prompt_attention(q, k, v, _indptr(lens), Hq, Hkv, D, v_head_dim=Dv)
    assert out.dtype == torch.bfloat16 and out.shape == (sum(lens), Hq * Dv)
    _check_attention(out, q, k, v, lens, Hq, Hkv, D, Dv)


@pytest.mark.parametrize("window", [1, 2, 64, 127, 128, 129, 300, 100000])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_attention_window_sinks(window, sinks, D):
    from sglang_neuron_b200.ops.prompt import prompt_attention
    lens, Hq, Hkv = [700, 33, 128, 1, 513], 8, 2
    q, k, v = _qkv(sum(lens), Hq, Hkv, D, D, torch.bfloat16, seed=window)
    sk = torch.randn(Hq, device=DEV) * 3 if sinks else None
    out = prompt_attention(q, k, v, _indptr(lens), Hq, Hkv, D, window=window, sinks=sk)
    _check_attention(out, q, k, v, lens, Hq, Hkv, D, D, window=window, sinks=sk)


@pytest.mark.parametrize("mult", [1e-3, 1.0, 4.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_attention_magnitudes(dtype, mult):
    """From near-uniform weights to rows that one key rules; a scale of its own."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    lens, Hq, Hkv, D = [1500, 700], 4, 2, 128
    q, k, v = _qkv(sum(lens), Hq, Hkv, D, D, dtype, mult=mult)
    out = prompt_attention(q, k, v, _indptr(lens), Hq, Hkv, D, sm_scale=0.11)
    _check_attention(out, q, k, v, lens, Hq, Hkv, D, D, scale=0.11)


def test_prompt_attention_rising_scores():
    """Scores that grow along the row move the running maximum in every block."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    n, Hq, Hkv, D = 2000, 2, 1, 128
    q, k, v = _qkv(n, Hq, Hkv, D, D, torch.bfloat16, seed=5)
    ramp = torch.linspace(-40, 40, n, device=DEV)[:, None]
    k = (torch.ones_like(k) * ramp / 8).to(torch.bfloat16)
    q = torch.ones_like(q)
    for kk in (k, k.flip(0)):
        out = prompt_attention(q, kk, v, _indptr([n]), Hq, Hkv, D)
        _check_attention(out, q, kk, v, [n], Hq, Hkv, D, D)


def test_prompt_attention_many_prompts_and_gaps():
    from sglang_neuron_b200.ops.prompt import prompt_attention
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 200, (300,), generator=g).tolist()
    Hq, Hkv, D = 4, 2, 64
    T = sum(lens)
    q, k, v = _qkv(T, Hq, Hkv, D, D, torch.bfloat16)
    out = prompt_attention(q, k, v, _indptr(lens), Hq, Hkv, D)
    _check_attention(out, q, k, v, lens, Hq, Hkv, D, D)
    # tokens before the first and after the last prompt are nobody's: their rows stay as they are
    lens2 = [40, 200, 9]
    bounds = torch.tensor([30, 70, 270, 279], dtype=torch.int32, device=DEV)
    mark = torch.full((T, Hq * D), 7.0, device=DEV, dtype=torch.bfloat16)
    out = prompt_attention(q, k, v, bounds, Hq, Hkv, D, out=mark)
    assert out.data_ptr() == mark.data_ptr()
    assert bool((out[:30] == 7).all()) and bool((out[279:] == 7).all())
    _check_attention(out[30:279], q[30:279], k[30:279], v[30:279], lens2, Hq, Hkv, D, D)


@pytest.mark.parametrize("pad", [0, 8, 64])
def test_prompt_attention_strides(pad):
    """Views of a wider projection, rows that need a copy first, and an output with a row stride."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    lens, Hq, Hkv, D = [150, 61], 4, 2, 128
    T = sum(lens)
    q, k, v = _qkv(T, Hq, Hkv, D, D, torch.bfloat16, pad=pad)
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), _indptr(lens), Hq, Hkv, D)
    assert torch.equal(prompt_attention(q, k, v, _indptr(lens), Hq, Hkv, D), want)
    wide = torch.empty(T, Hkv * D + 3, device=DEV, dtype=torch.bfloat16)
    odd = wide[:, 3:]
    odd.copy_(k)
    assert torch.equal(prompt_attention(q, odd, v, _indptr(lens), Hq, Hkv, D), want)
    host = torch.zeros(T, Hq * D + 16, device=DEV, dtype=torch.bfloat16)
    out = prompt_attention(q, k, v, _indptr(lens), Hq, Hkv, D, out=host[:, 8:8 + Hq * D])
    assert torch.equal(out, want) and bool((host[:, :8] == 0).all()) and bool((host[:, 8 + Hq * D:] == 0).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_prompt_attention_masked_places_hold_anything(bad, where):
    """A NaN or infinity in a key or value reaches only the rows that see it: not earlier rows of its prompt, not
    the neighbouring prompts, not rows whose window has passed it."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    lens, Hq, Hkv, D, window = [100, 190, 150], 4, 2, 64, 50
    q, k, v = (x.clone() for x in _qkv(sum(lens), Hq, Hkv, D, D, torch.bfloat16, seed=9))
    clean = prompt_attention(q, k, v, _indptr(lens), Hq, Hkv, D, window=window)
    t = 100 + 77
    (k if where == "k" else v)[t, :D] = bad  # the first KV head: query heads 0 and 1
    out = prompt_attention(q, k, v, _indptr(lens), Hq, Hkv, D, window=window)
    hit = torch.zeros(sum(lens), Hq * D, dtype=torch.bool, device=DEV)
    hit[t:t + window, :2 * D] = True
    # rows that recompute without the tile's shared steps round their weights differently
    tol = (4 * U[torch.bfloat16] + 8e-4) * v.float()[~(v != v) & (v.abs() < 1e4)].abs().max().item()
    assert bool(torch.isfinite(out[~hit].float()).all())
    assert ((out.float() - clean.float()).abs()[~hit] <= tol).all()
    if math.isnan(bad):
        assert bool(torch.isnan(out[hit].float()).all())


def test_prompt_attention_no_tokens_and_refusals():
    from sglang_neuron_b200.ops.prompt import prompt_attention
    q, k, v = _qkv(10, 4, 2, 64, 64, torch.bfloat16)
    e = prompt_attention(q[:0], k[:0], v[:0], torch.zeros(1, dtype=torch.int32, device=DEV), 4, 2, 64)
    assert e.shape == (0, 256)
    ip = _indptr([10])
    for args, kw in [((q, k, v, ip, 4, 3, 64), {}), ((q, k[:9], v, ip, 4, 2, 64), {}),
                     ((q, k.half(), v, ip, 4, 2, 64), {}), ((q.float(), k.float(), v.float(), ip, 4, 2, 64), {}),
                     ((q, k, v, ip.long(), 4, 2, 64), {}), ((q, k, v, ip, 4, 2, 64), dict(sinks=torch.zeros(3))),
                     ((q, k, v, ip, 4, 2, 64), dict(out=torch.empty(9, 256, device=DEV, dtype=q.dtype))),
                     ((q, k, v, ip, 8, 4, 32), {})]:
        with pytest.raises(ValueError):
            prompt_attention(*args, **kw)


def test_prompt_attention_side_stream_and_graph():
    from sglang_neuron_b200.ops.prompt import prompt_attention
    lens, Hq, Hkv, D = [200, 64], 4, 2, 128
    q, k, v = _qkv(sum(lens), Hq, Hkv, D, D, torch.bfloat16)
    ip = _indptr(lens)
    want = prompt_attention(q, k, v, ip, Hq, Hkv, D)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = prompt_attention(q, k, v, ip, Hq, Hkv, D)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        prompt_attention(q, k, v, ip, Hq, Hkv, D, out=out)
    out.zero_()
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ---- log-probabilities from logits --------------------------------------------------------------------------
def _stats64(x, ids, top):
    x = x.double()
    lp = torch.log_softmax(x, -1)
    lse = torch.logsumexp(x, -1)
    ent = -torch.where(lp == -math.inf, torch.zeros_like(lp), lp.exp() * lp).sum(-1)
    _, idx = torch.sort(x, dim=-1, descending=True, stable=True)
    return lp.gather(1, ids[:, None])[:, 0], ent, lse, lp.gather(1, idx[:, :top]), idx[:, :top]


def _near(a, b, tol):
    a, b = a.double(), b.double()
    same = (a == b) | (torch.isnan(a) & torch.isnan(b))
    return bool((same | ((a - b).abs() <= tol + 2.0 ** -22 * b.abs())).all())


def _check_stats(r, x, ids, top, tol=3e-4, ids_too=True):
    lp, ent, lse, tl, ti = _stats64(x, ids, top)
    assert _near(r.logprobs, lp, tol) and _near(r.lse, lse, tol)
    # entropy adds the error of sum e y / s: the weights' relative error times the mean |y|
    assert _near(r.entropy, ent, tol + 3e-6 * 128)
    if top:
        assert _near(r.top_logprobs, tl, tol)
        if ids_too:
            assert torch.equal(r.top_ids, ti)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (3, 5, 5), (1, 33, 32), (2, 255, 20), (7, 1000, 8), (1, 32768, 1),
                                     (5, 100003, 5), (64, 151936, 20), (700, 5003, 32), (1, 201088, 32), (9, 4096, 0)])
def test_token_logprobs(dtype, N, V, top):
    from sglang_neuron_b200.ops.logprobs import token_logprobs
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (torch.randn(N, V, device=DEV, generator=g) * 3).to(dtype)  # 16-bit values tie often
    ids = torch.randint(0, V, (N,), device=DEV, generator=g)
    _check_stats(token_logprobs(x, ids, top_k=top), x, ids, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("off", [0, 1, 3, 7])
def test_token_logprobs_strides_and_padding(dtype, off):
    """Rows at every alignment, a row stride, and padding columns that hold NaN and infinities."""
    from sglang_neuron_b200.ops.logprobs import token_logprobs
    g = torch.Generator(device=DEV).manual_seed(off)
    wide = (torch.randn(6, 3001 + 13, device=DEV, generator=g) * 2).to(dtype)
    x = wide[:, off:off + 3005]
    V = 2999
    x[:, V] = math.nan
    x[:, V + 1:] = math.inf
    ids = torch.randint(0, V, (6,), device=DEV, generator=g)
    r = token_logprobs(x, ids.int(), top_k=9, valid_vocab=V)
    _check_stats(r, x[:, :V], ids, 9)
    t = token_logprobs(wide.t()[:100], torch.zeros(100, dtype=torch.long, device=DEV), top_k=2)
    _check_stats(t, wide.t()[:100], torch.zeros(100, dtype=torch.long, device=DEV), 2)


@pytest.mark.parametrize("N", [1, 700])
def test_token_logprobs_special_rows(N):
    from sglang_neuron_b200.ops.logprobs import token_logprobs
    V = 9001
    x = torch.randn(N, V, device=DEV)
    ids = torch.full((N,), 17, device=DEV)
    lo = torch.finfo(torch.float32).min
    # masked vocabularies: -inf or the type's lowest value in all but three places
    for fill in (-math.inf, lo):
        y = torch.full_like(x, fill)
        y[:, [4, 17, 8999]] = x[:, [4, 17, 8999]]
        r = token_logprobs(y, ids, top_k=5)
        _check_stats(r, y, ids, 5)
    # everything masked
    r = token_logprobs(torch.full_like(x, -math.inf), ids, top_k=3)
    assert bool((r.logprobs == -math.inf).all()) and bool((r.lse == -math.inf).all())
    assert bool((r.entropy == 0).all()) and bool((r.top_logprobs == -math.inf).all())
    assert torch.equal(r.top_ids, torch.arange(3, device=DEV).expand(N, 3))
    # constant rows tie everywhere: the lowest ids
    for c in (0.0, lo):
        y = torch.full_like(x, c)
        _check_stats(token_logprobs(y, ids, top_k=32), y, ids, 32)
    y = x.clone()
    y[:, ::2] = -0.0
    y[:, 1::2] = 0.0
    assert torch.equal(token_logprobs(y, ids, top_k=4).top_ids, torch.arange(4, device=DEV).expand(N, 4))
    # ascending and descending rows
    y = torch.arange(V, device=DEV).float().div(500).expand(N, V)
    for z in (y.contiguous(), y.flip(1).contiguous()):
        _check_stats(token_logprobs(z, ids, top_k=32), z, ids, 32)
    # a NaN or an infinity anywhere makes the row's results NaN
    for b in (math.nan, math.inf):
        y = x.clone()
        y[:, 5000] = b
        r = token_logprobs(y, ids, top_k=1)
        assert bool(torch.isnan(r.logprobs).all()) and bool(torch.isnan(r.entropy).all())
        assert bool((r.top_ids == 5000).all())
    # an id of another shard
    r = token_logprobs(x, torch.full((N,), V + 100, device=DEV), top_k=2, vocab_offset=100)
    assert bool((r.logprobs == -math.inf).all()) and int(r.top_ids.min()) >= 100
    r2 = token_logprobs(x, ids + 100, top_k=2, vocab_offset=100)
    assert torch.equal(r2.top_ids, r.top_ids) and bool(torch.isfinite(r2.logprobs).all())


def test_token_logprobs_one_thread_holds_all_the_best():
    """The best entries all in the columns that one thread reads."""
    from sglang_neuron_b200.ops.logprobs import token_logprobs
    V = 60000
    x = torch.randn(2, V, device=DEV).clamp(-3, 3)
    for i in range(40):
        x[:, i * 1024:i * 1024 + 4] = 10 + torch.rand(2, 4, device=DEV)
    ids = torch.zeros(2, dtype=torch.long, device=DEV)
    _check_stats(token_logprobs(x, ids, top_k=32), x, ids, 32)


def test_token_logprobs_long_batch_of_short_rows():
    """More rows than a grid axis holds."""
    from sglang_neuron_b200.ops.logprobs import token_logprobs
    x = torch.randn(70000, 24, device=DEV).to(torch.bfloat16)
    ids = torch.randint(0, 24, (70000,), device=DEV)
    _check_stats(token_logprobs(x, ids, top_k=3), x, ids, 3)


def test_token_logprobs_past_32_bit_offsets():
    """2^31 logits in one batch: the last rows lie past what 32 bits address."""
    from sglang_neuron_b200.ops.logprobs import token_logprobs
    V, N = 131072, 16500
    x = torch.zeros(N, V, device=DEV, dtype=torch.bfloat16)
    x[-2:] = torch.randn(2, V, device=DEV).to(torch.bfloat16)
    ids = torch.full((N,), V - 1, device=DEV)
    r = token_logprobs(x, ids, top_k=4)
    tail = type(r)(*(t[-2:] for t in r))
    _check_stats(tail, x[-2:], ids[-2:], 4)


def test_token_logprobs_refusals():
    from sglang_neuron_b200.ops.logprobs import token_logprobs
    x = torch.randn(4, 50, device=DEV)
    ids = torch.zeros(4, dtype=torch.long, device=DEV)
    for args, kw in [((x[0], ids), {}), ((x.double(), ids), {}), ((x, ids[:3]), {}), ((x, ids.float()), {}), ((x, ids), dict(top_k=33)),
                     ((x, ids), dict(top_k=-1)), ((x, ids), dict(valid_vocab=51)),
                     ((x, ids), dict(top_k=20, valid_vocab=10))]:
        with pytest.raises(ValueError):
            token_logprobs(*args, **kw)
    e = token_logprobs(x[:0], ids[:0], top_k=3)
    assert e.logprobs.shape == (0,) and e.top_ids.shape == (0, 3)


# ---- log-probabilities from hidden rows ---------------------------------------------------------------------
def _head(N, H, V, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randn(N, H, device=DEV, generator=g).to(dtype)
    w = (torch.randn(V, H, device=DEV, generator=g) * 0.03).to(dtype)
    return h, w, torch.randint(0, V, (N,), device=DEV, generator=g)


def _check_head(r, h, w, ids):
    # a logit is a sum of H exact products, added up in fp32 16 at a time: H / 16 + 4 roundings of its partial sums
    z = h.double() @ w.double().t()
    mag = (h.double().abs() @ w.double().abs().t()).max().item()
    tol = 3e-4 + (h.shape[1] / 16 + 4) * 2.0 ** -23 * mag
    lp, ent, lse, _, _ = _stats64(z, ids, 0)
    assert _near(r.logprobs, lp, 2 * tol) and _near(r.lse, lse, tol)
    assert _near(r.entropy, ent, 3e-4 + 3e-6 * 128 + 8 * tol)  # d entropy = sum p y dz, |y| a few units here


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,H,V", [(1, 64, 1), (1, 128, 257), (3, 8, 100), (33, 2048, 5000), (127, 200, 256),
                                   (128, 1024, 511), (129, 72, 513), (300, 576, 10003), (1000, 256, 777),
                                   (257, 2880, 20000)])
def test_head_logprobs(dtype, N, H, V):
    from sglang_neuron_b200.ops.logprobs import head_logprobs
    h, w, ids = _head(N, H, V, dtype, seed=N)
    _check_head(head_logprobs(h, w, ids), h, w, ids)


def test_head_logprobs_padding_offset_strides_tiled():
    from sglang_neuron_b200.ops.gemm import TiledWeight
    from sglang_neuron_b200.ops.logprobs import head_logprobs
    h, w, ids = _head(70, 192, 1100, torch.bfloat16)
    V = 1003
    ids = ids % V
    w[V:] = math.nan
    want = head_logprobs(h, w[:V], ids)
    _check_head(want, h, w[:V], ids)
    wide_h = torch.zeros(70, 192 + 8, device=DEV, dtype=h.dtype)
    wide_h[:, 4:196] = h
    for hh, ww in ((h, w), (wide_h[:, 4:196], w), (h, TiledWeight(w)), (h, TiledWeight(w, keep_rowmajor=True))):
        r = head_logprobs(hh, ww, ids.int(), valid_vocab=V)
        for a, b in zip(r[:3], want[:3]):
            assert torch.equal(a, b)
    r = head_logprobs(h, w, ids + 5000, vocab_offset=5000, valid_vocab=V)
    assert torch.equal(r.logprobs, want.logprobs)
    r = head_logprobs(h, w, ids, vocab_offset=5000, valid_vocab=V)
    assert bool((r.logprobs == -math.inf).all()) and torch.equal(r.lse, want.lse)
    # a row of NaN stays its own
    h2 = h.clone()
    h2[5] = math.nan
    r = head_logprobs(h2, w, ids, valid_vocab=V)
    keep = torch.arange(70, device=DEV) != 5
    assert torch.equal(r.lse[keep], want.lse[keep]) and bool(torch.isnan(r.lse[5])) and bool(torch.isnan(r.logprobs[5]))


def test_head_logprobs_refusals():
    from sglang_neuron_b200.ops.logprobs import head_logprobs
    h, w, ids = _head(4, 64, 100, torch.bfloat16)
    for args, kw in [((h, w[:, :32], ids), {}), ((h, w.half(), ids), {}), ((h.float(), w.float(), ids), {}),
                     ((h, w, ids[:2]), {}), ((h[:, :36], w[:, :36], ids), {}), ((h, w, ids), dict(valid_vocab=101))]:
        with pytest.raises(ValueError):
            head_logprobs(*args, **kw)
    assert head_logprobs(h[:0], w, ids[:0]).lse.shape == (0,)


def test_logprobs_shards_merge():
    """Two vocabulary shards joined equal the whole, for both operators."""
    from sglang_neuron_b200.ops.logprobs import head_logprobs, merge_shards, token_logprobs
    h, w, ids = _head(40, 256, 3000, torch.bfloat16)
    x = torch.nn.functional.linear(h, w)
    cuts = [(0, 1024), (1024, 3000)]
    whole = token_logprobs(x, ids, top_k=6)
    m = merge_shards([token_logprobs(x[:, a:b], ids, top_k=6, vocab_offset=a) for a, b in cuts])
    assert torch.equal(m.top_ids, whole.top_ids)
    for a, b in zip(m[:4], whole[:4]):
        assert _near(a, b, 1e-3)
    whole = head_logprobs(h, w, ids)
    m = merge_shards([head_logprobs(h, w[a:b], ids, vocab_offset=a) for a, b in cuts])
    for a, b in zip(m[:3], whole[:3]):
        assert _near(a, b, 1e-3)


def test_operators_agree():
    """Hidden rows to log-probabilities directly and through fp32 logits."""
    from sglang_neuron_b200.ops.logprobs import head_logprobs, token_logprobs
    h, w, ids = _head(50, 512, 4000, torch.bfloat16)
    a = head_logprobs(h, w, ids)
    b = token_logprobs(h.float() @ w.float().t(), ids)
    for x, y in zip(a[:3], b[:3]):
        assert _near(x, y, 1e-3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_attention_masked_scores_tower_over_seen_ones(dtype):
    """Keys that a row does not see score far above those that it sees: later tokens, and tokens behind the window."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    n, Hq, Hkv, D = 300, 2, 1, 64
    _, _, v = _qkv(n, Hq, Hkv, D, D, dtype, seed=21)
    q = torch.ones(n, Hq * D, device=DEV, dtype=dtype)
    for step, window in ((0.5, 0), (-0.5, 20), (4.0, 0), (-4.0, 7)):
        k = (torch.arange(n, device=DEV).float()[:, None] * step).expand(n, D).to(dtype).contiguous()
        out = prompt_attention(q, k, v, _indptr([n]), Hq, Hkv, D, window=window)
        _check_attention(out, q, k, v, [n], Hq, Hkv, D, D, window=window)


def test_prompt_attention_all_scores_minus_infinity():
    """Rows whose every score is -inf give zero, as the paged operators do; with a sink too."""
    from sglang_neuron_b200.ops.prompt import prompt_attention
    n, Hq, Hkv, D = 140, 2, 1, 64
    q, k, v = (x.clone() for x in _qkv(n, Hq, Hkv, D, D, torch.bfloat16, seed=22))
    q = q.abs() + 0.1
    k[:50] = -math.inf
    for sinks in (None, torch.zeros(Hq, device=DEV)):
        out = prompt_attention(q, k, v, _indptr([n]), Hq, Hkv, D, sinks=sinks)
        assert bool((out[:50] == 0).all()) and bool(torch.isfinite(out.float()).all())
        seen = prompt_attention(q[50:], k[50:], v[50:], _indptr([n - 50]), Hq, Hkv, D, sinks=sinks)
        tol = (4 * U[torch.bfloat16] + 8e-4) * v.float().abs().max().item()
        assert ((out[50:].float() - seen.float()).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N", [2, 600])
def test_token_logprobs_low_rows(dtype, N):
    """Rows near the type's lowest value, with a few logits above it, and with -inf beside it; huge positive rows."""
    from sglang_neuron_b200.ops.logprobs import token_logprobs
    V, lo = 5003, torch.finfo(dtype).min
    g = torch.Generator(device=DEV).manual_seed(N)
    ids = torch.randint(0, V, (N,), device=DEV, generator=g)
    step = 64.0 if dtype == torch.float16 else abs(lo) / 64
    x = torch.full((N, V), lo, device=DEV, dtype=dtype)
    x[:, ::7] = lo + step
    x[:, 1::9] = -math.inf
    _check_stats(token_logprobs(x, ids, top_k=4), x, ids, 4)
    x[:, 4000] = 0.5
    x[:, 17] = -1.25
    _check_stats(token_logprobs(x, ids, top_k=4), x, ids, 4)
    y = (torch.randn(N, V, device=DEV, generator=g) * 3).to(dtype)
    y[:, ::2] = lo
    y[:, 1::4] = -math.inf
    _check_stats(token_logprobs(y, ids, top_k=20), y, ids, 20)
    hi = torch.full((N, V), 6e4 if dtype == torch.float16 else 2e38, device=DEV, dtype=dtype)
    hi[:, ::3] = 1.0
    _check_stats(token_logprobs(hi, ids, top_k=2), hi, ids, 2)
