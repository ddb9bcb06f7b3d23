"""Workloads of the prompt-scoring operators: attention over packed whole prompts, log-probabilities from logits,
and log-probabilities straight from hidden rows and the LM head's weight.

Each case is one pass of one operator at a shape that the served models or their tests have. `run` computes it in
a plain form (elementary torch operations in 32 bits) or, with `own` set, through the package's operators.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # eight chat-sized prompts of one scoring request, 16 / 8 heads: the launch and the tails count
        dict(name="attn_short", op="attention", lens="1,7,130,33,64,129,2,90", heads=16, kv_heads=8, dim=128,
             v_dim=128, window=0, sinks=False, dtype="bf16"),
        # one packed prefill step of documents of very different length, 32 / 8 heads, fp16 activations
        dict(name="attn_ragged", op="attention", lens="4096,2048,1025,513,511,77,1", heads=32, kv_heads=8, dim=128,
             v_dim=128, window=0, sinks=False, dtype="fp16"),
        # a sliding-window layer with learned sinks, 64 / 8 heads of 64: four prompts near 1024 tokens
        dict(name="attn_window", op="attention", lens="1024,1087,900,1056", heads=64, kv_heads=8, dim=64, v_dim=64,
             window=128, sinks=True, dtype="bf16"),
        # the full-attention layer of the same model on a long and a middling prompt
        dict(name="attn_sinks", op="attention", lens="4096,1500", heads=64, kv_heads=8, dim=64, v_dim=64, window=0,
             sinks=True, dtype="bf16"),
        # decompressed latent attention: 16 heads with keys of 192 and values of 128, no shared heads
        dict(name="attn_latent", op="attention", lens="4096,777", heads=16, kv_heads=16, dim=192, v_dim=128,
             window=0, sinks=False, dtype="bf16"),
        # one long document, 32 / 8 heads: the compute-bound end
        dict(name="attn_long", op="attention", lens="8192", heads=32, kv_heads=8, dim=128, v_dim=128, window=0,
             sinks=False, dtype="bf16"),
        # one sampled row with five alternatives: latency
        dict(name="logits_one", op="logits", rows=1, vocab=151936, valid=151936, top=5, dtype="bf16"),
        # a decode batch that returns the twenty alternatives an OpenAI client may ask for, fp32 logits
        dict(name="logits_decode", op="logits", rows=64, vocab=201088, valid=201088, top=20, dtype="fp32"),
        # a prompt's rows, five alternatives, head padded past the vocabulary
        dict(name="logits_prompt", op="logits", rows=4096, vocab=151936, valid=151669, top=5, dtype="bf16"),
        # a few short continuations scored against the whole vocabulary: the weight's stream
        dict(name="head_few", op="head", rows=33, hidden=2048, vocab=102400, valid=102400, dtype="bf16"),
        # a middling prompt, hidden size that is no power of two
        dict(name="head_mid", op="head", rows=1000, hidden=2880, vocab=201088, valid=201088, dtype="bf16"),
        # a packed scoring step: the product's rate
        dict(name="head_prompt", op="head", rows=4096, hidden=4096, vocab=151936, valid=151936, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "logits", "head"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "attention":
        heads, kv, dim, v_dim = rng.choice([(16, 8, 128, 128), (32, 8, 128, 128), (32, 4, 128, 128), (64, 8, 64, 64),
                                            (8, 1, 64, 64), (16, 16, 192, 128), (2, 2, 192, 128), (6, 2, 128, 128),
                                            (5, 5, 64, 64)])
        longest = _log_int(rng, 1, 6000)
        # the plain form's padded scores stay under those of the largest listed case
        most = max(1, min(48, int(32 * 8192 ** 2 / (heads * longest ** 2)), 8192 // longest))
        lens = [longest] + [rng.randint(1, longest) for _ in range(rng.randint(0, most - 1))]
        rng.shuffle(lens)
        return dict(op=op, lens=",".join(map(str, lens)), heads=heads, kv_heads=kv, dim=dim, v_dim=v_dim,
                    window=rng.choice([0, 0, 0, 128, _log_int(rng, 1, 2000)]), sinks=rng.random() < 0.3, dtype=dtype)
    if op == "logits":
        vocab = _log_int(rng, 1000, 201088)
        return dict(op=op, rows=_log_int(rng, 1, 3000), vocab=vocab, valid=vocab - rng.choice([0, 0, 1, 37, 64]),
                    top=rng.choice([0, 1, 2, 5, 8, 20, 32]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    vocab = _log_int(rng, 1000, 150000)
    return dict(op=op, rows=_log_int(rng, 1, 3000), hidden=8 * rng.randint(16, 512), vocab=vocab,
                valid=vocab - rng.choice([0, 0, 1, 64]), dtype=dtype)


def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


def prepare(case, seed):
    dev, dt = "cuda", DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    if case["op"] == "attention":
        lens = _lens(case)
        T, Hq, Hkv, D, Dv = sum(lens), case["heads"], case["kv_heads"], case["dim"], case["v_dim"]
        # the projection's output holds q, k and v of a token side by side: the operands are views with its stride
        qkv = torch.randn(T, Hq * D + Hkv * (D + Dv), device=dev, generator=g).to(dt)
        s["q"], s["k"], s["v"] = qkv.split([Hq * D, Hkv * D, Hkv * Dv], dim=1)
        ends = torch.tensor(lens, dtype=torch.int64).cumsum(0)
        s["indptr"] = torch.cat([ends.new_zeros(1), ends]).to(torch.int32).to(dev)
        s["longest"] = max(lens)
        s["sink"] = torch.randn(Hq, device=dev, generator=g) if case["sinks"] else None
    elif case["op"] == "logits":
        N, V = case["rows"], case["vocab"]
        # a head's logits: spread of a few units around each row's own level
        x = torch.randn(N, V, device=dev, generator=g)
        s["logits"] = (x.mul_(2.5) + torch.randn(N, 1, device=dev, generator=g)).to(dt)
        s["ids"] = torch.randint(0, case["valid"], (N,), device=dev, generator=g)
    else:
        N, H, V = case["rows"], case["hidden"], case["vocab"]
        # rows as the final norm leaves them, weights of a random-init head
        s["hidden_rows"] = torch.randn(N, H, device=dev, generator=g).to(dt)
        s["weight"] = (torch.randn(V, H, device=dev, generator=g) * 0.02).to(dt)
        s["ids"] = torch.randint(0, case["valid"], (N,), device=dev, generator=g)
    return s


def _plain_attention(s):
    """Softmax attention of every prompt with itself: the prompts padded to the longest, fp32 throughout."""
    Hq, Hkv, D, Dv, L = s["heads"], s["kv_heads"], s["dim"], s["v_dim"], s["longest"]
    indptr = s["indptr"].long()
    B, T, dev = indptr.numel() - 1, s["q"].shape[0], s["q"].device
    pos = torch.arange(L, device=dev)
    inside = pos[None, :] < (indptr[1:] - indptr[:-1])[:, None]  # [B, L]
    row = (indptr[:-1, None] + pos[None, :]).clamp(max=T - 1)
    q = s["q"].float().view(T, Hkv, Hq // Hkv, D)[row].permute(0, 2, 3, 1, 4)  # [B, Hkv, G, L, D]
    k = s["k"].float().view(T, Hkv, 1, D)[row].permute(0, 2, 3, 4, 1)  # [B, Hkv, 1, D, L]
    v = s["v"].float().view(T, Hkv, 1, Dv)[row].permute(0, 2, 3, 1, 4)  # [B, Hkv, 1, L, Dv]
    back = pos[:, None] - pos[None, :]
    seen = back >= 0
    if s["window"] > 0:
        seen = seen & (back < s["window"])
    score = torch.matmul(q, k).mul_(D ** -0.5)
    score.masked_fill_(~(seen & inside[:, None, :])[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].float().view(1, Hkv, -1, 1, 1)
        top = torch.maximum(top, sink)
    e = score.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - top)
    o = torch.matmul(e, v) / total
    return o.permute(0, 3, 1, 2, 4)[inside].reshape(T, Hq * Dv).to(s["q"].dtype)


def _plain_stats(x, ids):
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    entropy = lse - (e * x).sum(-1, keepdim=True) / total
    logprob = x.gather(1, ids[:, None]) - lse
    return logprob[:, 0], entropy[:, 0], lse[:, 0]


def run(s):
    if s["op"] == "attention":
        if own:
            from sglang_neuron_b200.ops.prompt import prompt_attention
            return prompt_attention(s["q"], s["k"], s["v"], s["indptr"], s["heads"], s["kv_heads"], s["dim"],
                                    v_head_dim=s["v_dim"], window=s["window"], sinks=s["sink"])
        return _plain_attention(s)
    if s["op"] == "logits":
        if own:
            from sglang_neuron_b200.ops.logprobs import token_logprobs
            r = token_logprobs(s["logits"], s["ids"], top_k=s["top"], valid_vocab=s["valid"])
            out = (r.logprobs, r.entropy, r.lse)
            return out + (r.top_logprobs, r.top_ids) if s["top"] else out
        x = s["logits"][:, :s["valid"]].float()
        logprob, entropy, lse = _plain_stats(x, s["ids"])
        if not s["top"]:
            return logprob, entropy, lse
        best, at = torch.sort(x, dim=-1, descending=True, stable=True)  # ties to the lowest id
        return logprob, entropy, lse, best[:, :s["top"]] - lse[:, None], at[:, :s["top"]].contiguous()
    if own:
        from sglang_neuron_b200.ops.logprobs import head_logprobs
        r = head_logprobs(s["hidden_rows"], s["weight"], s["ids"], valid_vocab=s["valid"])
        return r.logprobs, r.entropy, r.lse
    x = torch.matmul(s["hidden_rows"].float(), s["weight"][:s["valid"]].float().t())
    return _plain_stats(x, s["ids"])


def work(case):
    el = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        Hq, Hkv, D, Dv, w = case["heads"], case["kv_heads"], case["dim"], case["v_dim"], case["window"]
        T, pairs = 0, 0
        for n in _lens(case):
            T += n
            full = n if w <= 0 else min(n, w)
            pairs += full * (full + 1) // 2 + (n - full) * full
        return {"bytes": el * T * (Hq * (D + Dv) + Hkv * (D + Dv)), "flops": 2.0 * pairs * Hq * (D + Dv)}
    if case["op"] == "logits":
        N, V, k = case["rows"], case["valid"], case["top"]
        # per logit: subtract, exponential, two sums with a product
        return {"bytes": N * (V * el + 8 + 12 + 12 * k), "flops": 5.0 * N * V}
    N, H, V = case["rows"], case["hidden"], case["valid"]
    return {"bytes": el * H * (N + V) + 20 * N, "flops": 2.0 * N * H * V}


def exact(case, seed):
    """The operators' definitions in 64 bits, prompt by prompt and with torch's own log_softmax."""
    s = prepare(case, seed)
    if case["op"] == "attention":
        Hq, Hkv, D, Dv = case["heads"], case["kv_heads"], case["dim"], case["v_dim"]
        out, at = [], 0
        for n in _lens(case):
            q = s["q"][at:at + n].double().view(n, Hq, D).transpose(0, 1)
            k = s["k"][at:at + n].double().view(n, Hkv, D).transpose(0, 1)
            v = s["v"][at:at + n].double().view(n, Hkv, Dv).transpose(0, 1)
            heads = []
            for h in range(Hq):
                a = q[h] @ k[h * Hkv // Hq].t() / math.sqrt(D)
                t = torch.arange(n, device=a.device)
                dark = t[None, :] > t[:, None]
                if case["window"] > 0:
                    dark |= t[None, :] <= t[:, None] - case["window"]
                a[dark] = -math.inf
                if case["sinks"]:
                    a = torch.cat([a, s["sink"][h].double().expand(n, 1)], dim=1)
                heads.append(torch.softmax(a, dim=-1)[:, :n] @ v[h * Hkv // Hq])
            out.append(torch.stack(heads, dim=1).reshape(n, Hq * Dv))
            at += n
        return torch.cat(out)
    if case["op"] == "logits":
        x = s["logits"][:, :case["valid"]]
    else:
        x = None
    parts = []
    for r in range(0, case["rows"], 512):
        if x is not None:
            lp = torch.log_softmax(x[r:r + 512].double(), dim=-1)
            lse = x[r:r + 512, 0].double() - lp[:, 0]
        else:
            z = s["hidden_rows"][r:r + 512].double() @ s["weight"][:case["valid"]].double().t()
            lp = torch.log_softmax(z, dim=-1)
            lse = z[:, 0] - lp[:, 0]
        given = lp.gather(1, s["ids"][r:r + 512, None])[:, 0]
        row = [given, -(lp.exp() * lp).sum(-1), lse]
        if case["op"] == "logits" and case["top"]:
            row.append(lp.topk(case["top"], dim=-1).values)
        parts.append(row)
    out = tuple(torch.cat(p) for p in zip(*parts))
    if case["op"] == "logits" and case["top"]:
        out += (None,)
    return out
