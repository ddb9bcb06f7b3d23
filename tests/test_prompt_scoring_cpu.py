"""Prompt scoring on the CPU tier: the operators' PyTorch forms against independent ones, Engine.score against the
logits of the engine's own prefill steps for a dense, a sliding-window and a latent-attention model, and the
vocabulary-sharded run (TP = 2, gloo) against the whole."""
import math
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

from sglang_neuron_b200.configs import model_config as mc
from sglang_neuron_b200.engine import Engine
from sglang_neuron_b200.ops.logprobs import TokenLogprobs, head_logprobs, merge_shards, token_logprobs
from sglang_neuron_b200.ops.prompt import prompt_attention
from sglang_neuron_b200.parallel.state import destroy_parallel
from sglang_neuron_b200.server_args import ServerArgs

DENSE = dict(mc.PRESETS["qwen3-0.6b"], num_hidden_layers=2, vocab_size=1000, hidden_size=128, intermediate_size=256,
             num_attention_heads=4, num_key_value_heads=2, head_dim=32)
SINKS = dict(mc.PRESETS["gpt-oss-20b"], num_hidden_layers=2, vocab_size=500, hidden_size=128, intermediate_size=64,
             num_attention_heads=4, num_key_value_heads=2, head_dim=32, num_local_experts=4, num_experts_per_tok=2,
             sliding_window=8)
LATENT = dict(mc.PRESETS["deepseek-v2-lite"], num_hidden_layers=2, vocab_size=700, hidden_size=128,
              intermediate_size=256, moe_intermediate_size=64, n_routed_experts=4, num_experts_per_tok=2,
              num_attention_heads=2, kv_lora_rank=32, qk_nope_head_dim=16, qk_rope_head_dim=8, v_head_dim=16)


def _args(preset, **kw):
    mc.PRESETS["score-tiny"] = preset
    base = dict(model="score-tiny", device="cpu", dtype="float32", context_length=256, max_running_requests=4,
                chunked_prefill_size=64, random_weight_std=0.05)
    base.update(kw)
    return ServerArgs(**base)


def _prompts(vocab, lens=(9, 1, 30, 2, 17)):
    g = torch.Generator().manual_seed(4)
    return [torch.randint(1, vocab, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("window", [0, 1, 5])
@pytest.mark.parametrize("sinks", [False, True])
def test_prompt_attention_reference(window, sinks):
    g = torch.Generator().manual_seed(0)
    lens, Hq, Hkv, D, Dv = [3, 0, 11, 1], 4, 2, 6, 4
    T = sum(lens)
    q, k, v = (torch.randn(T, h * d, generator=g, dtype=torch.float64) for h, d in ((Hq, D), (Hkv, D), (Hkv, Dv)))
    sk = torch.randn(Hq, generator=g) if sinks else None
    ip = torch.tensor([0, 3, 3, 14, 15], dtype=torch.int32)
    out = prompt_attention(q, k, v, ip, Hq, Hkv, D, v_head_dim=Dv, window=window, sinks=sk)
    for b in range(4):
        for t in range(int(ip[b]), int(ip[b + 1])):
            lo = max(int(ip[b]), t - window + 1) if window else int(ip[b])
            for h in range(Hq):
                s = k[lo:t + 1, h // 2 * D:h // 2 * D + D] @ q[t, h * D:h * D + D] / math.sqrt(D)
                w = s.exp()
                den = w.sum() + (sk[h].double().exp() if sinks else 0)
                want = (w[:, None] * v[lo:t + 1, h // 2 * Dv:h // 2 * Dv + Dv]).sum(0) / den
                # the reference computes in fp32: a few roundings of values of order one
                assert (out[t, h * Dv:h * Dv + Dv] - want).abs().max() < 1e-5


def test_token_logprobs_reference():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 40, generator=g) * 3
    x[1, ::2] = -math.inf
    x[2] = -math.inf
    x[:, 37:] = math.nan
    ids = torch.tensor([0, 1, 2, 36, 50])
    r = token_logprobs(x, ids, top_k=4, valid_vocab=37)
    lp = torch.log_softmax(x[:, :37].double(), -1)
    for i in (0, 1, 3):
        assert abs(r.logprobs[i] - lp[i, ids[i]]) < 1e-5
    assert r.logprobs[4] == -math.inf and r.logprobs[2] == -math.inf and r.entropy[2] == 0
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    assert (r.entropy - ent)[[0, 1, 3, 4]].abs().max() < 1e-5
    assert torch.equal(r.top_ids[2], torch.arange(4))
    assert torch.equal(r.top_ids[0], lp[0].topk(4).indices)
    c = torch.zeros(2, 9)
    assert torch.equal(token_logprobs(c, torch.zeros(2, dtype=torch.long), top_k=3).top_ids, torch.arange(3).expand(2, 3))


def test_shards_merge_reference():
    g = torch.Generator().manual_seed(2)
    h, w = torch.randn(6, 16, generator=g), torch.randn(50, 16, generator=g)
    ids = torch.randint(0, 50, (6,), generator=g)
    x = h @ w.t()
    whole = token_logprobs(x, ids, top_k=5)
    shards = [token_logprobs(x[:, a:b], ids, top_k=5, vocab_offset=a) for a, b in ((0, 20), (20, 45), (45, 50))]
    m = merge_shards(shards)
    assert torch.equal(m.top_ids, whole.top_ids)
    for a, b in zip(m[:4], whole[:4]):
        assert (a - b).abs().max() < 1e-5
    hs = merge_shards([head_logprobs(h, w[a:b], ids, vocab_offset=a) for a, b in ((0, 20), (20, 50))])
    for a, b in zip(hs[:3], whole[:3]):
        assert (a - b).abs().max() < 1e-5
    # an empty shard changes nothing
    none = torch.full((6,), -math.inf)
    e = TokenLogprobs(none, torch.zeros(6), none, none[:, None].expand(6, 5), torch.zeros(6, 5, dtype=torch.long))
    m2 = merge_shards(shards + [e])
    assert torch.equal(m2.top_ids, whole.top_ids)
    for a, b in zip(m2[:4], m[:4]):
        assert (a - b).abs().max() < 1e-6


def test_operators_refuse():
    q = torch.zeros(4, 8)
    ip = torch.tensor([0, 4], dtype=torch.int32)
    for args, kw in [((q, q, q, ip, 3, 2, 4), {}), ((q, q[:3], q, ip, 2, 2, 4), {}),
                     ((q, q, q.half(), ip, 2, 2, 4), {}), ((q, q, q, ip.long(), 2, 2, 4), {}),
                     ((q, q, q, ip, 2, 2, 4), dict(sinks=torch.zeros(3))),
                     ((q, q, q, ip, 2, 2, 4), dict(sm_scale=-1.0)), ((q, q, q, ip, 2, 2, 4), dict(window=-1))]:
        with pytest.raises(ValueError):
            prompt_attention(*args, **kw)
    x, ids = torch.zeros(3, 10), torch.zeros(3, dtype=torch.long)
    for args, kw in [((x, ids[:2]), {}), ((x, ids), dict(top_k=11)), ((x, ids), dict(valid_vocab=11)),
                     ((x, ids.bool()), {}), ((x[0], ids), {})]:
        with pytest.raises(ValueError):
            token_logprobs(*args, **kw)
    with pytest.raises(ValueError):
        head_logprobs(x, torch.zeros(5, 9), ids)


def _oracle(eng, prompts, vocab):
    """Log-softmax rows of every prompt position, from single-request prefills through the paged path."""
    rows = {}
    for i, p in enumerate(prompts):
        got = []
        eng.runner.logits_hook = lambda fb, lg: got.append(lg[:, :vocab].double().clone())
        # each prefix is a request of its own: its last token's logits
        for n in range(1, len(p)):
            eng.generate([p[:n]], {"max_new_tokens": 1})
        rows[i] = torch.log_softmax(torch.cat(got), -1) if got else torch.zeros(0, vocab)
    eng.runner.logits_hook = None
    return rows


@pytest.mark.parametrize("preset", [DENSE, SINKS, LATENT], ids=["dense", "sinks", "latent"])
def test_engine_score_matches_prefill(preset):
    destroy_parallel()
    vocab = preset["vocab_size"]
    eng = Engine(_args(preset, disable_radix_cache=True))
    prompts = _prompts(vocab, (9, 1, 14, 2))
    want = _oracle(eng, prompts, vocab)
    plain = eng.score(prompts)
    top = eng.score(prompts, top_logprobs_num=3)
    assert "input_top_logprobs" not in plain[0]
    for i, (p, a, b) in enumerate(zip(prompts, plain, top)):
        for d in (a, b):
            assert d["prompt_tokens"] == len(p) and [t for _, t in d["input_token_logprobs"]] == p
            assert d["input_token_logprobs"][0][0] is None and d["input_entropies"][0] is None
            assert len(d["input_token_logprobs"]) == len(d["input_entropies"]) == len(p)
        lp = want[i]
        for n in range(1, len(p)):
            row = lp[n - 1]
            for d in (a, b):
                assert abs(d["input_token_logprobs"][n][0] - row[p[n]].item()) < 1e-3
                assert abs(d["input_entropies"][n] + (row.exp() * row).sum().item()) < 1e-3
            vals = [v for v, _ in b["input_top_logprobs"][n]]
            assert max(abs(v - w) for v, w in zip(vals, row.topk(3).values.tolist())) < 1e-3
        assert b["input_top_logprobs"][0] is None and len(b["input_top_logprobs"]) == len(p)


def test_engine_score_groups_and_refusals():
    """Packing into several forwards changes nothing; what cannot be scored is refused."""
    destroy_parallel()
    eng = Engine(_args(DENSE))
    prompts = _prompts(1000)
    one = eng.score(prompts, top_logprobs_num=2)
    eng.args.max_prefill_tokens = 20
    many = eng.score(prompts, top_logprobs_num=2)
    eng.runner.SCORE_ROWS = 3
    small = eng.score(prompts, top_logprobs_num=2)
    for a, b, c in zip(one, many, small):
        for x in (b, c):
            assert [t for _, t in a["input_token_logprobs"]] == [t for _, t in x["input_token_logprobs"]]
            assert all(abs(u[0] - v[0]) < 1e-4 for u, v in
                       zip(a["input_token_logprobs"][1:], x["input_token_logprobs"][1:]))
    assert eng.score([]) == []
    for bad, kw in [([[]], {}), ([[1, 1000]], {}), ([[-1, 3]], {}), ([[1] * 257], {}), ([[1, 2]], dict(top_logprobs_num=33)),
                    ([[1, 2]], dict(top_logprobs_num=-1)), (["text"], {})]:
        with pytest.raises(ValueError):
            eng.score(bad, **kw)
    # generation is untouched by scoring in between
    a = eng.generate([prompts[0]], {"max_new_tokens": 4})[0]["output_ids"]
    eng.score(prompts)
    assert eng.generate([prompts[0]], {"max_new_tokens": 4})[0]["output_ids"] == a


def _tp_run(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), WORLD_SIZE=str(world), RANK=str(rank),
                      LOCAL_RANK=str(rank))
    destroy_parallel()
    eng = Engine(_args(DENSE, tp_size=world))
    q.put((rank, (eng.score(_prompts(1000)), eng.score(_prompts(1000), top_logprobs_num=4))))
    if world > 1:
        import torch.distributed as dist
        dist.barrier()
        dist.destroy_process_group()


def _launch(world):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    ps = [ctx.Process(target=_tp_run, args=(r, world, port, q)) for r in range(world)]
    for p in ps:
        p.start()
    res = dict(q.get(timeout=300) for _ in ps)
    for p in ps:
        p.join(timeout=60)
    return res


def test_sharded_scores_equal_tp1():
    one, two = _launch(1)[0], _launch(2)
    assert two[0] == two[1]
    for a, b in zip(one, two[0]):
        for x, y in zip(a, b):
            assert all(abs(u[0] - v[0]) < 1e-4 and u[1] == v[1] for u, v in
                       zip(x["input_token_logprobs"][1:], y["input_token_logprobs"][1:]))
            assert all(abs(u - v) < 1e-4 for u, v in zip(x["input_entropies"][1:], y["input_entropies"][1:]))
            if "input_top_logprobs" in x:
                assert [[t for _, t in r] for r in x["input_top_logprobs"][1:]] == \
                       [[t for _, t in r] for r in y["input_top_logprobs"][1:]]


def test_kernel_entries_refuse_without_a_crash():
    """The compiled entries' own checks come back as exceptions (ValueError through the operators)."""
    from sglang_neuron_b200 import _ext
    if not _ext.available():
        pytest.skip("extension not built")
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    ids, st, ip = torch.zeros(4, dtype=torch.long), torch.zeros(4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for op, name, args in [("prompt_attention", "prompt_attention", (x, x, x, ip, 3, 2, 4, 4, 0, 0.1, None, None, st)),
                           ("token_logprobs", "logits_stats", (x, 99, ids, 0, 0, st)),
                           ("head_logprobs", "head_stats", (x, x, 0, False, 0, ids, 0, st))]:
        with pytest.raises(ValueError, match=op):
            _ext.checked(op, name, *args)
