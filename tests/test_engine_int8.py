"""The rollout engine with 8-bit projections and with min-p: against a recomputation of whole sequences.

The recomputation runs the same model with every projection replaced by the 8-bit product of its rows, so both
sides make the same roundings to 8 bits except where the values before them differ (fp32 on the CPU: order of sums;
bf16 on the GPU: tilings of the attention).
"""

import asyncio
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from accerl_agent_b200 import ops
from accerl_agent_b200.models.config import ModelConfig, get_preset
from accerl_agent_b200.models.transformer import build_model
from accerl_agent_b200.rollout.engine import GenerationEngine
from accerl_agent_b200.rollout.generation import SamplingParams, uniform_numbers

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make(device, preset="tiny-qwen2", **kw):
    if device == "cpu":
        cfg, dtype = get_preset(preset), torch.float32
    else:
        cfg, dtype = ModelConfig(vocab_size=4096, hidden_size=256, num_hidden_layers=2, num_attention_heads=4,
                                 num_key_value_heads=2, head_dim=128, intermediate_size=512), torch.bfloat16
    m = build_model(cfg, "full", torch.device(device), dtype, with_grads=False)
    m.init_weights(seed=7, std=0.08 if device == "cpu" else 0.05)
    return cfg, m, lambda **more: GenerationEngine(cfg, torch.device(device), dtype, params=m.params, num_blocks=512,
                                                   block_size=16, **{**kw, **more})


async def collect(eng, prompt, params, rid):
    last = None
    async for out in eng.generate({"prompt_token_ids": prompt}, params, request_id=rid):
        last = out
    return last


def generate(eng, prompts, params):
    params = params if isinstance(params, list) else [params] * len(prompts)

    async def run():
        outs = await asyncio.gather(*[collect(eng, p, q, f"r{i}") for i, (p, q) in enumerate(zip(prompts, params))])
        await eng.shutdown()
        return outs

    return [o.outputs[0] for o in asyncio.run(run())]


def int8_projections(monkeypatch, cfg, tp=1):
    """Replace the layers' products by 8-bit ones (the LM head stays); with ``tp`` ranks a row-parallel weight
    (hidden_size rows) and its input are quantised shard by shard."""
    plain = ops.linear

    def linear(x, w, bias=None, residual=None, out=None):
        if w.shape[0] == cfg.vocab_size:
            return plain(x, w, bias, residual, out)
        if tp > 1 and w.shape[0] == cfg.hidden_size:
            parts = [ops.linear_int8(ops.quantize_rows(xs.contiguous()), ops.quantize_rows(ws.contiguous()),
                                     out_dtype=x.dtype) for xs, ws in zip(x.chunk(tp, 1), w.chunk(tp, 1))]
            return sum(parts) + residual
        return ops.linear_int8(ops.quantize_rows(x.contiguous()), ops.quantize_rows(w), bias, residual, out,
                               None if out is not None else x.dtype)

    def linear_swiglu(x, w, keep_gu=False):
        return ops.swiglu(linear(x, w)), None

    monkeypatch.setattr(ops, "linear", linear)
    monkeypatch.setattr(ops, "linear_swiglu", linear_swiglu)


def recompute(m, ids):
    ids = torch.tensor(ids, device=m.params.device)
    n = len(ids)
    logits = m.forward_logits_full(ids, torch.arange(n, device=ids.device),
                                   torch.tensor([0, n], dtype=torch.int32, device=ids.device), n)
    return logits


PROMPTS = [[5, 6, 7, 8, 9, 10, 11, 12, 13], [1, 2, 3], [5, 6, 7, 8, 9, 10, 11, 12, 40, 41], list(range(60, 95))]
GREEDY = SamplingParams(temperature=0.0, max_tokens=8, logprobs=1, ignore_eos=True)


def check_greedy(m, prompts, outs, tol):
    """Each token is the recomputation's largest logit given the tokens before it, with its log-probability, to
    within ``tol``. Logits have a spread of about 1 here.

    fp32 on the CPU, 0.05: a value whose 8-bit rounding falls to the other side moves a projection's output by one
    127th of one of its K products, about 1 / (127 sqrt(K)) < 1e-3 of the output's spread; with a few dozen such
    values among some hundred thousand, the logits move by less than a hundredth.

    bf16 on the GPU, 0.2: tilings of the attention move any of its outputs by a bf16 step, 2^-8 of the value, which is
    up to half of an 8-bit step (1 / 127 of the row's largest value), so up to half of a row's values may round to
    the other side. A row's largest value is about 4 standard deviations: K such steps of 4 / 127 with probability
    1/2 are sqrt(1/2) 4 / 127 = 2.2 % of the projection's output spread. Four projections in each of two layers
    that do so independently: 2.2 % sqrt(8) = 6 % at most, twice that for the difference of two logits."""
    for p, o in zip(prompts, outs):
        logp = torch.log_softmax(recompute(m, p + o.token_ids).float(), -1)
        for j, t in enumerate(o.token_ids):
            row = logp[len(p) - 1 + j]
            assert row[t] >= row.max() - tol and abs(o.logprobs[j][t] - row[t].item()) < tol


@pytest.mark.parametrize("preset", ["tiny-qwen2", "tiny-qwen2-moe"])
def test_int8_greedy_equals_recompute(monkeypatch, preset):
    """Whole prompts and chunks of 7 tokens (prefix caching on), the MoE model with its experts in fp32."""
    cfg, m, engine = make("cpu", preset)
    outs = generate(engine(quantization="int8"), PROMPTS, GREEDY)
    chunked = generate(engine(quantization="int8", max_num_batched_tokens=7), PROMPTS, GREEDY)
    plain = generate(engine(), PROMPTS, GREEDY)
    lp8 = [v for o in outs for e in o.logprobs for v in e.values()]
    lp = [v for o in plain for e in o.logprobs for v in e.values()]
    assert lp8 != lp  # the 8-bit path did run
    if not cfg.is_moe:
        int8_projections(monkeypatch, cfg)
        check_greedy(m, PROMPTS, outs, 0.05)
        check_greedy(m, PROMPTS, chunked, 0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
def test_int8_engine_gpu(monkeypatch, graphs):
    """Greedy choices and log-probabilities against the recomputation on the GPU, with and without graphs."""
    cfg, m, engine = make("cuda")
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, cfg.vocab_size, (20 + 37 * i,), generator=g).tolist() for i in range(9)]
    eng = engine(quantization="int8", use_cuda_graphs=graphs, max_num_batched_tokens=300)
    outs = generate(eng, prompts, GREEDY)
    assert bool(eng._graphs) == graphs
    int8_projections(monkeypatch, cfg)
    check_greedy(m, prompts, outs, 0.2)
    ops.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("device", DEVICES)
def test_weight_updates_renew_the_8_bit_copies(device):
    cfg, m, engine = make(device)
    eng = engine(quantization="int8")
    first = generate_without_shutdown(eng, PROMPTS[:2], "a")
    pointers = {n: w.q.data_ptr() for n, w in eng._w8.items()}
    other = build_model(cfg, "full", torch.device(device), m.params.dtype, with_grads=False)
    other.init_weights(seed=8, std=0.08)
    if device == "cuda":
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        eng.load_flat_weights(other.params, stream=side)
    else:
        eng.load_flat_weights(other.params)
    second = generate_without_shutdown(eng, PROMPTS[:2], "b")
    assert first != second
    for n, w in eng._w8.items():
        expect = ops.quantize_rows(other.w(n))
        assert torch.equal(w.q, expect.q) and torch.equal(w.scale, expect.scale)
        assert w.q.data_ptr() == pointers[n]  # captured graphs go on reading them
    eng.set_weight_source(other.layout, tensor=other.params)
    other.params.mul_(1.5)
    eng.pull_weights()
    generate_without_shutdown(eng, PROMPTS[:1], "c")
    name = "model.layers.0.self_attn.qkv_proj.weight"
    assert torch.equal(eng._w8[name].scale, ops.quantize_rows(other.w(name)).scale)
    asyncio.run(eng.shutdown())


def generate_without_shutdown(eng, prompts, tag):
    async def run():
        outs = await asyncio.gather(*[collect(eng, p, GREEDY, f"{tag}{i}") for i, p in enumerate(prompts)])
        return [(o.outputs[0].token_ids, [list(e.values()) for e in o.outputs[0].logprobs]) for o in outs]

    return asyncio.run(run())


def test_quantization_refusals():
    cfg, m, engine = make("cpu")
    with pytest.raises(ValueError, match="quantization"):
        engine(quantization="int4")


@pytest.mark.parametrize("device", DEVICES)
def test_min_p_rows(device):
    """min-p 1 leaves the largest logit whatever the temperature; a smaller one samples from the request's own
    numbers, alone or among rows without min-p, whose tokens do not change."""
    cfg, m, engine = make(device)
    graphs = {} if device == "cpu" else {"use_cuda_graphs": True}
    base = dict(max_tokens=6, ignore_eos=True, logprobs=1)
    best = generate(engine(**graphs), PROMPTS, SamplingParams(temperature=3.0, min_p=1.0, seed=1, **base))
    for p, o in zip(PROMPTS, best):
        logits = recompute(m, p + o.token_ids).float()
        for j, t in enumerate(o.token_ids):
            row = logits[len(p) - 1 + j]
            assert row[t] >= row.max() - (1e-4 if device == "cpu" else 0.1)
    mixed = [SamplingParams(temperature=1.0, seed=10 + i, min_p=0.0 if i % 2 else 0.05, top_k=0 if i < 2 else 20, **base)
             for i in range(4)]
    outs = generate(engine(**graphs), PROMPTS, mixed)
    if device == "cpu":
        for i, (p, o) in enumerate(zip(PROMPTS, outs)):
            if i % 2:
                continue
            logits = recompute(m, p + o.token_ids)
            for j, t in enumerate(o.token_ids):
                u = torch.from_numpy(uniform_numbers(np.array([10 + i]), np.array([j])))
                tok, lp = ops.sample_inverse_cdf(logits[len(p) - 1 + j : len(p) + j], u, torch.ones(1),
                                                 top_k=torch.tensor([20 if i >= 2 else 0], dtype=torch.int32),
                                                 min_p=torch.tensor([0.05]))
                assert int(tok) == t
                assert abs(float(lp) - o.logprobs[j][t]) < 1e-4
        again = generate(engine(), [PROMPTS[0]], mixed[0])
        assert again[0].token_ids == outs[0].token_ids
    else:
        # on the GPU the rows without min-p are bit for bit what they are in a batch without any
        for i in (1, 3):
            alone = [SamplingParams(temperature=1.0, seed=10 + j, top_k=0 if j < 2 else 20, **base) for j in range(4)]
        ref = generate(engine(**graphs), PROMPTS, alone)
        assert outs[1].token_ids == ref[1].token_ids and outs[3].token_ids == ref[3].token_ids
        assert all(len(o.token_ids) == 6 for o in outs)


def test_min_p_out_of_range_is_refused():
    _, _, engine = make("cpu")
    eng = engine()
    with pytest.raises(ValueError, match="min_p"):
        generate(eng, [[1, 2]], SamplingParams(min_p=1.5))


def test_uniform_numbers():
    """In [0, 1), a function of seed and position alone, evenly spread: of 4096 numbers every sixteenth of the
    range holds 256 +- 5 standard deviations (sqrt(240))."""
    seeds = np.repeat(np.arange(64, dtype=np.int64) * 977, 64)
    pos = np.tile(np.arange(64, dtype=np.int64), 64)
    u = uniform_numbers(seeds, pos)
    assert u.dtype == np.float32 and u.min() >= 0 and u.max() < 1 and len(np.unique(u)) > 4090
    assert np.array_equal(u[100:110], uniform_numbers(seeds[100:110], pos[100:110]))
    counts = np.histogram(u, 16, (0, 1))[0]
    assert np.abs(counts - 256).max() <= 5 * 240 ** 0.5


def _tp_rank(rank, port, q):
    """One of two ranks of a tensor-parallel engine with 8-bit shards; the leader's outputs, and those of a second
    pass after the weights changed, go to ``q``."""
    import os
    import traceback

    import torch.distributed as dist

    try:
        os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
        dist.init_process_group("gloo", rank=rank, world_size=2)
        cmd = dist.new_group(backend="gloo")
        cfg = get_preset("tiny-qwen2")
        cfg.vocab_size = 512
        m = build_model(cfg, "full", torch.device("cpu"), torch.float32, with_grads=False)
        m.init_weights(seed=11, std=0.08)
        eng = GenerationEngine(cfg, torch.device("cpu"), torch.float32, max_num_seqs=8, max_num_batched_tokens=64,
                               num_blocks=64, block_size=4, tp_group=dist.group.WORLD, cmd_group=cmd,
                               quantization="int8")
        eng.set_weight_source(m.layout, tensor=m.params)
        if rank == 0:
            results = []
            for scale in (1.0, 1.2):
                m.params.mul_(scale)
                eng.pull_weights("all")
                eng.allocator.clear_cache()  # keys and values of the old weights, as the service's pause clears them
                results.append([(o, lps) for o, lps in generate_without_shutdown(eng, PROMPTS[:2], f"t{scale}")])
            asyncio.run(eng.shutdown())
            eng.stop_followers()
            q.put(results)
        else:
            m.params.mul_(1.0)
            original = eng._pull_local

            def pull(scope, calls=[0]):
                if calls[0] == 1:
                    m.params.mul_(1.2)
                calls[0] += 1
                return original(scope)

            eng._pull_local = pull
            eng.serve_follower()
            name = "model.layers.0.mlp.down_proj.weight"
            expect = ops.quantize_rows(eng.model.w(name))
            q.put(bool(torch.equal(eng._w8[name].q, expect.q) and torch.equal(eng._w8[name].scale, expect.scale)))
        dist.destroy_process_group()
    except Exception:  # pragma: no cover
        q.put(traceback.format_exc())


def test_int8_tensor_parallel_cpu(monkeypatch):
    """Two ranks, each with its own shards in 8 bits (row-parallel weights get a scale per channel and shard), before
    and after a weight update, against the recomputation with the same shards."""
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    procs = [ctx.Process(target=_tp_rank, args=(r, port, queue)) for r in range(2)]
    for p in procs:
        p.start()
    got = [queue.get(timeout=240) for _ in procs]
    for p in procs:
        p.join(60)
    assert not any(isinstance(g, str) for g in got), [g for g in got if isinstance(g, str)]
    assert True in got  # the follower's copies follow its weights
    tp = next(g for g in got if isinstance(g, list))
    cfg = get_preset("tiny-qwen2")
    cfg.vocab_size = 512
    m = build_model(cfg, "full", torch.device("cpu"), torch.float32, with_grads=False)
    m.init_weights(seed=11, std=0.08)
    int8_projections(monkeypatch, cfg, tp=2)
    for scale, outs in zip((1.0, 1.2), tp):
        m.params.mul_(scale)
        got = [SimpleNamespace(token_ids=toks, logprobs=[{t: v[0]} for t, v in zip(toks, lps)]) for toks, lps in outs]
        check_greedy(m, PROMPTS, got, 0.05)
