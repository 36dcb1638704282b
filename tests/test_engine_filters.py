"""Filters of sampled requests: top-k, top-p and min-p in captured decode steps, alone and side by side; min-p with tensor
parallelism and from the command line's options."""

import asyncio

import numpy as np
import pytest
import torch

from accerl_agent_b200 import ops
from accerl_agent_b200.core.config import make_args, validate_args
from accerl_agent_b200.models.config import get_preset
from accerl_agent_b200.models.transformer import build_model
from accerl_agent_b200.rollout.engine import GenerationEngine
from accerl_agent_b200.rollout.generation import SamplingParams, uniform_numbers
from accerl_agent_b200.rollout.inference import InferenceService, build_engine
from test_engine_int8 import PROMPTS, collect, generate, int8_projections, make, recompute


def prompts_of(cfg, n):
    g = torch.Generator().manual_seed(5)
    return [torch.randint(0, cfg.vocab_size, (9 + 7 * i,), generator=g).tolist() for i in range(n)]


def check_nucleus(m, prompt, o, temperature, top_p, noise=0.15):
    """The weights of the tokens that are above the sampled one by more than the logits' bf16 noise (as in the greedy
    tests: tilings differ) sum to less than ``top_p``."""
    logits = recompute(m, prompt + list(o.token_ids)).float()
    for j, t in enumerate(o.token_ids):
        row = logits[len(prompt) - 1 + j]
        w = torch.softmax(row / temperature, 0)
        assert w[row > row[t] + noise].sum() < top_p, (j, t)


@pytest.mark.gpu
@pytest.mark.parametrize("quantization", [None, "int8"])
def test_captured_steps_apply_top_k_and_top_p(monkeypatch, quantization):
    """At a temperature that makes 4096 tokens nearly equal: top-k 1 is the largest logit in every step, top-p 0.01 never
    leaves the nucleus (an unfiltered token lies in either by chance once in 4096 or 100), with min-p rows, plain rows
    and greedy rows in the same steps."""
    cfg, m, engine = make("cuda")
    base = dict(max_tokens=8, ignore_eos=True, logprobs=1)
    kinds = [dict(temperature=6.0, top_k=1), dict(temperature=6.0, top_p=0.01), dict(temperature=6.0, top_p=0.01, min_p=1e-9),
             dict(temperature=6.0), dict(temperature=0.0), dict(temperature=6.0, top_k=1, top_p=0.5)]
    prompts = prompts_of(cfg, 12)
    params = [SamplingParams(seed=40 + i, **kinds[i % 6], **base) for i in range(12)]
    eng = engine(use_cuda_graphs=True, quantization=quantization)
    outs = generate(eng, prompts, params)
    assert eng._graphs
    if quantization:
        int8_projections(monkeypatch, cfg)
    for p, q, o in zip(prompts, params, outs):
        assert len(o.token_ids) == 8
        if q.top_k == 1 or q.temperature == 0.0:
            check_nucleus(m, p, o, 6.0, 1e-12, 0.2)
        elif q.top_p < 1.0:
            check_nucleus(m, p, o, 6.0, 0.01, 0.2)


@pytest.mark.gpu
def test_rows_without_filters_draw_the_same_tokens_among_filtered_ones():
    g = torch.Generator().manual_seed(2)
    logits = (torch.randn(40, 4096, generator=g) * 2).bfloat16().cuda()
    temps = torch.full((40,), 1.3, device="cuda")
    seeds, offs = torch.arange(40, device="cuda") * 7 + 1, torch.arange(40, device="cuda")
    top_k = torch.tensor([0, 5, 0, 0] * 10, dtype=torch.int32, device="cuda")
    top_p = torch.tensor([1.0, 1.0, 0.3, 1.0] * 10, device="cuda")
    plain = ops.sample(logits, temps, seeds, offs)
    mixed = ops.sample(logits, temps, seeds, offs, top_k=top_k, top_p=top_p)
    off = (top_k == 0) & (top_p == 1.0)
    assert torch.equal(plain[0][off], mixed[0][off]) and torch.equal(plain[1][off], mixed[1][off])
    assert not torch.equal(plain[0], mixed[0])


@pytest.mark.gpu
def test_captured_min_p_rows_get_their_own_numbers(monkeypatch):
    """What reaches the operator in captured steps whose batch mixes min-p rows with others: each request's settings and
    the numbers of its seed and position; the tokens are those of the CPU form on the same logits, and come out."""
    cfg, m, engine = make("cuda")
    prompts = prompts_of(cfg, 10)
    base = dict(max_tokens=7, ignore_eos=True, logprobs=1)
    params = [SamplingParams(seed=70 + i, temperature=0.7 + 0.1 * i, top_p=0.6 + 0.03 * i, top_k=(0, 500)[i % 2],
                             min_p=(0.0, 0.01, 0.05)[i % 3], **base) for i in range(10)]
    real, seen = ops.sample_inverse_cdf, []

    def spy(logits, u, temperature, top_k=None, top_p=None, min_p=None):
        tok, lp = real(logits, u, temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        seen.append([a.clone() for a in (logits, u, temperature, top_k, top_p, min_p, tok, lp)])
        return tok, lp

    monkeypatch.setattr(ops, "sample_inverse_cdf", spy)
    eng = engine(use_cuda_graphs=True)
    outs = generate(eng, prompts, params)
    assert eng._graphs
    torch.cuda.synchronize()
    rows = [i for i in range(10) if i % 3]
    by_temp = {float(np.float32(params[i].temperature)): i for i in rows}
    got = {i: [] for i in rows}
    for logits, u, t, k, p, mp, tok, lp in [[a.cpu() for a in call] for call in seen]:
        etok, elp = real(logits, u, t, top_k=k, top_p=p, min_p=mp)
        assert torch.equal(tok, etok)
        torch.testing.assert_close(lp, elp, rtol=2.0 ** -23, atol=1e-12)
        for r in range(len(u)):
            i = by_temp[float(t[r])]
            q = params[i]
            assert float(p[r]) == float(np.float32(q.top_p)) and float(mp[r]) == float(np.float32(q.min_p))
            assert int(k[r]) == max(q.top_k, 0)
            assert float(u[r]) == uniform_numbers(np.array([70 + i]), np.array([len(got[i])]))[0]
            got[i].append((int(tok[r]), float(lp[r])))
    for i in rows:
        # a step more may be in flight when a request ends
        assert [a for a, _ in got[i]][:7] == list(outs[i].token_ids)
        assert [e[t] for e, t in zip(outs[i].logprobs, outs[i].token_ids)] == [b for _, b in got[i]][:7]


def _tp_rank(rank, port, q):
    """One of two ranks of a tensor-parallel engine that samples with min-p; the leader's outputs go to ``q``."""
    import os
    import traceback

    import torch.distributed as dist

    try:
        os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
        dist.init_process_group("gloo", rank=rank, world_size=2)
        cmd = dist.new_group(backend="gloo")
        cfg, m = tp_model()
        eng = GenerationEngine(cfg, torch.device("cpu"), torch.float32, max_num_seqs=8, max_num_batched_tokens=64,
                               num_blocks=64, block_size=4, tp_group=dist.group.WORLD, cmd_group=cmd)
        eng.set_weight_source(m.layout, tensor=m.params)
        if rank == 0:
            eng.pull_weights("all")

            async def run():
                outs = await asyncio.gather(*[collect(eng, p, s, f"r{i}") for i, (p, s) in enumerate(zip(PROMPTS, TP_PARAMS))])
                return [o.outputs[0].token_ids for o in outs]

            outs = asyncio.run(run())
            asyncio.run(eng.shutdown())
            eng.stop_followers()
            q.put(outs)
        else:
            eng.serve_follower()
        dist.destroy_process_group()
    except Exception:  # pragma: no cover
        q.put(traceback.format_exc())


TP_PARAMS = [SamplingParams(temperature=1.0 + 0.2 * i, seed=20 + i, min_p=0.02 * i, top_p=(1.0, 0.9)[i % 2], max_tokens=8,
                            ignore_eos=True, logprobs=1) for i in range(4)]


def tp_model():
    cfg = get_preset("tiny-qwen2")
    cfg.vocab_size = 512
    m = build_model(cfg, "full", torch.device("cpu"), torch.float32, with_grads=False)
    m.init_weights(seed=11, std=0.08)
    return cfg, m


def test_min_p_tensor_parallel_cpu():
    """Followers sample min-p rows as the leader does: were they not to, their next input tokens, and with them the sums
    over the ranks, would be others. Each token is the operator's on the recomputed logits."""
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
    got = queue.get(timeout=240)
    for p in procs:
        p.join(60)
    assert not isinstance(got, str), got
    cfg, m = tp_model()
    for i in (1, 2, 3):
        q, toks = TP_PARAMS[i], list(got[i])
        logits = recompute(m, PROMPTS[i] + toks)
        for j, t in enumerate(toks):
            u = torch.from_numpy(uniform_numbers(np.array([q.seed]), np.array([j])))
            row = logits[len(PROMPTS[i]) - 1 + j : len(PROMPTS[i]) + j]
            tok, _ = ops.sample_inverse_cdf(row, u, torch.tensor([q.temperature]), top_p=torch.tensor([q.top_p]),
                                            min_p=torch.tensor([q.min_p]))
            assert int(tok) == t, (i, j)


def test_options_reach_the_engine():
    """``--infer-quantization`` and ``--infer-min-p``: the service's engine quantises, its requests carry min-p, and with
    min-p 1 every token is the largest logit at any temperature."""
    args = make_args(model_path="tiny-qwen2", infer_quantization="int8", infer_min_p=1.0, infer_temperature=3.0)
    service = InferenceService(args, torch.device("cpu"))
    eng = service.engine
    assert eng.quantization == "int8" and service.runner.min_p == 1.0
    assert service.runner.sampling_kwargs(5)["min_p"] == 1.0
    eng.model.init_weights(seed=7, std=0.08)
    eng.weights_changed()

    async def run():
        res = await service.request_batch(PROMPTS[0], 6)
        greedy = await collect(eng, PROMPTS[0], SamplingParams(temperature=0.0, max_tokens=6, logprobs=1), "greedy")
        await eng.shutdown()
        return list(res.output_tokens), list(greedy.outputs[0].token_ids)

    sampled, greedy = asyncio.run(run())
    assert sampled == greedy and sampled
    plain = build_engine(make_args(model_path="tiny-qwen2"), torch.device("cpu"))
    assert plain.quantization is None
    with pytest.raises(ValueError, match="min-p"):
        args = make_args(model_path="tiny-qwen2", infer_min_p=1.5)
        validate_args(args, check_games=False)
