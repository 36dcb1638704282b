"""Filters of sampled requests in captured decode steps: top-k, top-p and min-p, alone and side by side."""

import pytest
import torch

from accerl_agent_b200 import ops
from accerl_agent_b200.rollout.generation import SamplingParams
from test_engine_int8 import generate, int8_projections, make, recompute


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
