"""Sampling from given random numbers against a sort in 64 bits, written here from the definition.

Tokens are compared exactly: both sides hold the cumulative weights to about 1e-13 and the random numbers are
32-bit, so a difference would need a number within 1e-13 of a border. Log-probabilities are 64-bit values
rounded once to fp32 (2^-24 of the value) on either side.
"""

import math

import pytest
import torch

from accerl_agent_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def oracle_row(x, u, t, k=0, p=1.0, m=0.0):
    """(token, log-probability) of one row of Python floats."""
    live = [i for i, v in enumerate(x) if v > -math.inf]
    if not live:
        return 0, -math.inf
    live.sort(key=lambda i: (-x[i], i))
    top = x[live[0]]

    def weight(v, temp):
        if v == top:
            return 1.0
        return 0.0 if math.isinf(top) else math.exp((v - top) / temp)

    n = len(live) if k <= 0 else min(k, len(live))
    if not t > 0:
        n, t = 1, 1.0
    w = [weight(x[i], t) for i in live[:n]]
    if m > 0:
        while len(w) > 1 and not w[-1] >= m:
            w.pop()
    if p < 1:
        total, run, keep = math.fsum(w), 0.0, 0
        for v in w:
            if keep and not run < p * total:
                break
            run += v
            keep += 1
        w = w[:keep]
    target = min(max(u if u == u else 0.0, 0.0), 1 - 2.0 ** -53) * math.fsum(w)
    run, at = 0.0, None
    for j, v in enumerate(w):
        run += v
        if run > target:
            at = j
            break
    if at is None:
        at = max(j for j, v in enumerate(w) if v > 0)
    z = math.fsum(weight(v, 1.0) for v in x if v > -math.inf)
    gap = 0.0 if x[live[at]] == top else x[live[at]] - top
    return live[at], gap - math.log(z)


def check(logits, u, t, k=None, p=None, m=None):
    rows = logits.shape[0]
    tok, lp = ops.sample_inverse_cdf(logits, u, t, top_k=k, top_p=p, min_p=m)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32 and tok.shape == lp.shape == (rows,)
    xs = logits.double().tolist()
    for r in range(rows):
        et, el = oracle_row(xs[r], float(u[r]), float(t[r]), int(k[r]) if k is not None else 0,
                            float(p[r]) if p is not None else 1.0, float(m[r]) if m is not None else 0.0)
        assert int(tok[r]) == et, (r, int(tok[r]), et)
        got = float(lp[r])
        if el < -torch.finfo(torch.float32).max:  # beyond fp32: rounds to -inf
            el = -math.inf
        assert got == el or abs(got - el) <= 2.0 ** -23 * abs(el) + 1e-12, (r, got, el)
    return tok, lp


def full(rows, v, device, dtype=torch.float32):
    return torch.full((rows,), v, dtype=dtype, device=device)


def make(rows, v, device, dtype, seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g) * scale
    x[torch.arange(rows), torch.randint(0, v, (rows,), generator=g)] += 6
    return x.to(dtype).to(device), torch.rand(rows, generator=g).to(device), g


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,v", [(1, 1), (4, 2), (3, 7), (5, 8), (3, 33), (2, 1000), (40, 4097), (300, 257), (2, 32003),
                                    (160, 1024)])
def test_plain(device, dtype, rows, v):
    x, u, _ = make(rows, v, device, dtype)
    check(x, u, full(rows, 1.0, device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,v", [(24, 5003), (3, 70001)])
def test_every_filter_mixed(device, dtype, rows, v):
    x, u, g = make(rows, v, device, dtype, seed=rows)

    def pick(options, dt=torch.float32):
        return torch.tensor(options, dtype=dt)[torch.randint(0, len(options), (rows,), generator=g)].to(device)

    t = pick([0.0, -1.0, 0.3, 0.8, 1.0, 1.7])
    k = pick([-1, 0, 1, 2, 5, 50, 1000, v - 1, v, v + 5], torch.int32)
    p = pick([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 1.5])
    m = pick([0.0, 1e-9, 0.01, 0.3, 1.0, 2.0])
    off = full(rows, 1.0, device)
    check(x, u, t, k, p, m)
    check(x, u, off, k)
    check(x, u, off, None, p)
    check(x, u, off, None, None, m)
    check(x, u, t, k, None, m)
    check(x, u, t, None, p, m)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,v", [(1, 151936), (7, 151936), (40, 151936), (1, 524208), (1, 65528), (80, 65529), (160, 32000)])
def test_large_vocabularies(rows, v):
    """Cluster sizes from one CTA a row to eight; compared with the sort on the CPU path."""
    x, u, _ = make(rows, v, "cuda", torch.bfloat16, seed=v)
    t, p = full(rows, 0.9, "cuda"), full(rows, 0.97, "cuda")
    tok, lp = ops.sample_inverse_cdf(x, u, t, top_p=p)
    etok, elp = ops.sample_inverse_cdf(x.cpu(), u.cpu(), t.cpu(), top_p=p.cpu())
    assert torch.equal(tok.cpu(), etok)
    torch.testing.assert_close(lp.cpu(), elp, rtol=2.0 ** -23, atol=1e-12)
    tok1, _ = ops.sample_inverse_cdf(x, u, full(rows, 1.0, "cuda"))
    etok1, _ = ops.sample_inverse_cdf(x.cpu(), u.cpu(), full(rows, 1.0, "cpu"))
    assert torch.equal(tok1.cpu(), etok1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,v", [(160, 40001), (90, 140003), (5, 300007)])
@pytest.mark.parametrize("value", [0.5, -3.0, 0.0, 1000.0, 1e-13])
def test_every_place_of_long_rows(dtype, rows, v, value):
    """Rows of one value: the draw's number alone names the token, in every part of rows that start at any alignment
    (fp16 1000 and bf16 1e-13 lie outside the counters' window; fp16 rounds 1e-13 to zero)."""
    x = torch.full((rows, v), value, dtype=torch.float64).to(dtype).cuda()
    u = ((torch.arange(rows) + 0.5) / rows).float()
    u[0], u[-1] = 0.0, 1.0 - 2.0 ** -24
    tok, lp = ops.sample_inverse_cdf(x, u.cuda(), full(rows, 1.0, "cuda"))
    assert tok.tolist() == [int(float(n) * v) for n in u]  # a product below 2^53 of 24 and 19 bits: exact
    torch.testing.assert_close(lp.cpu(), full(rows, -math.log(v), "cpu"), rtol=2.0 ** -23, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,v", [(150, 40001), (80, 70003)])
def test_many_long_rows(dtype, rows, v):
    x, u, _ = make(rows, v, "cuda", dtype, seed=rows)
    t, p, k = full(rows, 0.9, "cuda"), full(rows, 0.97, "cuda"), full(rows, 500, "cuda", torch.int32)
    for kk, pp in ((None, None), (k, None), (None, p), (k, p)):
        tok, lp = ops.sample_inverse_cdf(x, u, t, top_k=kk, top_p=pp)
        etok, elp = ops.sample_inverse_cdf(x.cpu(), u.cpu(), t.cpu(), top_k=kk.cpu() if kk is not None else None,
                                           top_p=pp.cpu() if pp is not None else None)
        assert torch.equal(tok.cpu(), etok)
        torch.testing.assert_close(lp.cpu(), elp, rtol=2.0 ** -23, atol=1e-12)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_ties_go_to_the_lowest_index(device, dtype):
    """Equal logits (all of them; two values; zeros of both signs): the j-th of n equal tokens owns
    [j / n, (j + 1) / n)."""
    v = 600
    x = torch.zeros(6, v)
    x[1] = 3.5
    x[2, 100:] = 1.0
    x[3, ::2] = -0.0
    x[4, ::3] = -5.0
    x[5, :] = -0.0
    x[5, 7] = 0.0
    x = x.to(dtype).to(device)
    for uu in (0.0, 0.25, 0.5, 0.7501, 0.999999):
        tok, _ = check(x, full(6, uu, device), full(6, 1.0, device))
        assert int(tok[0]) == int(uu * v) or abs(uu * v - round(uu * v)) < 1e-3
        assert int(tok[3]) == int(tok[0]) == int(tok[1]) == int(tok[5])
    tok, _ = check(x, full(6, 0.99, device), full(6, 1.0, device), full(6, 10, device, torch.int32))
    assert tok[0] == 9 and tok[2] == 109 and tok[3] == 9
    tok, _ = check(x, full(6, 0.3, device), full(6, 0.0, device))
    assert tok.tolist() == [0, 0, 100, 0, 1, 0]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_masked_and_special_logits(device, dtype):
    inf, nan, big = float("inf"), float("nan"), torch.finfo(dtype).max
    rows = [
        [-inf] * 50,                          # nothing left
        [nan] * 50,
        [nan, -inf] * 25,
        [-inf] * 20 + [1.0] + [-inf] * 29,    # one left
        [inf] + [0.0] * 48 + [inf],           # two share the mass
        [-big] * 50,                          # masked with the type's lowest value, all alike
        [-big] * 49 + [2.0],
        [big, -big] * 25,
        [nan, 1.0] * 25,
        [torch.finfo(dtype).smallest_normal * i for i in range(50)],
        [-1e-4 * i for i in range(50)],
    ]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype).to(device)
    n = x.shape[0]
    for uu in (0.0, 0.4, 0.75, 0.9999999):
        for t in (0.0, 1e-30, 1.0, 50.0, inf):
            for p, m in ((None, None), (full(n, 0.6, device), full(n, 0.1, device))):
                check(x, full(n, uu, device), full(n, t, device), None, p, m)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [70, 9001])
def test_values_outside_the_usual_range(device, dtype, v):
    """Rows with logits that are tiny, huge, or masked with low numbers that do or do not weigh something:
    the kernel counts such values apart."""
    x, u, g = make(10, v, device, dtype, seed=11)
    x[0, 3] = 1e-13 if dtype == torch.bfloat16 else 90.0
    x[1] *= 1e-14 if dtype == torch.bfloat16 else 20.0
    x[2, ::2] = torch.finfo(dtype).min
    x[3, 1:] = torch.finfo(dtype).min
    x[4] = torch.finfo(dtype).min
    x[5, ::3] = -1e4
    x[6, ::5] = -70.0
    x[7, 5:9] = torch.finfo(dtype).max
    x[8, v // 2:] = float("inf")
    x[9, ::4] = -x[9].abs().max()
    t = full(10, 1.0, device)
    check(x, u, t)
    check(x, u, full(10, 300.0, device))  # -1e4 and -70 weigh something
    check(x, u, full(10, 1e5, device), full(10, v - 3, device, torch.int32))
    check(x, u, full(10, 0.7, device), full(10, 30, device, torch.int32), full(10, 0.9, device), full(10, 0.01, device))
    check(x, u, full(10, 0.0, device))


@pytest.mark.parametrize("device", DEVICES)
def test_numbers_outside_their_range(device):
    x, _, _ = make(1, 300, device, torch.bfloat16)
    x = x.expand(6, -1)
    nan = float("nan")
    u = torch.tensor([-1.0, 0.0, nan, 1.0, 2.0, 0.99999994], device=device)
    tok, _ = check(x, u, full(6, 1.0, device))
    assert tok[0] == tok[1] == tok[2] and tok[3] == tok[4]
    check(x, full(6, 0.5, device), full(6, 1.0, device), None, full(6, nan, device), full(6, nan, device))
    tok, _ = check(x, full(6, 0.5, device), full(6, nan, device))
    assert bool((tok == x[0].float().argmax()).all())


@pytest.mark.parametrize("device", DEVICES)
def test_strides(device):
    base, u, _ = make(6, 1100, device, torch.bfloat16)
    t = full(6, 1.0, device)
    for lo, hi in ((0, 1000), (1, 1000), (3, 1100), (8, 1009)):
        check(base[:, lo:hi], u, t)
    check(base[::2, 5:900], u[:3].contiguous(), t[:3].contiguous())
    assert ops.sample_inverse_cdf(base[:0], u[:0], t[:0])[0].shape == (0,)


@pytest.mark.parametrize("device", DEVICES)
def test_frequencies(device):
    """Numbers spread evenly over [0, 1) give every token its share to within one draw."""
    n, v = 4000, 20
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, v, generator=g).bfloat16().to(device).expand(n, -1)
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float().to(device)
    tok, _ = ops.sample_inverse_cdf(x, u, full(n, 0.7, device))
    share = torch.softmax(x[0].double() / 0.7, 0) * n  # temperature 0.7 in fp32 differs by 2^-25
    assert bool((torch.bincount(tok, minlength=v).double() - share).abs().max() <= 1.001)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_do_not_depend_on_the_batch(device):
    x, u, _ = make(9, 9000, device, torch.bfloat16)
    t, p = full(9, 0.8, device), full(9, 0.9, device)
    tok, lp = ops.sample_inverse_cdf(x, u, t, top_p=p)
    for r in (0, 4, 8):
        one = slice(r, r + 1)
        a, b = ops.sample_inverse_cdf(x[one], u[one], t[one], top_p=p[one])
        assert torch.equal(a, tok[one])
        torch.testing.assert_close(b, lp[one], rtol=2.0 ** -23, atol=0)


def test_refusals():
    x, u, _ = make(4, 30, "cpu", torch.bfloat16)
    t = full(4, 1.0, "cpu")
    for kw in ({"u": u[:3]}, {"u": u.double()}, {"temperature": t[:2]}, {"top_k": t}, {"top_p": t.double()},
               {"min_p": torch.stack([t, t], 1)[:, 0]}, {"logits": x[0]}, {"logits": x[:, :0]},
               {"logits": torch.zeros(30, 4).bfloat16().t()}):
        args = {"logits": x, "u": u, "temperature": t, **kw}
        with pytest.raises(ValueError):
            ops.sample_inverse_cdf(**args)


@pytest.mark.gpu
def test_refusals_gpu():
    x, u, _ = make(4, 30, "cuda", torch.bfloat16)
    t = full(4, 1.0, "cuda")
    with pytest.raises(ValueError, match="bf16 or fp16"):
        ops.sample_inverse_cdf(x.float(), u, t)
    with pytest.raises(ValueError, match="u must"):
        ops.sample_inverse_cdf(x, u.cpu(), t)


@pytest.mark.gpu
def test_in_a_graph_and_on_another_stream():
    x, u, _ = make(5, 50000, "cuda", torch.bfloat16)
    t, k = full(5, 0.9, "cuda"), full(5, 40, "cuda", torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = ops.sample_inverse_cdf(x, u, t, top_k=k)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tok, lp = ops.sample_inverse_cdf(x, u, t, top_k=k)
    g.replay()
    assert torch.equal(tok, eager[0]) and torch.equal(lp, eager[1])
    u.copy_(1 - u)
    t.fill_(1.4)
    g.replay()
    again = ops.sample_inverse_cdf(x, u, t, top_k=k)
    assert torch.equal(tok, again[0]) and torch.equal(lp, again[1])


@pytest.mark.gpu
def test_from_hidden_rows_to_tokens():
    """The last part of a decode step as the engine would run it: norm, 8-bit LM head, token."""
    rows, hidden, vocab = 24, 512, 5000
    g = torch.Generator().manual_seed(0)
    h = torch.randn(rows, hidden, generator=g).bfloat16().cuda()
    norm = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
    head = ops.quantize_rows((torch.randn(vocab, hidden, generator=g) * 0.2).bfloat16().cuda())
    u = torch.rand(rows, generator=g).cuda()
    x8 = ops.rmsnorm_quantize(h, norm, 1e-6)
    logits = ops.linear_int8(x8, head)
    assert torch.equal(logits.cpu(), ops.linear_int8(ops.Int8Rows(x8.q.cpu(), x8.scale.cpu(), hidden),
                                                     ops.Int8Rows(head.q.cpu(), head.scale.cpu(), hidden)))
    check(logits, u, full(rows, 0.8, "cuda"), full(rows, 30, "cuda", torch.int32), full(rows, 0.9, "cuda"),
          full(rows, 0.05, "cuda"))
