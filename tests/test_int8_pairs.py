"""The 8-bit product for many tokens (persistent CTA pairs): several tiles a pair, ragged edges in every direction, both
ways of storing, every output type, bias, residual, ``residual`` = ``out``, graphs. Tolerances as in test_int8."""

import pytest
import torch

from accerl_agent_b200 import ops
from test_int8 import check_product, product64, randn

pytestmark = pytest.mark.gpu

# M, K, N: whether TMA can store a contiguous bf16 result; 63 to 340 tiles for 74 pairs, a last group of one token block
SHAPES = [(4099, 520, 5000), (4097, 128, 4104), (4352, 40, 4096), (3000, 1024, 3000), (2300, 4096, 1536), (300, 1536, 20000),
          (2300, 4096, 1537), (4099, 4000, 4601), (2049, 1001, 1800)]


def operands(m, k, n, aligned=None, vec=None):
    """8-bit operands of a product that the pairs take (``aligned``: TMA can store the result)."""
    aligned = n % 8 == 0 if aligned is None else aligned
    assert ops._native_module().int8_plan(m, n, k, aligned, n % 4 == 0 if vec is None else vec) == (0, 1)
    r = ops.quantize_rows(randn(m, k, device="cuda"))
    w = ops.quantize_rows(randn(n, k, seed=1, device="cuda", scale=0.05))
    return r, w


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_pairs(m, k, n):
    r, w = operands(m, k, n)
    bias, res = randn(n, seed=2, device="cuda"), randn(m, n, seed=3, device="cuda")
    check_product(ops.linear_int8(r, w), *product64(r, w))
    check_product(ops.linear_int8(r, w, bias=bias, residual=res), *product64(r, w, bias, res))
    ops.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k,n", [(4099, 520, 5000), (2300, 4096, 1537)])
def test_pairs_types(dtype, m, k, n):
    """Each output type with bias and residual in 16 and 32 bits, and the residual that is the result itself."""
    r, w = operands(m, k, n)
    for kind in (torch.float32, torch.float16):
        bias, res = randn(n, seed=2, device="cuda", dtype=kind), randn(m, n, seed=3, device="cuda", dtype=kind)
        check_product(ops.linear_int8(r, w, bias, res, out_dtype=dtype), *product64(r, w, bias, res))
        check_product(ops.linear_int8(r, w, bias, out_dtype=dtype), *product64(r, w, bias))
    out = randn(m, n, seed=4, device="cuda", dtype=dtype)
    expect = product64(r, w, None, out)
    assert ops.linear_int8(r, w, residual=out, out=out) is not None
    check_product(out, *expect)


@pytest.mark.parametrize("lead,pad", [(0, 24), (8, 16), (3, 5)])
def test_pairs_strided(lead, pad):
    """Rows inside a wider buffer (16-byte aligned and not), nothing written around them, ``residual`` = ``out``."""
    m, k, n = 4099, 4000, 4104
    r, w = operands(m, k, n, lead % 8 == 0, lead % 8 == 0)
    buf = randn(m + 2, lead + n + pad, seed=4, device="cuda")
    before = buf.clone()
    view = buf[1 : m + 1, lead : lead + n]
    expect = product64(r, w, None, view)
    ops.linear_int8(r, w, residual=view, out=view)
    check_product(view, *expect)
    view.copy_(before[1 : m + 1, lead : lead + n])
    assert torch.equal(buf, before)


def test_pairs_extreme_sums_and_rows_without_values():
    m, k, n = 4099, 8960, 1300
    x = torch.ones(m, k, dtype=torch.bfloat16, device="cuda")
    x[1::2, ::2] = -1
    x[4098] = 0
    x[300, 7] = float("nan")
    wt = torch.ones(n, k, dtype=torch.bfloat16, device="cuda")
    wt[1::2] = -1
    wt[:, ::3] = 0.5
    wt[1299, 3] = float("inf")
    operands(m, k, n, True, True)  # fp32 rows of 1300 are aligned
    r, w = ops.quantize_rows(x), ops.quantize_rows(wt)
    y = ops.linear_int8(r, w, out_dtype=torch.float32)
    rows, cols = torch.arange(m, device="cuda") != 300, torch.arange(n, device="cuda") != 1299
    assert bool(y[300].isnan().all()) and bool(y[:, 1299].isnan().all()) and not y[4098][cols].any()
    y64, mag = product64(r, w)
    check_product(y[rows][:, cols], y64[rows][:, cols], mag[rows][:, cols])


def test_pairs_in_a_graph():
    m, k, n = 4099, 1536, 3000
    x, (_, w) = randn(m, k, device="cuda"), operands(m, k, n)
    eager = ops.linear_int8(x, w)
    check_product(eager, *product64(ops.quantize_rows(x), w))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.linear_int8(x, w)
    for seed in (0, 5, 6):
        x.copy_(randn(m, k, seed=seed, device="cuda"))
        g.replay()
        assert torch.equal(y, ops.linear_int8(x, w))
    assert not torch.equal(y, eager)
    ops.check_status(torch.device("cuda", 0))


def test_both_kernels_give_the_same_bits():
    """Products on either side of the plan's border: a row's result does not depend on how many rows there are."""
    k, n = 1536, 2048
    r, w = operands(4099, k, n)
    bias = randn(n, seed=2, device="cuda")
    whole = ops.linear_int8(r, w, bias)
    assert ops._native_module().int8_plan(70, n, k, True, True)[0] > 0
    for lo, hi in ((0, 1), (100, 170), (4090, 4099)):
        part = ops.linear_int8(ops.Int8Rows(r.q[lo:hi], r.scale[lo:hi], k), w, bias)
        assert torch.equal(part, whole[lo:hi])


@pytest.mark.parametrize("dtype,n,pitch", [(torch.bfloat16, 4103, 4104), (torch.bfloat16, 4097, 4104), (torch.float16, 4100, 4104),
                                           (torch.float32, 4101, 4104), (torch.float32, 4103, 4104), (torch.float32, 4102, 4108),
                                           (torch.bfloat16, 143, 144)])
def test_aligned_rows_that_end_inside_16_bytes(dtype, n, pitch):
    """Rows that start on 16 bytes but do not end there: nothing is written behind their ends."""
    for m, k in ((4099, 4000), (2128, 103), (70, 1536)):
        r = ops.quantize_rows(randn(m, k, device="cuda"))
        w = ops.quantize_rows(randn(n, k, seed=1, device="cuda", scale=0.05))
        bias = randn(n, seed=2, device="cuda")
        buf = torch.full((m + 1, pitch), 7.0, dtype=dtype, device="cuda")
        out = ops.linear_int8(r, w, bias, out=buf[:m, :n])
        check_product(out, *product64(r, w, bias))
        assert bool((buf[m] == 7).all()) and bool((buf[:, n:] == 7).all())


def test_calls_on_several_streams_at_once():
    """Both kernels, rows behind SwiGLU and the sampler on streams of their own at the same time: the bits of the calls made
    one after the other."""
    k, n = 1536, 4096
    x = randn(4099, k, device="cuda")
    w = ops.quantize_rows(randn(n, k, seed=1, device="cuda", scale=0.05))
    gu = randn(2048, 2 * 1544, seed=2, device="cuda", scale=2.0)
    logits = randn(60, 50000, seed=3, device="cuda", scale=2.0)
    u, t = torch.rand(60, device="cuda"), torch.full((60,), 0.9, device="cuda")
    calls = [lambda: ops.linear_int8(x, w), lambda: ops.linear_int8(x[:64], w), lambda: ops.linear_int8(x[:7], w),
             lambda: ops.swiglu_quantize(gu).q, lambda: torch.stack([a.double() for a in ops.sample_inverse_cdf(logits, u, t, top_p=t)])]
    expect = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    for _ in range(30):
        for i, (s, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[i].append(c())
    torch.cuda.synchronize()
    for e, results in zip(expect, got):
        assert all(torch.equal(e, r) for r in results)
    ops.check_status(torch.device("cuda", 0))
