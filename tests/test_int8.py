"""8-bit linear layers: rows to int8 and their products, against plain implementations in 64 bits.

Tolerances. The whole numbers are decided exactly, so they are equal. A product's only errors are five fp32
roundings (the accumulator's conversion, the product of the scales, the scaling, bias and residual), each at
most 2^-24 of the largest term, and the final rounding, at most eps/2 of the result.
"""

import pytest
import torch

from accerl_agent_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def quantize64(x):
    """(q, scale, finite) in 64 bits."""
    xd = x.double()
    a = xd.abs().amax(1, keepdim=True)
    ok = torch.isfinite(a)
    q = torch.round(127.0 * xd / torch.where(ok & (a > 0), a, torch.ones_like(a)))
    q = torch.where(ok, q, torch.zeros_like(q))
    return q, torch.where(ok, a / 127.0, torch.full_like(a, float("nan"))).squeeze(1), ok.squeeze(1)


def check_rows(x, r):
    q, scale, ok = quantize64(x)
    k = x.shape[1]
    assert r.shape == (x.shape[0], k) and r.q.shape[1] == (k + 15) // 16 * 16
    assert torch.equal(r.q[:, :k].double(), q)
    assert not r.q[:, k:].any()
    # one rounding of the quotient; below fp32's normal range half a subnormal step
    err = (r.scale[ok].double() - scale[ok]).abs()
    assert bool((err <= scale[ok] * 2.0 ** -24 + 2.0 ** -150).all())
    assert bool(r.scale[~ok].isnan().all())


def product64(r, w, bias=None, residual=None):
    """(y, magnitude of the largest term) in 64 bits."""
    y = (r.q.double() @ w.q.double().t()) * r.scale.double().unsqueeze(1) * w.scale.double().unsqueeze(0)
    mag = y.abs()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    if residual is not None:
        y, mag = y + residual.double(), mag + residual.double().abs()
    return y, mag


def check_product(y, y64, mag):
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps  # half a subnormal step and more
    tol = torch.finfo(y.dtype).eps / 2 * y64.abs() + 6 * 2.0 ** -24 * mag + tiny
    over = y64.abs() > torch.finfo(y.dtype).max
    assert bool((((y.double() - y64).abs() <= tol) | over).all())


def randn(*shape, seed=0, device="cpu", dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(device)


# ------------------------------------------------------------------------------------------------
# rows to 8 bits
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 1536), (3, 7), (5, 8), (7, 24), (130, 1001), (33, 8960), (2, 16400),
                                    (2, 40000), (0, 64), (6001, 256), (2500, 1544), (700, 8960), (5000, 24), (800, 32768)])
def test_quantize_rows(device, dtype, rows, k):
    x = randn(rows, k, device=device, dtype=dtype)
    check_rows(x, ops.quantize_rows(x))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_rows_borders(device, dtype):
    """Every quotient of significands, so every tie between two whole numbers, at every distance below the
    maximum that rounds to something."""
    bits = 8 if dtype == torch.bfloat16 else 11
    step = 1 if dtype == torch.bfloat16 else 9
    lo, hi = 1 << (bits - 1), 1 << bits
    a = torch.arange(lo, hi, step, dtype=torch.float64)
    m = torch.arange(lo, hi, dtype=torch.float64)
    x = torch.cat([m * 2.0 ** -e for e in range(10)])
    x = torch.cat([x, -x]).unsqueeze(0).expand(a.numel(), -1).clone()
    x = torch.where(x.abs() <= a.unsqueeze(1), x, torch.zeros_like(x))
    x[:, 0] = a
    x = (x * 2.0 ** -7).to(dtype)
    check_rows(x.to(device), ops.quantize_rows(x.to(device)))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_rows_extremes(device, dtype):
    """Zeros, subnormals, the largest values, infinities and NaN: each row by itself."""
    fi = torch.finfo(dtype)
    tiny = fi.smallest_normal * fi.eps  # the smallest subnormal
    x = torch.zeros(9, 40, dtype=torch.float64)
    x[1] = torch.arange(40) * tiny
    x[2] = torch.linspace(-1, 1, 40) * fi.smallest_normal
    x[3] = torch.linspace(-1, 1, 40) * fi.max
    x[4, 3] = float("inf")
    x[5, 39] = float("-inf")
    x[6] = 1.0
    x[6, 0] = float("nan")
    x[7, 5] = -tiny
    x[8] = -1.0
    for width in (40, 37):  # 16-byte accesses, single elements
        xs = x[:, 40 - width:].to(dtype).to(device)
        check_rows(xs, ops.quantize_rows(xs))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,stride", [(1, 5), (6, 6), (9, 20), (257, 263), (1001, 1001), (2056, 2063), (4100, 4111)])
def test_quantize_rows_at_every_alignment(device, dtype, k, stride):
    """Rows that start anywhere between 16-byte boundaries, NaN all around them."""
    rows = 11
    for first in range(9):
        flat = torch.full((first + rows * stride + 8,), float("nan"), dtype=dtype, device=device)
        x = flat.as_strided((rows, k), (stride, 1), first)
        x.copy_(randn(rows, k, seed=first, device=device, dtype=dtype))
        check_rows(x, ops.quantize_rows(x))


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_rows_strides_and_out(device):
    base = randn(12, 200, device=device)
    for x in (base[:, 8:72], base[:, 3:80], base[::2, :64], base[2:3].expand(4, -1), base[:, :1]):
        check_rows(x, ops.quantize_rows(x))
    out = ops.Int8Rows(torch.full((12, 208), 77, dtype=torch.int8, device=device), torch.zeros(12, device=device), 200)
    assert ops.quantize_rows(base, out=out) is out
    check_rows(base, out)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,k", [(1, 8), (5, 128), (64, 1536), (9, 4104), (3, 16384), (0, 64), (6001, 200), (2500, 1544),
                                    (701, 8960), (2, 32768), (4000, 8960), (30000, 136)])
def test_swiglu_quantize_is_the_two_calls(device, rows, k):
    gu = randn(rows, 2 * k, device=device, scale=2.0)
    if rows > 4:
        gu[1] *= 40  # gates far into the saturated range
        gu[2, 3], gu[3, 5] = float("inf"), float("nan")
    r = ops.swiglu_quantize(gu)
    check_rows(ops.swiglu(gu), r)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,k", [(1, 8), (5, 128), (64, 1536), (9, 4104), (3, 16384), (0, 64), (6001, 200), (2500, 1544),
                                    (701, 8960), (2, 32768)])
def test_rmsnorm_quantize(device, rows, k):
    """Against the norm in 64 bits: the two bf16 roundings may each fall to the other side (2^-8 of the
    value each), the maximum likewise, and the rounding to whole numbers is half a step."""
    x = randn(rows, k, device=device, scale=3.0)
    w = (1 + 0.1 * randn(k, seed=1, device=device, dtype=torch.float32)).bfloat16()
    r = ops.rmsnorm_quantize(x, w, 1e-6)
    assert not r.q[:, k:].any()
    xd = x.double()
    y = xd * torch.rsqrt(xd.pow(2).mean(1, keepdim=True) + 1e-6) * w.double()
    a = y.abs().amax(1, keepdim=True)
    tol = y.abs() * 2.0 ** -6.9 + a * 2.0 ** -6.9 / 127 + 0.5 * a / 127 * (1 + 2.0 ** -6.9) + 1e-6
    assert bool(((r.dequantize().double() - y).abs() <= tol).all())
    assert bool((r.q[:, :k].abs().amax(1) == 127).all())


@pytest.mark.parametrize("device", DEVICES)
def test_rmsnorm_quantize_empty_rows(device):
    x = torch.zeros(3, 64, dtype=torch.bfloat16, device=device)
    x[1, 5] = float("inf")
    r = ops.rmsnorm_quantize(x, torch.ones(64, dtype=torch.bfloat16, device=device), 1e-6)
    assert r.scale[0] == 0 and r.scale[2] == 0 and bool(r.scale[1].isnan()) and not r.q.any()


# ------------------------------------------------------------------------------------------------
# products
# ------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 16, 128), (1, 1536, 2048), (2, 17, 3), (15, 129, 130), (16, 128, 128), (17, 100, 257),
          (64, 1536, 384), (65, 640, 1000), (127, 8960, 256), (128, 64, 129), (129, 384, 127), (200, 1001, 333),
          (256, 2048, 512), (257, 256, 511), (512, 1536, 768), (1000, 333, 1111), (2100, 512, 640), (3, 40000, 20)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_int8(device, m, k, n):
    x = randn(m, k, device=device)
    w = ops.quantize_rows(randn(n, k, seed=1, device=device, scale=0.05))
    bias = randn(n, seed=2, device=device)
    res = randn(m, n, seed=3, device=device)
    r = ops.quantize_rows(x)
    check_product(ops.linear_int8(x, w), *product64(r, w))
    check_product(ops.linear_int8(r, w, bias=bias, residual=res), *product64(r, w, bias, res))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k,n", [(5, 200, 77), (300, 256, 520), (700, 1536, 640)])
def test_linear_int8_types(device, dtype, m, k, n):
    x = randn(m, k, device=device, dtype=torch.float16)
    w = ops.quantize_rows(randn(n, k, seed=1, device=device, dtype=torch.float16, scale=0.05))
    r = ops.quantize_rows(x)
    y = ops.linear_int8(x, w, out_dtype=dtype)
    assert y.dtype == dtype
    check_product(y, *product64(r, w))
    bias, res = randn(n, seed=2, device=device, dtype=torch.float32), randn(m, n, seed=3, device=device, dtype=torch.float32)
    check_product(ops.linear_int8(r, w, bias, res, out_dtype=dtype), *product64(r, w, bias, res))
    assert ops.linear_int8(x, w).dtype == torch.float16
    assert ops.linear_int8(r, w).dtype == torch.bfloat16


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m", [7, 600])
def test_linear_int8_extreme_sums(device, m):
    """Every product at its largest, both signs: the integer sum is exact far beyond 24 bits."""
    k, n = 8960, 130
    x = torch.ones(m, k, dtype=torch.bfloat16, device=device)
    wt = torch.ones(n, k, dtype=torch.bfloat16, device=device)
    wt[1::2] = -1
    wt[:, ::3] = 0.5
    w = ops.quantize_rows(wt)
    y = ops.linear_int8(x, w, out_dtype=torch.float32)
    check_product(y, *product64(ops.quantize_rows(x), w))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,k,n", [(6, 256, 100), (300, 512, 264), (600, 1536, 520)])
def test_linear_int8_strided_out_and_residual(device, m, k, n):
    """Strided ``out`` and ``residual`` (aligned and not), ``residual`` = ``out``, and nothing written
    outside the result."""
    x = randn(m, k, device=device)
    w = ops.quantize_rows(randn(n, k, seed=1, device=device, scale=0.05))
    r = ops.quantize_rows(x)
    for lead, pitch in ((0, n + 24), (8, n + 16), (3, n + 5)):
        buf = randn(m + 2, pitch, seed=4, device=device)
        before = buf.clone()
        view = buf[1 : m + 1, lead : lead + n]
        expect = product64(r, w, None, view)
        assert ops.linear_int8(r, w, residual=view, out=view).data_ptr() == view.data_ptr()
        check_product(view, *expect)
        buf[1 : m + 1, lead : lead + n] = before[1 : m + 1, lead : lead + n]
        assert torch.equal(buf, before)


@pytest.mark.parametrize("device", DEVICES)
def test_linear_int8_rows_without_values(device):
    """Rows of zeros give bias and residual alone; a non-finite token or channel is NaN and stays in its
    row or column."""
    m, k, n = 20, 96, 150
    x = randn(m, k, device=device)
    x[3] = 0
    x[7, 1] = float("nan")
    wt = randn(n, k, seed=1, device=device)
    wt[5] = 0
    wt[11, 2] = float("inf")
    bias = randn(n, seed=2, device=device)
    y = ops.linear_int8(x, ops.quantize_rows(wt), bias=bias)
    cols = torch.arange(n, device=device) != 11
    rows = torch.arange(m, device=device) != 7
    assert torch.equal(y[3][cols], bias[cols]) and torch.equal(y[rows][:, 5], bias[5].expand(m - 1))
    assert bool(y[7].isnan().all()) and bool(y[:, 11].isnan().all())
    assert not bool(y[rows][:, cols].isnan().any())


@pytest.mark.parametrize("device", DEVICES)
def test_linear_int8_empty(device):
    w = ops.quantize_rows(randn(40, 64, device=device))
    assert ops.linear_int8(randn(0, 64, device=device), w).shape == (0, 40)
    assert ops.linear_int8(randn(4, 64, device=device), ops.quantize_rows(randn(0, 64, device=device))).shape == (4, 0)


def test_refusals():
    x = randn(4, 64)
    w = ops.quantize_rows(randn(8, 64, seed=1))
    with pytest.raises(ValueError, match="inner dimensions"):
        ops.linear_int8(randn(4, 63), w)
    with pytest.raises(ValueError, match="inner dimensions"):
        ops.linear_int8(ops.quantize_rows(randn(4, 63)), w)
    with pytest.raises(ValueError, match="Int8Rows"):
        ops.linear_int8(x, randn(8, 64))
    with pytest.raises(ValueError, match="out must be"):
        ops.linear_int8(x, w, out=torch.empty(4, 9, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="out must be"):
        ops.linear_int8(x, w, out=torch.empty(8, 4, dtype=torch.bfloat16).t())
    with pytest.raises(ValueError, match="out_dtype"):
        ops.linear_int8(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="bias must be"):
        ops.linear_int8(x, w, bias=randn(9))
    with pytest.raises(ValueError, match="residual must be"):
        ops.linear_int8(x, w, residual=randn(5, 8))
    with pytest.raises(ValueError, match="one type"):
        ops.linear_int8(x, w, bias=randn(8), residual=randn(4, 8, dtype=torch.float32))
    long = ops.Int8Rows(torch.zeros(1, ops.INT8_MAX_K + 24, dtype=torch.int8), torch.ones(1), ops.INT8_MAX_K + 24)
    with pytest.raises(ValueError, match="at most"):
        ops.linear_int8(long, long)
    with pytest.raises(ValueError, match="rows, features"):
        ops.quantize_rows(randn(64))
    with pytest.raises(ValueError, match="contiguous"):
        ops.quantize_rows(randn(64, 4).t())
    with pytest.raises(ValueError, match="does not hold"):
        ops.quantize_rows(x, out=ops.quantize_rows(randn(5, 64)))
    with pytest.raises(ValueError, match="2K"):
        ops.swiglu_quantize(randn(4, 63))
    with pytest.raises(ValueError, match="norm weight"):
        ops.rmsnorm_quantize(x, randn(63), 1e-6)


@pytest.mark.gpu
def test_refusals_gpu():
    x = randn(4, 64, device="cuda")
    w = ops.quantize_rows(randn(8, 64, seed=1, device="cuda"))
    with pytest.raises(ValueError, match="device"):
        ops.linear_int8(x.cpu(), w)
    with pytest.raises(ValueError, match="device"):
        ops.linear_int8(x, w, bias=randn(8))
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        ops.quantize_rows(x.float())
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.swiglu_quantize(randn(4, 2 * 60, device="cuda"))
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.rmsnorm_quantize(randn(4, 60, device="cuda"), randn(60, device="cuda"), 1e-6)
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.rmsnorm_quantize(randn(4, 72, device="cuda")[:, 4:68], randn(64, device="cuda"), 1e-6)


@pytest.mark.gpu
def test_misaligned_rows_are_refused_or_taken():
    """Buffers that do not start on 16 bytes: int8 rows are refused, everything else is taken element by element."""
    buf = torch.zeros(4 * 64 + 64, dtype=torch.int8, device="cuda")
    q = buf[3 : 3 + 4 * 64].view(4, 64)
    x = randn(4, 64, device="cuda")
    w = ops.quantize_rows(randn(8, 64, seed=1, device="cuda"))
    with pytest.raises(ValueError, match="aligned"):
        ops.quantize_rows(x, out=ops.Int8Rows(q, torch.zeros(4, device="cuda"), 64))
    with pytest.raises(ValueError, match="aligned"):
        ops.linear_int8(ops.Int8Rows(q, torch.zeros(4, device="cuda"), 64), w)
    r = ops.quantize_rows(x)
    scales = torch.zeros(9, device="cuda")
    scales[1:] = w.scale
    bias = randn(9, seed=2, device="cuda")[1:]
    shifted = ops.Int8Rows(w.q, scales[1:], 64)
    check_product(ops.linear_int8(r, shifted, bias=bias), *product64(r, w, bias))


@pytest.mark.gpu
def test_many_rows():
    """More rows than a grid's second dimension holds of the smallest tile, and a broadcast residual."""
    m, k, n = 1_100_000, 16, 8
    x = randn(m, k, device="cuda")
    w = ops.quantize_rows(randn(n, k, seed=1, device="cuda"))
    r = ops.quantize_rows(x)
    res = randn(1, n, seed=2, device="cuda").expand(m, -1)
    check_product(ops.linear_int8(r, w, residual=res), *product64(r, w, None, res))


@pytest.mark.gpu
def test_linear_int8_in_a_graph_and_on_another_stream():
    """Capture with fixed buffers, then replay on new inputs; and the same call on a side stream."""
    for m, k, n in ((4, 1536, 2048), (300, 512, 640), (1024, 1536, 1024)):
        x = randn(m, k, device="cuda")
        w = ops.quantize_rows(randn(n, k, seed=1, device="cuda"))
        norm = torch.ones(k, dtype=torch.bfloat16, device="cuda")

        def call():
            return ops.linear_int8(ops.rmsnorm_quantize(x, norm, 1e-6), w)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = call()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call()
        g.replay()
        assert torch.equal(y, eager)
        x.copy_(randn(m, k, seed=5, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, call()) and not torch.equal(y, eager)
    ops.check_status(torch.device("cuda", 0))
