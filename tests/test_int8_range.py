"""8-bit products over the whole range of scales: neither the product of two scales nor a partial one may leave fp32's
range where the result does not."""

import pytest
import torch

from accerl_agent_b200 import ops
from test_int8 import check_product, product64, randn

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,k,n", [(5, 1536, 132), (7, 200, 77), (2300, 4096, 1536)])
def test_scales_far_from_one(device, m, k, n):
    """Tolerances as for ordinary scales: five fp32 roundings, none of them of a subnormal number (an accumulator is a
    whole number, so it times a scale is a multiple of the scale's own step)."""
    if device == "cpu" and m > 100:
        m, n = 300, 40
    for sx, sw in ((1e-20, 1e-20), (1e-25, 1e-17), (1e-38, 1.0), (1e37, 1e-37), (1e-37, 1e37), (1e30, 1e4), (1e-30, 1e-4)):
        x = randn(m, k, device=device, dtype=torch.float32)
        x = (x * sx).bfloat16()
        w = ops.quantize_rows((randn(n, k, seed=1, device=device, dtype=torch.float32) * sw).bfloat16())
        r = ops.quantize_rows(x)
        for dtype in (torch.float32, torch.bfloat16):
            y = ops.linear_int8(r, w, out_dtype=dtype)
            check_product(y, *product64(r, w))


@pytest.mark.parametrize("device", DEVICES)
def test_sums_of_zero_stay_zero(device):
    """Tokens and channels whose products are all zero, at scales whose product overflows: the result is the bias."""
    m, k, n = 9, 64, 40
    x = torch.zeros(m, k, device=device)
    x[:, 0] = 1e38
    wt = torch.zeros(n, k, device=device)
    wt[:, 1] = 1e38
    bias = randn(n, seed=2, device=device)
    y = ops.linear_int8(x.bfloat16(), ops.quantize_rows(wt.bfloat16()), bias=bias)
    assert torch.equal(y, bias.expand(m, -1))
