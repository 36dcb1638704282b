"""Sampling from given random numbers where weights and sums meet their borders: weights within a rounding of min-p,
and numbers at and above 1, whose token is the last candidate."""

import math

import pytest
import torch

from accerl_agent_b200 import ops
from test_sampler_counts import check, full, make

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def check_border(x, u, t, m):
    """Each token is the largest logit, or its weight is at least min_p to within a rounding of a 64-bit weight (half a
    step, 2^-53, for the exponential's argument and for its value); its log-probability is its own."""
    tok, lp = ops.sample_inverse_cdf(x, u, t, min_p=m)
    xs = x.double().cpu()
    z = torch.logsumexp(xs, 1)
    for r, (i, l) in enumerate(zip(tok.tolist(), lp.tolist())):
        assert 0 <= i < x.shape[1]
        gap = float(xs[r, i] - xs[r].max())
        assert gap == 0 or math.exp(gap / float(t[r])) >= float(m[r]) * (1 - 2.0 ** -52)
        want = float(xs[r, i] - z[r])
        assert abs(l - want) <= 2.0 ** -23 * abs(want) + 1e-12
    return tok


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_a_rounding_below_min_p(device, dtype):
    """Temperatures so high that weights are 1 or one rounding below it, with min-p 1: whatever is kept is drawn from,
    and nothing else. 3.0 weighs 1 - 2^-53 next to 4.0 at a temperature of 1.75e16."""
    temps = [1.75e16, 4e15, 9e15, 1e16, 1.2e16, 2e16, 5e16, 1e18, 1e30, 3e38, float("inf")]
    numbers = [0.0, 0.4, 0.6, 0.75, 0.9999]
    t = torch.tensor([a for a in temps for _ in numbers], dtype=torch.float32, device=device)
    u = torch.tensor(numbers * len(temps), dtype=torch.float32, device=device)
    m = torch.ones_like(u)
    n = u.shape[0]
    rows = [[4.0, 3.0], [3.0, 4.0, -3.0, 2.0, 3.984375, 0.0], [1.0, -1.0], [0.0, -0.5, -0.25, 0.0]]
    for row in rows:
        x = torch.tensor([row], dtype=dtype, device=device).expand(n, -1)
        tok = check_border(x, u, t, m)
        if row == rows[0]:
            assert tok[:5].tolist() == [0] * 5
    # a value outside the counters' window; rows spread over several blocks; odd starts
    x = torch.tensor([[4.0, 3.0, 1e-13, 100.0, 127.0, 200.0]], dtype=torch.float64).to(dtype).to(device).expand(n, -1)
    check_border(x, u, t, m)
    for width in (9001, 40001):
        base, _, _ = make(3, width, device, dtype, seed=width)
        for r in range(3):
            x = base[r : r + 1, r:].expand(8, -1)
            check_border(x, u[:8].contiguous(), t[:8].contiguous(), m[:8].contiguous())
            check_border(x, u[40:48].contiguous(), t[40:48].contiguous(), m[40:48].contiguous())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,v", [(16, 3001), (3, 30011)])
def test_numbers_from_one_on_take_the_last_candidate(device, dtype, rows, v):
    """u >= 1 counts as the largest number below 1, so it names the last token that the cuts leave, in every order of
    adding up the weights before it (each candidate holds at least 1e-7 of the mass, far above a rounding)."""
    x, _, _ = make(rows, v, device, dtype, seed=v)
    x[1] = x[1].abs()  # few groups of values
    x[2, ::3] = x[2, 0]
    off = full(rows, 1.0, device)
    for uu in (1.0, float("inf")):
        u = full(rows, uu, device)
        for k in (1, 7, 50, 333):
            kk = full(rows, k, device, torch.int32)
            check(x, u, off, kk)
            check(x, u, full(rows, 0.7, device), kk, full(rows, 0.9, device))
        for p in (0.05, 0.5, 0.95):
            check(x, u, off, None, full(rows, p, device))
            check(x, u, off, None, full(rows, p, device), full(rows, 0.001, device))


@pytest.mark.parametrize("device", DEVICES)
def test_one_column_of_any_stride(device):
    base, u, _ = make(5, 12, device, torch.bfloat16)
    x = base.t()[:, :1]  # [12, 1] with strides (1, 12)
    assert x.stride(1) != 1
    tok, lp = ops.sample_inverse_cdf(x, full(12, 0.5, device), full(12, 1.0, device))
    assert not tok.any() and not lp.any()
    one = base.t()[3:4, :1]
    tok, lp = ops.sample_inverse_cdf(one, full(1, 0.5, device), full(1, 1.0, device))
    assert not tok.any() and not lp.any()
