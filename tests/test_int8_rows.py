"""Rows behind SwiGLU in 8 bits where there are so many that a ring of bulk copies feeds them: every number of chunks a
thread holds, a last stage that is not full, strided rows, and the row counts on either side of the rule."""

import pytest
import torch

from accerl_agent_b200 import ops
from test_int8 import check_rows, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,k", [(30001, 64), (30001, 264), (30003, 520), (30005, 776), (30007, 1016), (14301, 2040),
                                    (7103, 4096), (3553, 8200), (3552, 8200), (3553, 9472), (3553, 9480)])
def test_swiglu_rows_of_many_rows(rows, k):
    gu = randn(rows, 2 * k, device="cuda", scale=2.0)
    gu[1] *= 40
    gu[2, 3], gu[rows - 1, 5] = float("inf"), float("nan")
    check_rows(ops.swiglu(gu), ops.swiglu_quantize(gu))
    ops.check_status(torch.device("cuda", 0))


def test_swiglu_rows_strided():
    """Rows 16 bytes apart from each other's end, NaN between them."""
    rows, k = 30001, 264
    buf = torch.full((rows, 2 * k + 8), float("nan"), dtype=torch.bfloat16, device="cuda")
    gu = buf[:, : 2 * k]
    gu.copy_(randn(rows, 2 * k, device="cuda", scale=2.0))
    check_rows(ops.swiglu(gu.contiguous()), ops.swiglu_quantize(gu))
