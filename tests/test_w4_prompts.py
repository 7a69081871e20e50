"""4-bit projections of prompts, the calls above LINEAR_ROWS and GATE_UP_ROWS that take the weights written out in 16 bits:
the same tokens, shapes and arguments as below the limits."""
import pytest
import torch

from kernel_pocs_b200 import w4
from kernel_pocs_b200.fused_mlp import check_status
from kernel_pocs_b200.w4 import w4_gate_up, w4_linear
from tests.test_w4 import DTYPES, assert_linear, make, tokens

gpu = pytest.mark.gpu
M = 450
ACTS = [("silu", 1.0, 1.0), ("silu", 0.7, 1.3), ("gelu_tanh", 1.0, 1.0), ("gelu_exact", 1.0, 1.0)]


def product_error(x64, w64, dtype):
    """What the weights' rounding to 16 bits and a library product, which may add one column after the other, are off by
    beside what assert_linear allows."""
    return (torch.finfo(dtype).eps / 2 + x64.shape[1] * 2.0 ** -23) * (x64.abs() @ w64.abs().t())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,extra", [(0, 0), (1, 0), (4, 0), (3, 8), (0, 5)])
def test_tokens_that_start_anywhere(dtype, offset, extra):
    assert M > max(w4.LINEAR_ROWS, w4.GATE_UP_ROWS)
    n, k = 64, 256
    wg, g64 = make(n, k, 64, True, dtype)
    wu, u64 = make(n, k, 64, False, dtype, seed=9)
    x = tokens(M, k, dtype)
    buf = torch.full((offset + M * (k + extra) + 8,), float("nan"), dtype=dtype, device="cuda")
    v = buf[offset:offset + M * (k + extra)].view(M, k + extra)[:, :k]
    v.copy_(x)
    assert_linear(w4_linear(v, wg), x, g64, k, 64, product_error(x.cpu().double(), g64, dtype))
    for act, gm, dm in ACTS:
        with torch.no_grad():
            assert torch.equal(w4_gate_up(v, wg, wu, act, gm, dm), w4_gate_up(x, wg, wu, act, gm, dm))
    check_status()
