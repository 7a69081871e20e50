"""4-bit projections of prompts, the calls above LINEAR_ROWS and GATE_UP_ROWS that take the weights written out in 16 bits:
the same tokens, shapes and arguments as below the limits."""
import pytest
import torch

from kernel_pocs_b200 import w4
from kernel_pocs_b200.fused_mlp import check_status
from kernel_pocs_b200.w4 import W4Weight, w4_gate_up, w4_linear
from tests.test_w4 import DTYPES, assert_gate_up, assert_linear, make, random_parts, tokens, weight64

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


def exact_weight(n, k, zeros, dtype, exponent, seed):
    """A weight whose scales are powers of two: (code - zero) * scale has at most 4 bits and is not rounded by 16."""
    packed, scales, z = random_parts(n, k, 64, zeros, dtype, seed)
    g = torch.Generator().manual_seed(seed)
    scales = torch.exp2(exponent - torch.randint(0, 2, scales.shape, generator=g)).to(dtype)
    return W4Weight(packed, scales, z, in_features=k, group_size=64).to("cuda"), weight64(packed, scales, z, k, 64)


def sums_error(x64, w64):
    """Beside what assert_gate_up allows: a library product may add one column after the other."""
    return x64.shape[1] * 2.0 ** -23 * (x64.abs() @ w64.abs().t())


@gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("act,gm,dm", ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k,zeros", [(64, 256, True), (37, 129, False), (48, 1000, True)])
def test_projections_are_not_rounded_on_the_way(captured, act, gm, dm, dtype, n, k, zeros):
    """Eager and in a graph, whichever product serves the sizes and the type; three-dimensional tokens."""
    wg, g64 = exact_weight(n, k, zeros, dtype, -6, 3)
    wu, u64 = exact_weight(n, k, not zeros, dtype, -6, 4)
    x = tokens(M, k, dtype).view(3, M // 3, k)
    with torch.no_grad():
        h = w4_gate_up(x, wg, wu, act, gm, dm)
        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                h = w4_gate_up(x, wg, wu, act, gm, dm)
            x.copy_(tokens(M, k, dtype, seed=8).view_as(x))
            graph.replay()
    check_status()
    assert h.shape == (3, M // 3, n)
    x = x.view(M, k)
    x64 = x.cpu().double()
    assert_gate_up(h.view(M, n), x, g64, u64, k, 64, act, gm, dm, torch.maximum(sums_error(x64, g64), sums_error(x64, u64)))


@gpu
@pytest.mark.parametrize("act,dm", [("silu", 2.0 ** -22), ("gelu_tanh", 1.0), ("gelu_exact", 1.0)])
@pytest.mark.parametrize("m", [8, M])
def test_fp16_projections_beyond_its_range(act, dm, m):
    """A gate of 2 * 10^5 times a small up, or with SiLU a small multiplier, is well within fp16."""
    n, k, dtype = 48, 128, torch.float16
    wg, g64 = exact_weight(n, k, False, dtype, 2, 1)
    wu, u64 = exact_weight(n, k, False, dtype, 2 if act == "silu" else -19, 2)
    x = tokens(m, k, dtype) * 400
    x64 = x.cpu().double()
    g = x64 @ g64.t()
    assert float(g.abs().max()) > 1.5 * 65504 and float((g * (x64 @ u64.t()) * dm).abs().max()) < 60000
    with torch.no_grad():
        h = w4_gate_up(x, wg, wu, act, 1.0, dm)
    assert_gate_up(h, x, g64, u64, k, 64, act, 1.0, dm, torch.maximum(sums_error(x64, g64), sums_error(x64, u64)))


@gpu
def test_a_prompt_is_worked_on_in_pieces(monkeypatch):
    """Projections in 32 bits are held for a few tokens at a time: any number of pieces gives the same."""
    n, k, dtype = 40, 200, torch.float16
    (wg, _), (wu, _) = exact_weight(n, k, True, dtype, -6, 5), exact_weight(n, k, False, dtype, -6, 6)
    x = tokens(M, k, dtype)
    whole = w4_gate_up(x, wg, wu)
    monkeypatch.setattr(w4, "PIECE_ROWS", 128)
    # pieces may take other products of the library: sums in another order, rounded once
    torch.testing.assert_close(w4_gate_up(x, wg, wu), whole, rtol=2 * torch.finfo(dtype).eps, atol=1e-4)


@gpu
@pytest.mark.parametrize("dtype,other", [(torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("m,n,k", [(8, 64, 256), (M, 64, 256), (M, 37, 129)])
def test_autocast_does_not_reach_the_products(dtype, other, m, n, k):
    wg, wu = make(n, k, 64, True, dtype)[0], make(n, k, 64, False, dtype, seed=9)[0]
    x = tokens(m, k, dtype)
    with torch.no_grad():
        want = [w4_linear(x, wg), *(w4_gate_up(x, wg, wu, act, gm, dm) for act, gm, dm in ACTS)]
        with torch.autocast("cuda", dtype=other):
            got = [w4_linear(x, wg), *(w4_gate_up(x, wg, wu, act, gm, dm) for act, gm, dm in ACTS)]
    check_status()
    assert all(a.dtype == dtype and torch.equal(a, b) for a, b in zip(got, want))
