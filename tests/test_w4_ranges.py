"""4-bit projections of tokens whose values are far apart: one large channel among small ones, magnitudes over the whole
range of the type, rows that read a single column.  The bounds are those of test_w4.py: fp32 sums, one rounding."""

import pytest
import torch

from kernel_pocs_b200.w4 import W4Weight, w4_gate_up, w4_linear
from tests.test_w4 import DTYPES, assert_gate_up, assert_linear, random_parts, tokens, weight64

gpu = pytest.mark.gpu


def blind_weight(n, k, group, zeros, dtype, columns, seed=0):
    """A weight whose even rows have the zero point as their code at `columns`: what stands there does not count, and the
    rest of the token has to be as exact as without it."""
    packed, scales, z = random_parts(n, k, group, zeros, dtype, seed)
    for c in columns:
        zero = (torch.full((n,), 8, dtype=torch.uint8) if z is None else z[:, c // group])[::2]
        byte = packed[::2, c // 2]
        packed[::2, c // 2] = (byte & 15) | (zero << 4) if c & 1 else (byte & 0xf0) | zero
    w64 = weight64(packed, scales, z, k, group)
    assert not bool(w64[::2, list(columns)].any())
    return W4Weight(packed, scales, z, in_features=k, group_size=group).to("cuda"), w64


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spike,typical", [(500.0, 0.1), (3000.0, 0.02), (30000.0, 0.01), (60000.0, 1e-4)])
@pytest.mark.parametrize("m,n,k,group,zeros", [(1, 64, 256, 128, False), (2, 40, 1000, 32, True), (1, 131, 14336, 128, True),
                                               (2, 70, 9000, 64, False), (1, 2731, 130, 64, True), (3, 40, 1000, 64, True)])
def test_a_large_channel_leaves_its_neighbours_exact(dtype, spike, typical, m, n, k, group, zeros):
    columns = sorted({0, 77, k // 2, k - 1})
    w, w64 = blind_weight(n, k, group, zeros, dtype, columns, seed=k)
    x = tokens(m, k, dtype).float() * typical
    for i, c in enumerate(columns):
        x[i % m, c] = spike if i & 1 else -spike
    x = x.to(dtype)
    y = w4_linear(x, w)
    assert_linear(y, x, w64, k, group)
    assert torch.equal(y, w4_linear(x, w))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,gm,dm", [("silu", 0.7, 1.3), ("gelu_tanh", 1.0, 1.0)])
@pytest.mark.parametrize("m", [1, 2])
def test_gate_up_beside_a_large_channel(dtype, act, gm, dm, m):
    n, k, group = 100, 700, 64
    columns = (5, 300, 699)
    wg, g64 = blind_weight(n, k, group, True, dtype, columns, seed=1)
    wu, u64 = blind_weight(n, k, group, False, dtype, columns, seed=2)
    x = tokens(m, k, dtype).float() * 0.05
    x[m - 1, list(columns)] = torch.tensor([20000.0, -8000.0, 30000.0], device="cuda")
    x = x.to(dtype)
    h = w4_gate_up(x, wg, wu, act, gm, dm)
    # the odd rows see the large channel and may leave fp16: their formula is of no use there
    assert_gate_up(h[:, ::2], x, g64[::2], u64[::2], k, group, act, gm, dm)


@gpu
@pytest.mark.parametrize("dtype,low,high", [(torch.float16, -24, 15), (torch.bfloat16, -30, 30), (torch.bfloat16, -70, 40)])
@pytest.mark.parametrize("m,k,group,zeros", [(1, 300, 64, True), (2, 1030, 32, False), (2, 512, 128, True)])
def test_rows_that_read_one_column(dtype, low, high, m, k, group, zeros):
    """Row j has column j alone (every other code is its zero point), so y[:, j] is x[:, j] times one weight, whatever
    stands beside it; magnitudes are spread over most of what the type holds."""
    n = k
    _, scales, z = random_parts(n, k, group, zeros, dtype, seed=3)
    scales = torch.ones_like(scales)
    zero = (torch.full((n, k), 8, dtype=torch.uint8) if z is None else z[:, torch.arange(k) // group])
    codes = torch.zeros(n, 32 * ((k + 31) // 32), dtype=torch.uint8)
    codes[:, :k] = zero
    diagonal = torch.arange(k)
    codes[diagonal, diagonal] = torch.where(zero[diagonal, diagonal] > 0, zero[diagonal, diagonal] - 1, 1).to(torch.uint8)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    w64 = weight64(packed, scales, z, k, group)
    assert bool((w64.abs() == torch.eye(k, dtype=torch.float64)).all())
    w = W4Weight(packed, scales, z, in_features=k, group_size=group).to("cuda")
    g = torch.Generator().manual_seed(k)
    x = torch.exp2(low + (high - low) * torch.rand(m, k, generator=g))
    x = (x * torch.where(torch.rand(m, k, generator=g) < 0.5, -1.0, 1.0)).to(dtype).cuda()
    x[:, 40:60] = 0.0
    y = w4_linear(x, w)
    assert_linear(y, x, w64, k, group)
    # a product with 1 or -1 and sums with zeros: nothing to round
    assert torch.equal(y.cpu().double(), x.cpu().double() @ w64.t())


@gpu
@pytest.mark.parametrize("m", [1, 2])
def test_tokens_smaller_than_the_normal_range_of_their_unit(m):
    """bf16 far below 2^-63, where the unit of the integers would leave fp32."""
    n, k, group = 33, 520, 64
    w, w64 = blind_weight(n, k, group, True, torch.bfloat16, (3,), seed=5)
    x = (tokens(m, k, torch.bfloat16).float() * 2.0 ** -100).to(torch.bfloat16)
    x[0, 256:] = 0.0
    assert_linear(w4_linear(x, w), x, w64, k, group)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 3, 12])
@pytest.mark.parametrize("k,group,zeros", [(300, 64, True), (256, 128, False), (2100, 32, True)])
def test_infinities_and_nan_go_through_the_formula(dtype, m, k, group, zeros):
    """An Inf gives Inf of the weight's sign, and NaN where its weight is zero or another Inf is against it; a NaN gives NaN.
    Every row has what the formula in float64 has, whatever the number of tokens."""
    n = 90
    w, w64 = blind_weight(n, k, group, zeros, dtype, (7,), seed=k)
    clean = tokens(m, k, dtype)
    at = min(k - 1, 1500)
    for values in ({7: float("inf")}, {at: float("-inf")}, {7: float("inf"), at: float("inf")}, {at: float("nan")},
                   {c: float("-inf") for c in range(8)}, {c: float("inf") for c in range(k)}):
        x = clean.clone()
        for c, v in values.items():
            x[m - 1, c] = v
        y = w4_linear(x, w).cpu().double()
        want = (x.cpu().double()[:, None, :] * w64).sum(-1)
        assert torch.equal(y.isnan(), want.isnan())
        assert torch.equal(y.isinf() & (y > 0), want == float("inf"))
        assert torch.equal(y.isinf() & (y < 0), want == float("-inf"))
        assert torch.equal(y[:m - 1], w4_linear(clean, w).cpu().double()[:m - 1])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,group,zeros", [(33, 130, 1000, 64, True), (64, 40, 520, 128, False), (100, 257, 264, 32, True)])
def test_many_tokens_beside_large_channels_infinities_and_nan(dtype, m, n, k, group, zeros):
    """The same of the tensor-core form: rows that do not see the large channels, and the formula for what is not finite."""
    columns = (0, 77, k - 1)
    w, w64 = blind_weight(n, k, group, zeros, dtype, columns, seed=k)
    x = tokens(m, k, dtype).float() * 0.01
    x[:, list(columns)] = 30000.0
    x = x.to(dtype)
    clean = w4_linear(x, w)
    assert_linear(clean, x, w64, k, group)
    x[1, 77], x[m - 1, 78], x[m // 2, 79] = float("inf"), float("-inf"), float("nan")
    y = w4_linear(x, w)
    hit = [1, m - 1, m // 2]
    want = (x[hit].cpu().double()[:, None, :] * w64).sum(-1)
    got = y[hit].cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf() & (got > 0), want == float("inf")) and torch.equal(got.isinf() & (got < 0), want == -float("inf"))
    keep = [i for i in range(m) if i not in hit]
    assert torch.equal(y[keep], clean[keep])
