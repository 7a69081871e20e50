"""Projections with 4-bit weights for a few tokens against their formula in float64, over both types, group sizes, zero
points, odd sizes, pitched and misaligned tokens; the weight layout, the quantiser and the refusals without a device."""
import math

import pytest
import torch

from kernel_pocs_b200 import _lib, w4
from kernel_pocs_b200.fused_mlp import check_status
from kernel_pocs_b200.w4 import W4Weight, quantize_w4, w4_gate_up, w4_linear, w4_mlp

gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
CODES = {torch.float16: 1, torch.bfloat16: 2}


def random_parts(n, k, group, zeros, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randint(0, 256, (n, 16 * ((k + 31) // 32)), generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(n, (k + group - 1) // group, generator=g)) / (4.6 * math.sqrt(k))).to(dtype)
    z = torch.randint(0, 16, scales.shape, generator=g, dtype=torch.uint8) if zeros else None
    return packed, scales, z


def weight64(packed, scales, zeros, k, group):
    """(code - zero) * scale in float64, by the plain definition."""
    q = torch.empty(packed.shape[0], 2 * packed.shape[1], dtype=torch.float64)
    q[:, 0::2], q[:, 1::2] = (packed.cpu() & 15).double(), (packed.cpu() >> 4).double()
    which = torch.arange(k) // group
    z = 8.0 if zeros is None else zeros.cpu().double()[:, which]
    return (q[:, :k] - z) * scales.cpu().double()[:, which]


def make(n, k, group=128, zeros=False, dtype=torch.bfloat16, seed=0):
    parts = random_parts(n, k, group, zeros, dtype, seed)
    w = W4Weight(*parts, in_features=k, group_size=group).to("cuda")
    return w, weight64(*parts, k, group)


def tokens(m, k, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g) * torch.exp(0.5 * torch.randn(1, k, generator=g))).to(dtype).cuda()


def sum_error(x64, w64, k, group):
    """Bound on the fp32 evaluation of x W^T: every addition that a product goes through is off by at most 2^-23 (the
    tensor pipe may truncate) of the magnitudes summed; a product passes a group's steps (two per eight columns, counted
    generously), the groups, and the joining of the parts."""
    return (group / 8 + k / 32 + 16) * 2.0 ** -23 * (x64.abs() @ w64.abs().t())


def act64(act, z):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z * torch.special.ndtr(z)


def assert_linear(y, x, w64, k, group, extra=0.0):
    x64 = x.cpu().double()
    want = x64 @ w64.t()
    half = torch.finfo(y.dtype).eps / 2
    bound = sum_error(x64, w64, k, group) + extra
    # the value that is rounded lies within `bound` of the exact one
    bound = bound + half * (want.abs() + bound) + torch.finfo(y.dtype).smallest_normal * half
    err = (y.cpu().double() - want).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.3f} of the bound"


def assert_gate_up(h, x, wg, wu, k, group, act, gm=1.0, dm=1.0, extra=0.0):
    x64 = x.cpu().double()
    g, u = x64 @ wg.t() * gm, x64 @ wu.t()
    dg, du = (sum_error(x64, wg, k, group) + extra) * gm, sum_error(x64, wu, k, group) + extra
    a = act64(act, g)
    want = a * u * dm
    # |act'| <= 1.13 for the three activations; the activation itself is evaluated within 1e-6 of |z|
    bound = ((1.13 * dg + 1e-6 * g.abs()) * (u.abs() + du) + (a.abs() + 1.13 * dg) * du) * dm
    half = torch.finfo(h.dtype).eps / 2
    bound = bound + half * (want.abs() + bound) + torch.finfo(h.dtype).smallest_normal * half
    err = (h.cpu().double() - want).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.3f} of the bound"


# ------------------------------------------------------------------------------------ no device needed


@pytest.mark.parametrize("n,k,group,zeros", [(1, 1, 32, True), (16, 128, 128, False), (17, 129, 64, True),
                                             (5, 1000, 32, True), (40, 160, 128, False)])
def test_layout_goes_there_and_back(n, k, group, zeros):
    packed, scales, z = random_parts(n, k, group, zeros, torch.bfloat16)
    w = W4Weight(packed, scales, z, in_features=k, group_size=group)
    assert torch.equal(w.packed, packed) and torch.equal(w.scales, scales)
    assert w.zeros is None if z is None else torch.equal(w.zeros, z)
    assert w.shape == (n, k) and w.dtype == torch.bfloat16 and w.to("cpu") is w
    # the documented place of one code: block (r, c), word (hi, g, t, u), its half by parity; and of its scale
    rows, cols, per = (n + 15) // 16, (k + 127) // 128, 128 // group
    size = 1024 + 32 * per + (16 * per if zeros else 0)
    assert w.blocks.shape == (rows, cols, size) and w.nbytes == rows * cols * size
    words = w.blocks[:, :, :1024].contiguous().view(torch.int32).view(rows, cols, 2, 8, 4, 4)
    tail = w.blocks[:, :, 1024:]
    for row, col in ((0, 0), (n - 1, k - 1), (n // 2, k // 2)):
        r, c, i = row // 16, col // 128, col % 8 // 2 + col % 2 * 4
        word = int(words[r, c, row // 8 % 2, row % 8, col // 8 % 4, col // 32 % 4]) & 0xffffffff
        byte = int(packed[row, col // 2])
        assert word >> (4 * i) & 15 == (byte >> 4 if col & 1 else byte & 15)
        at = (row % 8 * per + col % 128 // group) * 2 + row // 8 % 2
        assert tail[r, c, 2 * at:2 * at + 2].contiguous().view(torch.bfloat16) == scales[row, col // group]
        if zeros:
            assert tail[r, c, 32 * per + at] == z[row, col // group]


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(3, 40), (16, 256), (7, 1001)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_is_within_half_a_step(dtype, n, k, group, zero_points):
    g = torch.Generator().manual_seed(n + k)
    weight = torch.randn(n, k, generator=g).to(dtype)
    weight[0] = 0.0
    if zero_points:
        weight = weight.abs()                             # a group of one sign uses the range from zero
    w = quantize_w4(weight, group, zero_points)
    got = weight64(w.packed, w.scales, w.zeros, k, group)
    step = w.scales.double()[:, torch.arange(k) // group]
    # half a step, and up to half a step more at an end of the range: the scale is rounded to 16 bits (half a unit on
    # each of up to 15 steps)
    slack = 15 * torch.finfo(dtype).eps / 2
    assert bool(((got - weight.double()).abs() <= step * (0.5 + slack) + 1e-12).all())
    assert not bool(got[0].any())


def test_copies_have_blocks_of_their_own():
    import copy
    import pickle

    w = W4Weight(*random_parts(20, 200, 64, True, torch.float16), in_features=200, group_size=64)
    for other in (copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert torch.equal(other.blocks, w.blocks) and other.shape == w.shape and other.dtype == w.dtype
        assert other._operand()[0] == other.blocks.data_ptr() != w.blocks.data_ptr()
    with pytest.raises(AttributeError):
        w.blocks = w.blocks[:1]


def test_refusals():
    packed, scales, z = random_parts(4, 64, 32, True, torch.bfloat16)
    ok = dict(in_features=64, group_size=32)
    W4Weight(packed, scales, z, **ok)
    with pytest.raises(ValueError, match="group_size"):
        W4Weight(packed, scales, z, in_features=64, group_size=48)
    with pytest.raises(ValueError, match="bytes per row"):
        W4Weight(packed, scales, z, in_features=65, group_size=32)
    with pytest.raises(TypeError, match="uint8"):
        W4Weight(packed.to(torch.int8), scales, z, **ok)
    with pytest.raises(TypeError, match="bf16 or fp16"):
        W4Weight(packed, scales.float(), z, **ok)
    with pytest.raises(ValueError, match="scales must be of shape"):
        W4Weight(packed, scales[:, :1], z, **ok)
    with pytest.raises(ValueError, match="zeros must be of shape"):
        W4Weight(packed, scales, z[:2], **ok)
    with pytest.raises(ValueError, match="0..15"):
        W4Weight(packed, scales, z + 16, **ok)
    with pytest.raises(TypeError, match="zeros must be uint8"):
        W4Weight(packed, scales, z.int(), **ok)
    with pytest.raises(ValueError, match="at least one row"):
        W4Weight(packed[:0], scales[:0], None, **ok)
    w = W4Weight(packed, scales, z, **ok)
    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    for f in (lambda: w4_linear(x, w), lambda: w4_gate_up(x, w, w), lambda: w4_mlp(x, w, w, w), w.dequantize):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()
    with pytest.raises(ValueError, match="activation"):
        w4_gate_up(x, w, w, "relu")
    with pytest.raises(ValueError, match="no multipliers"):
        w4_gate_up(x, w, w, "gelu_tanh", 2.0)
    other = W4Weight(*random_parts(5, 64, 32, False, torch.bfloat16), **ok)
    with pytest.raises(ValueError, match="agree"):
        w4_gate_up(x, w, other)
    with pytest.raises(ValueError, match="not finite"):
        quantize_w4(torch.full((2, 32), float("nan"), dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="bf16 or fp16"):
        quantize_w4(torch.zeros(2, 32))
    with pytest.raises(ValueError, match="scale is not a finite"):
        quantize_w4(torch.full((2, 32), 1e9), dtype=torch.float16)
    with pytest.raises(ValueError, match="non-empty matrix"):
        quantize_w4(torch.zeros(0, 32, dtype=torch.float16))


def test_c_entries_refuse_bad_arguments_without_a_device():
    lin, gu, dq = _lib.lib.swiglu_b200_w4_linear, _lib.lib.swiglu_b200_w4_gate_up, _lib.lib.swiglu_b200_w4_dequantize
    p = 0x100000
    y, x, w = (p + i * 0x10000 for i in range(3))

    def linear(y=y, x=x, w=w, m=2, n=20, k=130, sx=136, sy=20, group=64, dtype=1):
        return lin(y, x, w, 1, m, n, k, sx, sy, group, dtype, -1, None)

    assert linear(dtype=0) == 1 and linear(dtype=5) == 1
    assert linear(group=16) == 10 and linear(group=0) == 10
    for bad in (dict(m=-1), dict(n=-1), dict(k=-1), dict(sx=129), dict(sy=19), dict(k=0), dict(n=1 << 32), dict(k=1 << 32),
                dict(m=1 << 40, sx=1 << 40)):
        assert linear(**bad) == 3
    for name in ("y", "x", "w"):
        assert linear(**{name: None}) == 2
    assert linear(x=x + 2) == 4 and linear(sx=130) == 4 and linear(y=y + 1) == 4 and linear(w=w + 8) == 4
    assert linear(y=x + 8) == 5 and linear(y=w + 512) == 5
    # two row tiles of two blocks of 1024 codes, two scales and two zero points for each of 16 rows
    assert linear(y=w + 4 * (1024 + 64 + 32) - 2) == 5
    assert linear(m=0, y=None, x=None) == 0 and linear(n=0, sy=0) == 0

    def gate_up(h=y, act=0, u=p + 0x60000, dtype=2):
        return gu(h, x, w, 1, u, 0, 2, 20, 130, 136, 20, 32, dtype, act, 1.0, 1.0, -1, None)

    assert gate_up(act=3) == 10 and gate_up(act=-1) == 10 and gate_up(dtype=0) == 1 and gate_up(u=None) == 2
    assert gate_up(h=p + 0x60000) == 5 and gate_up(h=w + 2) == 5

    def dequantize(out=y, n=20, k=130, so=130, group=128, dtype=1, w=w):
        return dq(out, w, 1, n, k, so, group, dtype, -1, None)

    assert dequantize(dtype=0) == 1 and dequantize(group=256) == 10 and dequantize(so=129) == 3
    assert dequantize(out=None) == 2 and dequantize(w=None) == 2 and dequantize(out=y + 1) == 4
    assert dequantize(out=w) == 5 and dequantize(n=0, out=None) == 0 and dequantize(k=0, so=0) == 0


# ------------------------------------------------------------------------------------ values


SHAPES = [(1, 1, 1), (1, 16, 128), (2, 17, 129), (1, 4096, 1024), (8, 33, 640), (9, 48, 1000), (16, 100, 384),
          (17, 64, 257), (32, 131, 2051), (3, 2731, 1000), (1, 31, 14336), (7, 5, 7), (31, 16, 100), (33, 40, 640), (64, 129, 300),
          (2, 70, 9000), (1, 64, 20000)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,zeros", [(128, False), (64, True), (32, False), (32, True), (128, True)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(dtype, group, zeros, m, n, k):
    w, w64 = make(n, k, group, zeros, dtype, seed=m + n + k)
    x = tokens(m, k, dtype)
    before = _lib.launch_count()
    y = w4_linear(x, w)
    assert _lib.launch_count() == before + 1 and y.shape == (m, n) and y.dtype == dtype
    assert_linear(y, x, w64, k, group)
    assert torch.equal(y, w4_linear(x, w))                # the order of every sum is fixed


def big(n, k, group, zeros, dtype, seed=0):
    """A weight made on the device and, of its rows, some with their float64 values: the first and last ones and a few
    from each part."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    packed = torch.randint(0, 256, (n, 16 * ((k + 31) // 32)), generator=g, dtype=torch.uint8, device="cuda")
    scales = ((0.5 + torch.rand(n, (k + group - 1) // group, generator=g, device="cuda")) / (4.6 * math.sqrt(k))).to(dtype)
    z = torch.randint(0, 16, scales.shape, generator=g, dtype=torch.uint8, device="cuda") if zeros else None
    rows = sorted({r for r in (*range(0, n, max(1, n // 90)), *range(min(n, 20)), *range(max(0, n - 150), n))})
    part = weight64(packed[rows], scales[rows], None if z is None else z[rows], k, group)
    return W4Weight(packed, scales, z, in_features=k, group_size=group), rows, part


# Sizes at which the weights are many enough for the tensor-core kernel with 16, 32 and 64 tokens to a launch: few tokens,
# full and ragged tiles of tokens, one and several of them, odd rows and columns, clusters of all kinds.
MANY = [(3, 7001, 16000), (8, 4096, 14336), (16, 11009, 5500), (17, 9000, 4104), (32, 5503, 6000), (31, 300, 100000),
        (33, 16, 128), (40, 1, 8), (48, 2731, 1000), (64, 129, 2048), (64, 11009, 5504), (65, 4096, 4096), (96, 5000, 136),
        (130, 333, 264), (200, 14336, 1024), (256, 600, 96)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,zeros", [(128, False), (64, True), (32, False), (128, True)])
@pytest.mark.parametrize("m,n,k", MANY)
def test_linear_with_many_weights(dtype, group, zeros, m, n, k):
    w, rows, w64 = big(n, k, group, zeros, dtype, seed=m)
    x = tokens(m, k, dtype)
    y = w4_linear(x, w)
    assert y.shape == (m, n)
    assert_linear(y[:, rows], x, w64, k, group)


@gpu
@pytest.mark.parametrize("act,gm,dm", [("silu", 0.7, 1.3), ("gelu_tanh", 1.0, 1.0), ("gelu_exact", 1.0, 1.0)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,group,zeros", [(5, 5120, 7000, 64, True), (8, 4096, 11008, 128, False),
                                               (16, 11008, 2048, 32, True), (30, 4001, 4096, 128, True),
                                               (33, 40, 264, 64, False), (64, 11008, 1024, 128, False),
                                               (90, 2731, 1000, 32, True), (200, 500, 640, 64, True)])
def test_gate_up_with_many_weights(act, gm, dm, dtype, m, n, k, group, zeros):
    wg, rows, g64 = big(n, k, group, zeros, dtype, seed=m)
    wu, _, u64 = big(n, k, group, not zeros, dtype, seed=m + 1)
    x = tokens(m, k, dtype)
    h = w4_gate_up(x, wg, wu, act, gm, dm)
    assert_gate_up(h[:, rows], x, g64, u64, k, group, act, gm, dm)


@gpu
@pytest.mark.parametrize("act,gm,dm", [("silu", 1.0, 1.0), ("silu", 0.7, 1.3), ("gelu_tanh", 1.0, 1.0),
                                       ("gelu_exact", 1.0, 1.0)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,group,zeros", [(1, 16, 128, 128, False), (1, 2731, 1000, 32, True),
                                               (8, 100, 4096, 64, True), (12, 77, 513, 128, False),
                                               (32, 40, 2048, 64, False), (5, 3, 9, 32, True),
                                               (96, 130, 260, 64, True), (2, 33, 6000, 128, True)])
def test_gate_up(act, gm, dm, dtype, m, n, k, group, zeros):
    wg, g64 = make(n, k, group, zeros, dtype, seed=n)
    wu, u64 = make(n, k, group, zeros, dtype, seed=n + 1)
    x = tokens(m, k, dtype)
    before = _lib.launch_count()
    h = w4_gate_up(x, wg, wu, act, gm, dm)
    assert _lib.launch_count() == before + 1
    assert_gate_up(h, x, g64, u64, k, group, act, gm, dm)


@gpu
def test_gate_up_takes_one_weight_with_zero_points_and_one_without():
    wg, g64 = make(50, 200, 64, True, seed=1)
    wu, u64 = make(50, 200, 64, False, seed=2)
    x = tokens(4, 200, torch.bfloat16)
    assert_gate_up(w4_gate_up(x, wg, wu), x, g64, u64, 200, 64, "silu")
    assert_gate_up(w4_gate_up(x, wu, wg), x, u64, g64, 200, 64, "silu")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,zeros", [(128, False), (64, True), (32, True)])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (100, 1000), (5, 2091), (33, 96), (64, 4096)])
def test_dequantize_is_exact(dtype, group, zeros, n, k):
    w, w64 = make(n, k, group, zeros, dtype, seed=k)
    got = w.dequantize()
    assert got.shape == (n, k) and torch.equal(got.cpu(), w64.to(dtype))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 6, 20])
@pytest.mark.parametrize("offset,extra", [(0, 0), (1, 0), (8, 8), (0, 3), (4, 12)])
def test_pitched_and_misaligned_tokens(dtype, m, offset, extra):
    n, k = 50, 600
    w, w64 = make(n, k, 64, True, dtype)
    x = tokens(m, k, dtype)
    buf = torch.full((offset + m * (k + extra) + 8,), float("nan"), dtype=dtype, device="cuda")
    v = buf[offset:offset + m * (k + extra)].view(m, k + extra)[:, :k]
    v.copy_(x)
    want = w4_linear(x, w)
    assert torch.equal(w4_linear(v, w), want)
    # the result between guards, at its own pitch
    out = torch.full((16 + m * (n + 5),), 55.0, dtype=dtype, device="cuda")
    y = out[8:8 + m * (n + 5)].view(m, n + 5)[:, :n]
    st = torch.cuda.current_stream().cuda_stream
    assert _lib.lib.swiglu_b200_w4_linear(y.data_ptr(), x.data_ptr(), *w._operand(), m, n, k, k, n + 5, 64,
                                          CODES[dtype], -1, st) == 0
    assert torch.equal(y, want)
    y.fill_(55.0)
    assert bool((out == 55.0).all())
    full = torch.full((n * (k + 7) + 16,), 55.0, dtype=dtype, device="cuda")
    d = full[5:5 + n * (k + 7)].view(n, k + 7)[:, :k]
    assert _lib.lib.swiglu_b200_w4_dequantize(d.data_ptr(), *w._operand(), n, k, k + 7, 64, CODES[dtype], -1, st) == 0
    assert torch.equal(d, w.dequantize())
    d.fill_(55.0)
    assert bool((full == 55.0).all())


@gpu
def test_leading_shapes_empty_batches_and_transposed_tokens():
    w, w64 = make(40, 256, 128)
    x = tokens(6, 256, torch.bfloat16)
    assert torch.equal(w4_linear(x.view(2, 3, 256), w), w4_linear(x, w).view(2, 3, 40))
    assert torch.equal(w4_linear(x[0], w), w4_linear(x, w)[0])
    assert torch.equal(w4_linear(x.t().contiguous().t(), w), w4_linear(x, w))
    assert torch.equal(w4_linear(x[:1].expand(6, 256), w), w4_linear(x[:1], w).expand(6, 40))
    for shape in ((0, 256), (2, 0, 256)):
        e = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        assert w4_linear(e, w).shape == (*shape[:-1], 40) and w4_gate_up(e, w, w).shape == (*shape[:-1], 40)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan_stay_in_their_token(dtype):
    w, w64 = make(60, 300, 64, True, dtype)
    x = tokens(5, 300, dtype)
    want = w4_linear(x, w)
    x[1, 7], x[3, 299] = float("nan"), float("inf")
    got = w4_linear(x, w)
    assert bool(torch.isnan(got[1]).all()) and not bool(torch.isfinite(got[3]).any())
    keep = [0, 2, 4]
    assert torch.equal(got[keep], want[keep])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,offset,extra", [(40, 60, 300, 8, 20), (70, 200, 129, 0, 7), (20, 9001, 4096, 16, 8)])
def test_many_tokens_in_pitched_rows_keep_what_is_around_them(dtype, m, n, k, offset, extra):
    """The tokens' and the results' neighbours: NaN beside the tokens is not read, memory beside the results not written;
    Inf and NaN stay in their tokens."""
    w, rows, w64 = big(n, k, 64, True, dtype)
    wide = torch.full((m + 1, offset + k + extra), float("nan"), dtype=dtype, device="cuda")
    x = wide[:m, offset:offset + k]
    x.copy_(tokens(m, k, dtype))
    assert_linear(w4_linear(x, w)[:, rows], x, w64, k, 64)
    # the C entry writes rows of any pitch
    aligned, pitch = w4._aligned_rows(x)
    y = torch.full((m + 2, n + 5), 7.0, dtype=dtype, device="cuda")
    assert _lib.lib.swiglu_b200_w4_linear(y[1].data_ptr(), aligned.data_ptr(), *w._operand(), m, n, k, pitch, n + 5, 64,
                                          CODES[dtype], 0, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(y[1:m + 1, :n], w4_linear(x, w))
    assert bool((y[0] == 7).all()) and bool((y[m + 1] == 7).all()) and bool((y[1:m + 1, n:] == 7).all())
    want = w4_linear(x, w)
    x[1, 7], x[m - 1, k - 1] = float("nan"), float("inf")
    got = w4_linear(x, w)
    assert bool(torch.isnan(got[1]).all()) and not bool(torch.isfinite(got[m - 1]).any())
    keep = [i for i in range(m) if i not in (1, m - 1)]
    assert torch.equal(got[keep], want[keep])


@gpu
def test_tensor_core_kernels_share_the_device():
    """Launches of several kernels that keep their sums in tensor memory, on two streams at once: each gets its own."""
    from kernel_pocs_b200.fused_mlp import gate_up_swiglu_forward

    dtype, k = torch.bfloat16, 1024
    w, _, _ = big(5000, k, 128, False, dtype)
    x = tokens(64, k, dtype)
    g = torch.Generator(device="cuda").manual_seed(0)
    wg, wu = (torch.randn(2048, k, generator=g, device="cuda").mul_(0.03).to(dtype) for _ in range(2))
    with torch.no_grad():
        want_y, want_h = w4_linear(x, w), gate_up_swiglu_forward(x, wg, wu)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = [[], []]
        for _ in range(20):
            with torch.cuda.stream(streams[0]):
                got[0].append(w4_linear(x, w))
            with torch.cuda.stream(streams[1]):
                got[1].append(gate_up_swiglu_forward(x, wg, wu))
                got[0].append(w4_linear(x, w))
        torch.cuda.synchronize()
    check_status()
    assert all(torch.equal(y, want_y) for y in got[0]) and all(torch.equal(h, want_h) for h in got[1])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(449, 64, 256), (600, 48, 1000), (512, 37, 129)])
def test_many_tokens_take_the_16_bit_weights(dtype, m, n, k):
    """Above the limits every weight is rounded to 16 bits once more: half a unit of each product's magnitude."""
    assert m > max(w4.LINEAR_ROWS, w4.GATE_UP_ROWS)
    w, w64 = make(n, k, 64, True, dtype)
    wu, u64 = make(n, k, 64, False, dtype, seed=9)
    x = tokens(m, k, dtype)
    x64, half = x.cpu().double(), torch.finfo(dtype).eps / 2
    # a library product may sum one column after the other: k additions
    extra = half * (x64.abs() @ w64.abs().t()) + k * 2.0 ** -23 * (x64.abs() @ w64.abs().t())
    extra_u = half * (x64.abs() @ u64.abs().t()) + k * 2.0 ** -23 * (x64.abs() @ u64.abs().t())
    assert_linear(w4_linear(x, w), x, w64, k, 64, extra)
    with torch.no_grad():
        h = w4_gate_up(x, w, wu, "gelu_tanh")
    check_status()
    # the projections may be rounded to 16 bits in front of the activation
    proj = half * torch.maximum((x64 @ w64.t()).abs() + extra, (x64 @ u64.t()).abs() + extra_u)
    assert_gate_up(h, x, w64, u64, k, 64, "gelu_tanh", extra=torch.maximum(extra, extra_u) + proj)


@gpu
def test_quantised_mlp_end_to_end():
    """quantize_w4 -> w4_mlp against the same three matrices in float64, rounding included step by step."""
    dtype, hidden, inter = torch.bfloat16, 320, 848
    g = torch.Generator().manual_seed(0)
    mats = [(torch.randn(*s, generator=g) / math.sqrt(s[1])).to(dtype).cuda()
            for s in ((inter, hidden), (inter, hidden), (hidden, inter))]
    ws = [quantize_w4(m, 64) for m in mats]
    w64 = [weight64(w.packed, w.scales, w.zeros, w.in_features, 64) for w in ws]
    x = tokens(3, hidden, dtype)
    with torch.no_grad():
        h = w4_gate_up(x, ws[0], ws[1])
        y = w4_mlp(x, *ws)
    assert_gate_up(h, x, w64[0], w64[1], hidden, 64, "silu")
    assert_linear(y, h, w64[2], inter, 64)


@gpu
def test_an_input_that_wants_a_gradient_is_refused():
    w, _ = make(16, 64, 64)
    x = tokens(1, 64, torch.bfloat16).requires_grad_()
    for f in (lambda: w4_linear(x, w), lambda: w4_gate_up(x, w, w)):
        with pytest.raises(RuntimeError, match="forward only"):
            f()
    with torch.no_grad():
        w4_linear(x, w)
    with pytest.raises(TypeError, match="scales are"):
        w4_linear(x.detach().half(), w)
    with pytest.raises(ValueError, match="does not end in"):
        w4_linear(x.detach()[:, :32], w)


@gpu
def test_captured_token_replays_on_new_inputs_and_streams():
    w, _ = make(400, 512, 64, True)
    wu, _ = make(400, 512, 64, True, seed=5)
    wd, _ = make(512, 400, 64, True, seed=6)
    x = tokens(2, 512, torch.bfloat16)
    w4_mlp(x, w, wu, wd)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                                    # two graphs of the same weights share nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(w4_mlp(x, w, wu, wd))
        graphs.append(graph)
    for seed in (7, 8):
        x.copy_(tokens(2, 512, torch.bfloat16, seed=seed))
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
        torch.cuda.synchronize()
        want = w4_mlp(x, w, wu, wd)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@gpu
@pytest.mark.parametrize("m", [64, 450])
def test_captured_gate_up_of_many_tokens(m):
    """Also above the limit, after and between eager calls of the fused projections it takes outside a graph."""
    dtype, n, k = torch.bfloat16, 64, 256
    wg, _ = make(n, k, 64, True, dtype)
    wu, _ = make(n, k, 64, False, dtype, seed=9)
    x = tokens(m, k, dtype)
    with torch.no_grad():
        for _ in range(300):
            w4_gate_up(x, wg, wu)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [w4_gate_up(x, wg, wu) for _ in range(300)]
        x.copy_(tokens(m, k, dtype, seed=5))
        graph.replay()
        eager = w4_gate_up(x, wg, wu)
        torch.cuda.synchronize()
    check_status()
    assert all(torch.equal(o, outs[0]) for o in outs)
    # projections rounded to bf16 on one side at most: two half units each, and one of the result
    scale = float(eager.float().abs().max())
    assert float((outs[0].float() - eager.float()).abs().max()) <= 6 * torch.finfo(dtype).eps / 2 * scale


@gpu
@pytest.mark.parametrize("m", [1, 2, 8, 24, 48, 100])
def test_launches_in_a_row_see_what_came_before_them(m):
    """Launches may start before the one in front of them has ended: tokens, weights and outputs that change from one
    call to the next, with nothing waited for in between, against the same calls one at a time."""
    dtype = torch.bfloat16
    w, _ = make(700, 512, 64, True, dtype)
    wu, _ = make(700, 512, 64, False, dtype, seed=5)
    wd, _ = make(512, 700, 128, True, dtype, seed=6)
    others = [make(700, 512, 64, True, dtype, seed=20 + i)[0].blocks for i in range(3)]
    start = tokens(m, 512, dtype)

    def chain(wait):
        x, seen = start.clone(), []
        for i in range(40):
            if i % 5 == 0:
                w.blocks.copy_(others[i // 5 % 3])        # new weights, enqueued right before they are read
            h = w4_gate_up(x, w, wu)
            if wait:
                torch.cuda.synchronize()
            y = w4_linear(h, wd)
            if wait:
                torch.cuda.synchronize()
            x.copy_(y / y.float().abs().amax(dim=1, keepdim=True).clamp(min=1e-20).to(dtype))
            seen += [y, h.clone()]
            del h
        return torch.stack([t.float().sum() for t in seen]), seen

    sums, want = chain(True)
    for _ in range(3):
        again, got = chain(False)
        torch.cuda.synchronize()
        assert bool(torch.isfinite(sums).all()) and torch.equal(again, sums)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
