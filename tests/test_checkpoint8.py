"""Gated activations that keep their inputs in 8 bits: the codes against their definition in float64, the forward
bit for bit against swiglu / geglu, the gradients bit for bit against this library's backward at the kept values,
against the formula in float64 and against central differences; layouts, refusals, graphs, streams."""
import math

import pytest
import torch

from kernel_pocs_b200 import _lib, checkpoint8
from kernel_pocs_b200.checkpoint8 import (
    Checkpoint8, ckpt8_backward, ckpt8_backward_recompute, ckpt8_forward, ckpt8_pack, geglu_ckpt8, geglu_packed_ckpt8,
    swiglu_ckpt8, swiglu_packed_ckpt8,
)
from kernel_pocs_b200.geglu import geglu_backward, geglu_backward_recompute, geglu_forward
from kernel_pocs_b200.swiglu import swiglu_backward, swiglu_backward_recompute, swiglu_forward

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = ["silu", "gelu_tanh", "gelu_exact"]


# ------------------------------------------------------------------------------------ the definition, in float64


def kept64(x: torch.Tensor) -> torch.Tensor:
    """The value each element is kept as, in float64 (rows along the last dimension, groups of 32 columns)."""
    x = x.detach().cpu().double()
    n = x.shape[-1]
    v = torch.nn.functional.pad(x.reshape(-1, n), (0, -n % 32)).view(-1, (n + 31) // 32, 32)
    top = v.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(v).all(-1, keepdim=True)
    top = torch.where(fine, top, 1.0)
    s = torch.frexp(top).exponent - 7
    s = s + (torch.ldexp(top, -s) >= 127.5)
    s = torch.where(top > 0, s, -126).clamp(min=-126)
    fine = fine & (s <= 121)  # the largest magnitude would be kept as 64 * 2^122, which is not a float
    q = torch.round(torch.ldexp(v, -s))
    assert bool((q.abs()[fine.expand_as(q)] <= 127).all())
    out = torch.where(fine, torch.ldexp(q, s), float("nan"))
    return out.view(-1, (n + 31) // 32 * 32)[:, :n].reshape(x.shape)


def act64(act: str, z: torch.Tensor):
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    cdf = torch.special.ndtr(z)
    return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def inputs(rows, cols, dtype, seed=0, std=1.5):
    g = torch.Generator().manual_seed(seed)
    return tuple((std * torch.randn(rows, cols, generator=g)).to(dtype).cuda() for _ in range(3))


def place(x: torch.Tensor, offset: int, pitch: int):
    """``x`` as a view whose rows are ``pitch`` elements apart, the first one ``offset`` elements into its storage."""
    rows, cols = x.shape
    buf = torch.full((offset + rows * pitch + 64,), 77.0, dtype=x.dtype, device=x.device)
    v = buf[offset:offset + rows * pitch].view(rows, pitch)[:, :cols]
    v.copy_(x)
    return v


def same_bits(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def forward_of(act, gate, up, gm=1.0, dm=1.0):
    if act == "silu":
        return swiglu_forward(gate, up, gm, dm)[0]
    return geglu_forward(gate, up, "tanh" if act == "gelu_tanh" else "none")[0]


def backward_of(act, dh, gate, up, gm=1.0, dm=1.0):
    if act == "silu":
        return swiglu_backward(dh, gate, up, gm, dm, preserve_inputs=True)
    return geglu_backward(dh, gate, up, "tanh" if act == "gelu_tanh" else "none", preserve_inputs=True)


def recompute_of(act, dh, gate, up, gm=1.0, dm=1.0):
    if act == "silu":
        return swiglu_backward_recompute(dh, gate, up, gm, dm, preserve_inputs=True)
    return geglu_backward_recompute(dh, gate, up, "tanh" if act == "gelu_tanh" else "none", preserve_inputs=True)


# ------------------------------------------------------------------------------------ refusals (no device needed)


def test_refusals():
    a, b = torch.zeros(4, 8), torch.zeros(4, 8)
    for f in (swiglu_ckpt8, geglu_ckpt8, ckpt8_forward, ckpt8_pack):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f(a, b)
        with pytest.raises(ValueError, match="same shape"):
            f(a, b[:3])
        with pytest.raises(TypeError, match="same dtype"):
            f(a, b.half())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        swiglu_packed_ckpt8(a)
    with pytest.raises(ValueError, match="must be even"):
        geglu_packed_ckpt8(torch.zeros(4, 7))
    with pytest.raises(ValueError, match="activation must be one of"):
        ckpt8_forward(a, b, "relu")
    with pytest.raises(ValueError, match="no multipliers"):
        ckpt8_pack(a, b, "gelu_tanh", 0.5)
    with pytest.raises(TypeError, match="real Python scalar"):
        swiglu_ckpt8(a, b, "1")
    with pytest.raises(TypeError, match="not a tensor"):
        swiglu_ckpt8(a, b, torch.tensor(1.0))
    with pytest.raises(ValueError, match="approximate"):
        geglu_ckpt8(a, b, "sigmoid")
    with pytest.raises(TypeError, match="fp16, bf16, and fp32"):
        ckpt8_forward(a.double(), b.double())
    kept = Checkpoint8(torch.ones(Checkpoint8.size((4, 8)), dtype=torch.uint8), (4, 8), torch.float32)
    with pytest.raises(ValueError, match="is 264 bytes"):
        Checkpoint8(torch.ones(263, dtype=torch.uint8), (4, 8), torch.float32)
    with pytest.raises(ValueError, match="in a row"):
        Checkpoint8(torch.ones(528, dtype=torch.uint8)[::2], (4, 8), torch.float32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ckpt8_backward(torch.zeros(4, 8), kept)
    with pytest.raises(ValueError, match="must be even"):
        checkpoint8.ForgePackedCkpt8Function.apply(torch.zeros(4, 7))
    with pytest.raises(ValueError, match="does not match"):
        ckpt8_backward(torch.zeros(4, 9), kept)
    with pytest.raises(TypeError, match="dtype and device"):
        ckpt8_backward(torch.zeros(4, 8, dtype=torch.float16), kept)
    with pytest.raises(ValueError, match="contiguous dout"):
        ckpt8_backward_recompute(torch.zeros(8, 4).t(), kept)


def test_c_entries_refuse_bad_arguments_without_a_device():
    f, b = _lib.lib.swiglu_b200_ckpt8_fwd, _lib.lib.swiglu_b200_ckpt8_bwd
    p = 0x100000
    h, gc, uc, gs, us, g, u = (p + i * 0x10000 for i in range(7))

    def fwd(h=h, gc=gc, uc=uc, gs=gs, us=us, g=g, u=u, rows=4, cols=40, si=40, so=40, dtype=_lib.BF16, act=0):
        return f(h, gc, uc, gs, us, g, u, rows, cols, si, so, dtype, act, 1.0, 1.0, -1, None)

    assert fwd(dtype=7) == 1 and fwd(act=3) == 10 and fwd(act=-1) == 10
    assert fwd(rows=-1) == 3 and fwd(si=39) == 3 and fwd(so=39) == 3
    assert fwd(rows=1 << 40, si=1 << 40) == 3  # past the address space
    for name in ("gc", "uc", "gs", "us", "g", "u"):
        assert fwd(**{name: None}) == 2
    assert fwd(gc=gc + 8) == 4 and fwd(g=g + 1) == 4 and fwd(h=h + 1) == 4
    assert fwd(h=g) == 5 and fwd(uc=gc) == 5 and fwd(gs=g + 16) == 5 and fwd(us=gs + 2) == 5 and fwd(gc=u) == 5
    assert fwd(rows=0, h=None, g=None) == 0 and fwd(cols=0, si=0, so=0) == 0

    dg, du, d = p + 0x90000, p + 0xa0000, p + 0xb0000

    def bwd(h=None, dg=dg, du=du, d=d, gc=gc, uc=uc, gs=gs, us=us, rows=4, cols=40, sg=40, sd=40, sh=40,
            dtype=_lib.F32, act=1):
        return b(h, dg, du, d, gc, uc, gs, us, rows, cols, sg, sd, sh, dtype, act, 1.0, 1.0, -1, None)

    assert bwd(dtype=-1) == 1 and bwd(act=9) == 10
    assert bwd(cols=-1) == 3 and bwd(sg=39) == 3 and bwd(sd=39) == 3 and bwd(h=h, sh=39) == 3
    for name in ("dg", "du", "d", "gc", "uc", "gs", "us"):
        assert bwd(**{name: None}) == 2
    assert bwd(uc=uc + 4) == 4 and bwd(d=d + 2) == 4 and bwd(h=h + 2) == 4
    assert bwd(dg=d) == 5 and bwd(du=dg) == 5 and bwd(h=dg) == 5 and bwd(h=d + 4) == 5 and bwd(dg=gc) == 5
    assert bwd(h=d, sh=41) == 5  # over dout, but with another pitch
    assert bwd(rows=0, dg=None) == 0


def test_dequantize_reads_the_codes_on_any_device():
    kept = Checkpoint8(torch.zeros(66, dtype=torch.uint8), (3,), torch.float32)
    kept.codes[0, 0, :3] = torch.tensor([127, -127, 1])
    kept.codes[1, 0, 0] = 5
    kept.steps[:] = torch.tensor([[[127]], [[255]]])
    g, u = kept.dequantize()
    assert g.tolist() == [127.0, -127.0, 1.0] and bool(torch.isnan(u).all())
    assert kept.nbytes == 66


# ------------------------------------------------------------------------------------ values


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (5, 33), (2, 15), (4, 17), (7, 100), (3, 1024),
                                       (2, 5503), (65, 512), (1, 4096)])
@pytest.mark.parametrize("act", ACTS)
def test_step_matches_the_definition_and_the_plain_kernels(dtype, rows, cols, act):
    gm, dm = (0.7, 1.3) if act == "silu" else (1.0, 1.0)
    gate, up, dh = inputs(rows, cols, dtype, seed=rows * 7919 + cols)
    before = _lib.launch_count()
    h, kept = ckpt8_forward(gate, up, act, gm, dm)
    assert _lib.launch_count() == before + 1
    assert same_bits(h, forward_of(act, gate, up, gm, dm))
    g, u = kept.dequantize()
    assert torch.equal(g.cpu().double(), kept64(gate)) and torch.equal(u.cpu().double(), kept64(up))
    groups = (cols + 31) // 32
    assert kept.codes.shape == (2, rows, 32 * groups) and not bool(kept.codes[:, :, cols:].any())

    # the kept values are numbers of the input type (7 bits times a power of two), so the plain backward takes them
    dgate, dup = ckpt8_backward(dh, kept)
    want = backward_of(act, dh, g.to(dtype), u.to(dtype), gm, dm)
    assert same_bits(dgate, want[0]) and same_bits(dup, want[1])
    h2, dgate2, dup2 = ckpt8_backward_recompute(dh, kept, preserve_inputs=True)
    want = recompute_of(act, dh, g.to(dtype), u.to(dtype), gm, dm)
    assert same_bits(h2, want[0]) and same_bits(dgate2, dgate) and same_bits(dup2, dup)
    over = dh.clone()
    h3, dgate3, dup3 = ckpt8_backward_recompute(over, kept)
    assert h3.data_ptr() == over.data_ptr() and same_bits(h3, h2) and same_bits(dgate3, dgate) and same_bits(dup3, dup)
    alone = ckpt8_pack(gate, up, act, gm, dm)
    assert torch.equal(alone.codes, kept.codes) and torch.equal(alone.steps, kept.steps)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_the_formula_and_differences(dtype, act):
    gate, up, dh = inputs(33, 321, dtype, seed=5)
    _, kept = ckpt8_forward(gate, up, act)
    dgate, dup = ckpt8_backward(dh, kept)
    g, u, d = kept64(gate), kept64(up), dh.cpu().double()
    a, da = act64(act, g)
    eps = 1e-6
    diff = (act64(act, g + eps)[0] - act64(act, g - eps)[0]) / (2 * eps)
    # central differences in float64: truncation eps^2/6 * |act'''| (below 2); each value off by a few 2^-53 * |g|,
    # divided by eps
    assert bool(((diff - da).abs() <= 1e-12 + 1e-9 * (1 + g.abs())).all())
    # one rounding to the type, half a step; the fp32 evaluation within 1e-6 of |dh * up| (the contract of the plain
    # kernels, which the bit-for-bit test above ties these to)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for slope in (da, diff):
        want = d * u * slope
        assert bool(((dgate.cpu().double() - want).abs() <= half * want.abs() + 1.01e-6 * (d * u).abs() * (1 + 1e-3)
                     + tiny).all())
    want = d * a
    assert bool(((dup.cpu().double() - want).abs() <= half * want.abs() + 1e-6 * want.abs() + tiny).all())
    # half a step of the kept form: the input itself is within 1/127 of its group's largest magnitude, halved
    n = gate.shape[-1]
    top = torch.nn.functional.pad(gate.cpu().double(), (0, -n % 32)).view(33, -1, 32).abs().amax(-1, keepdim=True)
    bound = (top / 127).expand(-1, -1, 32).reshape(33, -1)[:, :n]
    assert bool(((g - gate.cpu().double()).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_special_groups(dtype):
    info = torch.finfo(dtype)
    rows = []
    row = torch.zeros(64)
    rows.append(row.clone())                              # all zero
    rows.append(torch.linspace(-1, 1, 64))
    row[5] = 255.0 / 128.0                                # rounds to 128 steps of 2^-6: the step doubles
    row[6] = 1.0
    rows.append(row.clone())
    row[5] = 254.0 / 128.0                                # 127 steps
    rows.append(row.clone())
    row = torch.arange(64, dtype=torch.float32) / 2       # ties: 64 + odd halves
    row[63], row[31] = 100.0, 100.0
    rows.append(row.clone())
    rows.append(torch.full((64,), info.max))
    rows.append(torch.full((64,), -info.max))
    rows.append(torch.full((64,), info.smallest_normal))
    rows.append(torch.full((64,), info.smallest_normal * info.eps))
    row = torch.full((64,), info.smallest_normal * info.eps * 3)
    row[40] = info.max
    rows.append(row)
    for bad in (float("inf"), float("-inf"), float("nan")):
        row = torch.linspace(-2, 2, 64)
        row[35] = bad
        rows.append(row)
    x = torch.stack(rows).to(dtype).cuda()
    y = x.flip(0).contiguous()
    h, kept = ckpt8_forward(x, y)
    g, u = kept.dequantize()
    assert torch.equal(g.cpu().double().nan_to_num(123.0), kept64(x).nan_to_num(123.0))
    assert torch.equal(u.cpu().double().nan_to_num(123.0), kept64(y).nan_to_num(123.0))
    assert same_bits(h, swiglu_forward(x, y)[0])
    dgate, dup = ckpt8_backward(torch.ones_like(x), kept)
    # a step that overflowed does not come back finite
    bad = torch.isnan(kept64(x)).cuda()
    assert bool(bad.any()) and bool(torch.isnan(dup[bad]).all()) and bool(torch.isnan(dgate[bad]).all())
    assert bool(torch.isfinite(dup[~bad & (x.abs() < 100)]).all())


# ------------------------------------------------------------------------------------ layouts


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,offset,extra", [(64, 0, 0), (64, 1, 0), (64, 0, 3), (100, 5, 7), (511, 8, 1),
                                               (1536, 16, 0), (1537, 3, 30), (47, 2, 1), (544, 0, 16), (13, 1, 2)])
def test_pitched_and_misaligned_rows_equal_contiguous_ones(dtype, cols, offset, extra):
    rows = 9
    gate, up, dh = inputs(rows, cols, dtype, seed=cols + offset)
    h, kept = ckpt8_forward(gate, up)
    pg, pu = place(gate, offset, cols + extra), place(up, offset + 3, cols + extra)
    h2, kept2 = ckpt8_forward(pg, pu)
    assert same_bits(h, h2) and torch.equal(kept.codes, kept2.codes) and torch.equal(kept.steps, kept2.steps)
    dgate, dup = ckpt8_backward(dh, kept)
    dg2, du2 = ckpt8_backward(place(dh, offset + 1, cols + 2 * extra), kept)
    assert same_bits(dgate, dg2) and same_bits(dup, du2)

    # outputs at their own offsets and pitches, through the C entry: nothing beside the rows is written
    es, lib = dtype.itemsize, _lib.lib
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    st = torch.cuda.current_stream().cuda_stream
    groups = kept.steps.shape[2]

    def out(shift):
        buf = torch.full((offset + shift + rows * (cols + extra) + 64,), 55.0, dtype=dtype, device="cuda")
        return buf, buf[offset + shift:offset + shift + rows * (cols + extra)].view(rows, -1)[:, :cols]

    (hb, hv), (gb, gv), (ub, uv) = out(0), out(1), out(6)
    codes, steps = torch.empty_like(kept.codes), torch.empty_like(kept.steps)
    assert lib.swiglu_b200_ckpt8_fwd(hv.data_ptr(), codes[0].data_ptr(), codes[1].data_ptr(), steps[0].data_ptr(),
                                     steps[1].data_ptr(), gate.data_ptr(), up.data_ptr(), rows, cols, cols,
                                     cols + extra, code, 0, 1.0, 1.0, -1, st) == 0
    assert torch.equal(hv, h) and torch.equal(codes, kept.codes) and torch.equal(steps, kept.steps)
    assert lib.swiglu_b200_ckpt8_bwd(None, gv.data_ptr(), uv.data_ptr(), dh.data_ptr(), codes[0].data_ptr(),
                                     codes[1].data_ptr(), steps[0].data_ptr(), steps[1].data_ptr(), rows, cols,
                                     cols + extra, cols, 0, code, 0, 1.0, 1.0, -1, st) == 0
    assert torch.equal(gv, dgate) and torch.equal(uv, dup)
    for buf, view, want in ((hb, hv, h), (gb, gv, dgate), (ub, uv, dup)):
        view.fill_(55.0)
        assert bool((buf == 55.0).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_cols", [32, 40, 257, 1024, 5503])
@pytest.mark.parametrize("act", ACTS)
def test_packed_layout_and_autograd(dtype, n_cols, act):
    gate, up, dh = inputs(12, n_cols, dtype, seed=n_cols)
    packed = torch.cat((gate, up), dim=1).view(3, 4, 2 * n_cols)
    g, u = gate.view(3, 4, n_cols).clone().requires_grad_(), up.view(3, 4, n_cols).clone().requires_grad_()
    leaf = packed.clone().requires_grad_()
    if act == "silu":
        h, hp = swiglu_ckpt8(g, u, 0.7, 1.3), swiglu_packed_ckpt8(leaf, 0.7, 1.3)
    else:
        form = "tanh" if act == "gelu_tanh" else "none"
        h, hp = geglu_ckpt8(g, u, form), geglu_packed_ckpt8(leaf, form)
    dh3 = dh.view(3, 4, n_cols)
    dg, du = torch.autograd.grad(h, (g, u), dh3, retain_graph=True)
    again = torch.autograd.grad(h, (g, u), dh3)            # the codes are still there: nothing was overwritten
    (dp,) = torch.autograd.grad(hp, leaf, dh3)
    assert same_bits(h, hp) and same_bits(torch.cat((dg, du), dim=2), dp)
    assert same_bits(again[0], dg) and same_bits(again[1], du)
    assert same_bits(g.detach().view(12, n_cols), gate) and same_bits(leaf.detach(), packed)
    kept = ckpt8_pack(gate, up, act, *((0.7, 1.3) if act == "silu" else ()))
    want = ckpt8_backward(dh, kept)
    assert same_bits(dg.view(12, n_cols), want[0]) and same_bits(du.view(12, n_cols), want[1])
    # without a gradient nothing is kept, and the result is the same
    with torch.no_grad():
        h0 = swiglu_ckpt8(g, u, 0.7, 1.3) if act == "silu" else geglu_ckpt8(g, u, form)
        hp0 = swiglu_packed_ckpt8(leaf, 0.7, 1.3) if act == "silu" else geglu_packed_ckpt8(leaf, form)
    assert same_bits(h0, h) and same_bits(hp0, h)


@gpu
def test_broadcast_transposed_and_expanded_operands():
    gate, up, dh = inputs(24, 40, torch.float32, seed=3)
    t = gate.t().contiguous().t()                          # columns contiguous
    h, kept = ckpt8_forward(t, up)
    h0, kept0 = ckpt8_forward(gate, up)
    assert same_bits(h, h0) and torch.equal(kept.codes, kept0.codes)
    row = gate[:1].expand(24, 40)                          # rows on top of each other
    h, kept = ckpt8_forward(row, up)
    h0, kept0 = ckpt8_forward(row.contiguous(), up)
    assert same_bits(h, h0) and torch.equal(kept.codes, kept0.codes)
    leaf = gate[:1].clone().requires_grad_()
    up_leaf = up.clone().requires_grad_()
    swiglu_ckpt8(leaf.expand(24, 40), up_leaf).sum().backward()   # expanded dout, gradient summed over the rows
    dg, du = ckpt8_backward(torch.ones_like(up), kept0)
    # a sum of 24 fp32 terms, in whatever order: 23 roundings of at most half a step of the terms' sizes added up
    assert bool(((leaf.grad.double() - dg.double().sum(0)).abs() <= 23 * 2 ** -24 * dg.double().abs().sum(0)).all())
    assert same_bits(up_leaf.grad, du)


@gpu
@pytest.mark.parametrize("shape", [(0, 8), (4, 0), (2, 0, 5), (7,), (1,)])
def test_empty_and_one_dimensional(shape):
    gate = torch.randn(shape, device="cuda").requires_grad_()
    up = torch.randn(shape, device="cuda").requires_grad_()
    h = swiglu_ckpt8(gate, up)
    assert h.shape == gate.shape
    dg, du = torch.autograd.grad(h, (gate, up), torch.ones_like(h))
    assert dg.shape == gate.shape and du.shape == up.shape
    assert same_bits(h, swiglu_forward(gate.detach(), up.detach())[0])


@gpu
def test_rows_split_over_calls_give_the_same_bits():
    gate, up, dh = inputs(37, 777, torch.bfloat16, seed=9)
    h, kept = ckpt8_forward(gate, up)
    dg, du = ckpt8_backward(dh, kept)
    for lo, hi in ((0, 20), (20, 37)):
        hs, ks = ckpt8_forward(gate[lo:hi], up[lo:hi])
        assert same_bits(hs, h[lo:hi]) and torch.equal(ks.codes, kept.codes[:, lo:hi])
        a, b = ckpt8_backward(dh[lo:hi], ks)
        assert same_bits(a, dg[lo:hi]) and same_bits(b, du[lo:hi])


@gpu
def test_large_matrix_with_offsets_past_32_bits():
    rows, cols = 66000, 33000                              # 2.2e9 elements: byte offsets and element counts past 2^32, 2^31
    gate = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_()
    up = torch.empty_like(gate).normal_()
    h, kept = ckpt8_forward(gate, up)
    dg, du = ckpt8_backward(h, kept)
    for lo in (0, 40000, rows - 3):
        hs, ks = ckpt8_forward(gate[lo:lo + 3].clone(), up[lo:lo + 3].clone())
        assert same_bits(hs, h[lo:lo + 3]) and torch.equal(ks.codes, kept.codes[:, lo:lo + 3])
        a, b = ckpt8_backward(h[lo:lo + 3].clone(), ks)
        assert same_bits(a, dg[lo:lo + 3]) and same_bits(b, du[lo:lo + 3])


# ------------------------------------------------------------------------------------ autograd, graphs, streams


@gpu
def test_second_derivatives_are_refused_and_memory_is_what_it_says():
    gate, up, dh = inputs(512, 4096, torch.bfloat16)
    g, u = gate.requires_grad_(), up.requires_grad_()
    h = swiglu_ckpt8(g, u)
    saved = h.grad_fn.saved_tensors
    assert sum(t.numel() * t.element_size() for t in saved) == 2 * (512 * 4096 + 512 * 128)
    (dg,) = torch.autograd.grad(h, g, dh.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        dg.sum().backward()


@gpu
def test_captured_step_replays_on_new_inputs():
    gate, up, dh = inputs(64, 1000, torch.bfloat16, seed=1)
    h, kept = ckpt8_forward(gate, up)                      # binds the library
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        h, kept = ckpt8_forward(gate, up)
        grads = ckpt8_backward(dh, kept)
    for seed in (2, 3):
        for dst, src in zip((gate, up, dh), inputs(64, 1000, torch.bfloat16, seed=seed)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        h0, kept0 = ckpt8_forward(gate, up)
        want = ckpt8_backward(dh, kept0)
        assert same_bits(h, h0) and same_bits(grads[0], want[0]) and same_bits(grads[1], want[1])


@gpu
def test_captured_autograd_step():
    """Forward and gradients through autograd in one graph, the leaves made on the capturing stream."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        gate, up, dh = inputs(48, 321, torch.float16, seed=1)
        gate.requires_grad_(), up.requires_grad_()
        for _ in range(2):
            torch.autograd.grad(geglu_ckpt8(gate, up), (gate, up), dh)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        h = geglu_ckpt8(gate, up)
        grads = torch.autograd.grad(h, (gate, up), dh)
    with torch.no_grad():
        for dst, src in zip((gate, up, dh), inputs(48, 321, torch.float16, seed=2)):
            dst.copy_(src)
    graph.replay()
    torch.cuda.synchronize()
    h0, kept = ckpt8_forward(gate.detach(), up.detach(), "gelu_tanh")
    want = ckpt8_backward(dh, kept)
    assert same_bits(h.detach(), h0) and same_bits(grads[0], want[0]) and same_bits(grads[1], want[1])


@gpu
def test_side_stream():
    gate, up, dh = inputs(256, 2048, torch.float16, seed=4)
    want_h, kept = ckpt8_forward(gate, up)
    want = ckpt8_backward(dh, kept)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        h, kept = ckpt8_forward(gate, up)
        got = ckpt8_backward(dh, kept)
    side.synchronize()
    assert same_bits(h, want_h) and same_bits(got[0], want[0]) and same_bits(got[1], want[1])


# ------------------------------------------------------------------------------------ in the LoRA block


def _lora_operands(dtype, m, hidden, inter, r, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(*shape, std):
        return (std * torch.randn(shape, generator=g, device="cuda")).to(dtype)

    W = [t(inter, hidden, std=hidden ** -0.5), t(inter, hidden, std=hidden ** -0.5), t(hidden, inter, std=inter ** -0.5)]
    A = [t(r, hidden, std=hidden ** -0.5), t(r, hidden, std=hidden ** -0.5), t(r, inter, std=inter ** -0.5)]
    B = [t(inter, r, std=0.1), t(inter, r, std=0.1), t(hidden, r, std=0.1)]
    return t(2, m // 2, hidden, std=1.0), W, A, B


@gpu
@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("dtype,r", [(torch.bfloat16, 16), (torch.float32, 5), (torch.float16, 8)])
def test_lora_mlp_with_8_bit_checkpoints(dtype, r, activation):
    """The gradients are those of the block's own backward on the kept e and g, bit for bit; the forward is untouched."""
    from types import SimpleNamespace

    from kernel_pocs_b200.fused_mlp import check_status
    from kernel_pocs_b200.lora_mlp import LoRAMLP

    X, W, A, B = _lora_operands(dtype, 66, 128, 336, r)
    leaves = [X, *A, *B]
    for t in leaves:
        t.requires_grad_()

    def run(*checkpoint):
        return LoRAMLP.apply(X, W[0], A[0], B[0], 0.5, W[1], A[1], B[1], 2.0, W[2], A[2], B[2], 1.5, activation,
                             *checkpoint)

    plain, kept = run(), run("int8")
    assert same_bits(plain, kept)
    e, g = plain.grad_fn.saved_tensors[1:3]
    saved = kept.grad_fn.saved_tensors[1]
    assert saved.dtype == torch.uint8 and saved.numel() == Checkpoint8.size((66, 336))
    k = ckpt8_pack(e, g, activation)
    eh, gh = (t.to(dtype) for t in k.dequantize())
    dY = torch.randn_like(plain)
    got = torch.autograd.grad(kept, leaves, dY, retain_graph=True)
    again = torch.autograd.grad(kept, leaves, dY)            # nothing saved was overwritten
    ctx = SimpleNamespace(saved_tensors=(X, eh, gh, A[0], B[0], A[1], B[1], A[2], B[2]), base_weights=tuple(W),
                          scales=(0.5, 2.0, 1.5), activation=activation, kept=None)
    with torch.no_grad():
        want = LoRAMLP.backward(ctx, dY)
    want = [want[i] for i in (0, 2, 6, 10, 3, 7, 11)]
    for a, b, c in zip(got, want, again):
        assert same_bits(a, b) and same_bits(a, c)
    check_status()


@gpu
def test_lora_mlp_refuses_an_unknown_checkpoint():
    from kernel_pocs_b200.lora_mlp import LoRAMLP

    X, W, A, B = _lora_operands(torch.float32, 4, 16, 32, 4)
    with pytest.raises(ValueError, match="checkpoint must be"):
        LoRAMLP.apply(X, W[0], A[0], B[0], 1.0, W[1], A[1], B[1], 1.0, W[2], A[2], B[2], 1.0, "silu", "fp8")
