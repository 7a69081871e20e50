"""The gated MLP in fewer bits, as measured work: activations kept in 8 bits between the passes of a training step, and
frozen 4-bit weights applied to a few tokens.

Operators (the ``op`` of a case):

``step``        one training step of the gated activation that keeps ``gate`` and ``up`` as 8-bit codes: the forward,
                then the gradients of ``gate`` and ``up`` at the values the codes stand for.
``recompute``   the same for a block that makes its own ``h`` first and needs it again in the backward (a LoRA MLP):
                the codes are made from ``gate`` and ``up``, and the backward returns ``h``, ``dgate`` and ``dup``.
``linear``      a projection with 4-bit weights and group scales for a few tokens.
``gate_up``     both projections of a gated MLP with 4-bit weights and the activation, for a few tokens.
``dequantize``  a 4-bit weight written out in 16 bits, for the matrix products of a long prompt.

8-bit codes: along every row, each group of 32 columns shares a step 2^s; s is the smallest exponent (not below -126)
for which the group's largest magnitude rounds to at most 127 steps.  4-bit weights: byte j of a row holds columns 2j
(low half) and 2j + 1, rows are padded to a multiple of 32 columns; the value is (code - zero) * scale of its group.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
MAX_STEP_ELEMENTS = 16384 * 14336
MAX_WEIGHTS = 14336 * 4096


# ---------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # the activation of one large training batch: 16384 tokens at the 14336-wide MLP
        dict(name="step silu bf16 16384x14336", op="step", act="silu", dtype="bf16", rows=16384, cols=14336,
             packed=False, gm=1.0, dm=1.0),
        # a packed gate|up projection of odd half-width with multipliers: no row shares an alignment with the next
        dict(name="step silu fp16 packed 4099x11009", op="step", act="silu", dtype="fp16", rows=4099, cols=11009,
             packed=True, gm=0.7, dm=1.3),
        # a small step, where the launches count
        dict(name="step silu fp32 256x1024", op="step", act="silu", dtype="fp32", rows=256, cols=1024, packed=False,
             gm=1.0, dm=1.0),
        # a LoRA MLP with a GELU gate, one batch of 8192 tokens
        dict(name="recompute gelu_tanh bf16 8192x14336", op="recompute", act="gelu_tanh", dtype="bf16", rows=8192,
             cols=14336, packed=False, gm=1.0, dm=1.0),
        # the erf form in full precision, a ragged batch at an odd width
        dict(name="recompute gelu_exact fp32 1031x5503", op="recompute", act="gelu_exact", dtype="fp32", rows=1031,
             cols=5503, packed=False, gm=1.0, dm=1.0),
        # the down projection of one generated token
        dict(name="linear bf16 1x14336 to 4096", op="linear", dtype="bf16", m=1, k=14336, n=4096, group=128,
             zeros=False),
        # a batch of 32 sequences that each generate a token; odd output width, zero points
        dict(name="linear fp16 32x5504 to 11009", op="linear", dtype="fp16", m=32, k=5504, n=11009, group=64,
             zeros=True),
        # the gate and up projections of one generated token
        dict(name="gate_up silu bf16 1x4096 to 14336", op="gate_up", act="silu", dtype="bf16", m=1, k=4096, n=14336,
             group=128, zeros=False, gm=1.0, dm=1.0),
        # eight sequences, zero points, the 11008-wide MLP with a GELU gate
        dict(name="gate_up gelu_tanh fp16 8x4096 to 11008", op="gate_up", act="gelu_tanh", dtype="fp16", m=8, k=4096,
             n=11008, group=64, zeros=True, gm=1.0, dm=1.0),
        # a small MLP of odd sizes, three tokens of a draft
        dict(name="gate_up silu bf16 3x1000 to 2731", op="gate_up", act="silu", dtype="bf16", m=3, k=1000, n=2731,
             group=32, zeros=False, gm=1.0, dm=1.0),
        # a whole projection written out before a prompt is read
        dict(name="dequantize bf16 14336x4096", op="dequantize", dtype="bf16", n=14336, k=4096, group=128, zeros=False),
        # odd sizes: rows that start at every alignment
        dict(name="dequantize fp16 5503x2091", op="dequantize", dtype="fp16", n=5503, k=2091, group=32, zeros=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "recompute", "linear", "gate_up", "dequantize"])
    if op in ("step", "recompute"):
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        cols = _log_uniform(rng, 64, 28672)
        if rng.random() < 0.5:
            cols = max(32, cols // 32 * 32)
        rows = min(_log_uniform(rng, 64, 16384), max(1, MAX_STEP_ELEMENTS // (2 * cols)))
        act = rng.choice(["silu", "silu", "gelu_tanh", "gelu_exact"])
        scaled = act == "silu" and rng.random() < 0.5
        return dict(op=op, act=act, dtype=dtype, rows=rows, cols=cols,
                    packed=op == "step" and rng.random() < 0.5,
                    gm=round(rng.uniform(0.5, 1.5), 3) if scaled else 1.0,
                    dm=round(rng.uniform(0.5, 1.5), 3) if scaled else 1.0)
    case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5)
    k = _log_uniform(rng, 512, 16384)
    if rng.random() < 0.7:
        k = k // 32 * 32
    n = min(_log_uniform(rng, 512, 28672), MAX_WEIGHTS // k)
    case.update(k=k, n=n)
    if op != "dequantize":
        case["m"] = _log_uniform(rng, 1, 32)
    if op == "gate_up":
        case["act"] = rng.choice(["silu", "gelu_tanh", "gelu_exact"])
        scaled = case["act"] == "silu" and rng.random() < 0.5
        case["gm"] = round(rng.uniform(0.5, 1.5), 3) if scaled else 1.0
        case["dm"] = round(rng.uniform(0.5, 1.5), 3) if scaled else 1.0
    return case


# ---------------------------------------------------------------------------------------------- inputs


def _activations(gen, rows, cols, dtype):
    """Projections as an MLP makes them: about unit size, tokens and channels of different sizes, and the last
    rows of a padded batch all zero."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda"))
    x *= torch.exp(0.5 * torch.randn(1, cols, generator=gen, device="cuda"))
    x[rows - rows // 64:] = 0.0
    return x.to(dtype)


def _weight4(gen, n, k, group, zeros, dtype):
    """A projection of weights about 1/sqrt(k) in size, held in 4 bits."""
    pitch, groups = (k + 31) // 32 * 16, (k + group - 1) // group
    packed = torch.randint(0, 256, (n, pitch), generator=gen, device="cuda", dtype=torch.uint8)
    scales = ((0.6 + 0.8 * torch.rand(n, groups, generator=gen, device="cuda")) / (4.6 * math.sqrt(k))).to(dtype)
    z = torch.randint(5, 11, (n, groups), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    return packed, scales, z


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] in ("step", "recompute"):
        rows, cols = case["rows"], case["cols"]
        gate = _activations(gen, rows, cols, dtype)
        up = _activations(gen, rows, cols, dtype)
        if case["packed"]:
            state["gate_up"] = torch.cat((gate, up), dim=1)
        else:
            state["gate"], state["up"] = gate, up
        state["dh"] = torch.randn(rows, cols, generator=gen, device="cuda").to(dtype)
        return state
    names = ("w_gate", "w_up") if case["op"] == "gate_up" else ("w",)
    for name in names:
        state[name] = _weight4(gen, case["n"], case["k"], case["group"], case["zeros"], dtype)
        if own:
            from kernel_pocs_b200.w4 import W4Weight

            packed, scales, z = state[name]
            state[name] = W4Weight(packed, scales, z, in_features=case["k"], group_size=case["group"])
    if case["op"] != "dequantize":
        state["x"] = _activations(gen, case["m"], case["k"], dtype)
    return state


# ---------------------------------------------------------------------------------------------- the plain form


def _codes(x):
    """The values that the 8-bit codes of ``x`` (float32) stand for."""
    rows, cols = x.shape
    pad = -cols % 32
    v = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, 32)
    top = v.abs().amax(dim=2, keepdim=True)
    # half a step of 127 added to the magnitude's bits carries into the exponent where it would round to 128
    e = ((top.view(torch.int32) + 0x10000) >> 23) - 6
    e = e.clamp(min=1)
    step = (e << 23).view(torch.float32)
    inverse = ((254 - e) << 23).view(torch.float32)
    return (torch.round(v * inverse) * step).view(rows, -1)[:, :cols]


def _act(act, z):
    """The activation and its derivative."""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        s = 1.0 / (1.0 + torch.exp(-2.0 * c * (z + 0.044715 * z * z * z)))
        return z * s, s + z * s * (1.0 - s) * 2.0 * c * (1.0 + 3 * 0.044715 * z * z)
    cdf = 0.5 * torch.erfc(z * -math.sqrt(0.5))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)


def _halves(state):
    if state["packed"]:
        cols = state["cols"]
        return state["gate_up"][:, :cols], state["gate_up"][:, cols:]
    return state["gate"], state["up"]


def _plain_gradients(state, gate, up):
    gm, dm = state["gm"], state["dm"]
    g, u, d = _codes(gate), _codes(up), state["dh"].float() * dm
    a, da = _act(state["act"], g * gm)
    return a * u * dm, d * u * da * gm, d * a


def _plain_weight(w, case):
    packed, scales, z = w
    n, k, group = case["n"], case["k"], case["group"]
    q = torch.stack((packed & 15, packed >> 4), dim=2).view(n, -1)[:, :k].float()
    zero = z.float().repeat_interleave(group, dim=1)[:, :k] if z is not None else 8.0
    return (q - zero) * scales.float().repeat_interleave(group, dim=1)[:, :k]


def _plain(state):
    op, dtype = state["op"], DTYPES[state["dtype"]]
    if op in ("step", "recompute"):
        gate, up = (t.float() for t in _halves(state))
        h, dgate, dup = _plain_gradients(state, gate, up)
        if op == "recompute":
            return h.to(dtype), dgate.to(dtype), dup.to(dtype)
        h = _act(state["act"], gate * state["gm"])[0] * up * state["dm"]
        if state["packed"]:
            return h.to(dtype), torch.cat((dgate, dup), dim=1).to(dtype)
        return h.to(dtype), dgate.to(dtype), dup.to(dtype)
    if op == "dequantize":
        return _plain_weight(state["w"], state).to(dtype)
    x = state["x"].float()
    if op == "linear":
        return (x @ _plain_weight(state["w"], state).t()).to(dtype)
    gate = x @ _plain_weight(state["w_gate"], state).t()
    up = x @ _plain_weight(state["w_up"], state).t()
    return (_act(state["act"], gate * state["gm"])[0] * up * state["dm"]).to(dtype)


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    if not own:
        return _plain(state)
    from kernel_pocs_b200 import checkpoint8, w4

    op = state["op"]
    if op == "step":
        dh = state["dh"]
        if state["packed"]:
            leaf = state["gate_up"].detach().requires_grad_()
            if state["act"] == "silu":
                h = checkpoint8.swiglu_packed_ckpt8(leaf, state["gm"], state["dm"])
            else:
                h = checkpoint8.geglu_packed_ckpt8(leaf, _approximate(state["act"]))
            return (h.detach(), *torch.autograd.grad(h, (leaf,), dh))
        gate, up = state["gate"].detach().requires_grad_(), state["up"].detach().requires_grad_()
        if state["act"] == "silu":
            h = checkpoint8.swiglu_ckpt8(gate, up, state["gm"], state["dm"])
        else:
            h = checkpoint8.geglu_ckpt8(gate, up, _approximate(state["act"]))
        return (h.detach(), *torch.autograd.grad(h, (gate, up), dh))
    if op == "recompute":
        kept = checkpoint8.ckpt8_pack(state["gate"], state["up"], state["act"], state["gm"], state["dm"])
        return checkpoint8.ckpt8_backward_recompute(state["dh"], kept, preserve_inputs=True)
    if op == "dequantize":
        return state["w"].dequantize()
    if op == "linear":
        return w4.w4_linear(state["x"], state["w"])
    return w4.w4_gate_up(state["x"], state["w_gate"], state["w_up"], state["act"], state["gm"], state["dm"])


def _approximate(act):
    return "tanh" if act == "gelu_tanh" else "none"


# ---------------------------------------------------------------------------------------------- the definition


def _exact_codes(x):
    rows, cols = x.shape
    groups = (cols + 31) // 32
    v = torch.zeros(rows, groups * 32, dtype=torch.float64, device=x.device)
    v[:, :cols] = x.double()
    v = v.view(rows, groups, 32)
    top = v.abs().amax(dim=2, keepdim=True)
    exponent = torch.frexp(top).exponent - 7          # the largest magnitude lies in [64, 128) steps of 2^exponent
    exponent = exponent + (torch.ldexp(top, -exponent) >= 127.5)
    exponent = torch.where(top > 0, exponent, -126).clamp(min=-126)
    return torch.ldexp(torch.round(torch.ldexp(v, -exponent)), exponent).reshape(rows, -1)[:, :cols]


def _exact_act(act, z):
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z * z)
    phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    cdf = torch.special.ndtr(z)
    return z * cdf, cdf + z * phi


def _exact_weight(w, case):
    packed, scales, z = (w.packed, w.scales, w.zeros) if own else w
    n, k = case["n"], case["k"]
    value = torch.empty(n, packed.shape[1] * 2, dtype=torch.float64, device=packed.device)
    value[:, 0::2] = (packed % 16).double()
    value[:, 1::2] = (packed // 16).double()
    value = value[:, :k]
    which = torch.arange(k, device=packed.device) // case["group"]
    value -= z.double()[:, which] if z is not None else 8.0
    return value * scales.double()[:, which]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "dequantize":
        return _exact_weight(state["w"], case)
    if op in ("linear", "gate_up"):
        x = state["x"].double()
        if op == "linear":
            return x @ _exact_weight(state["w"], case).t()
        gate = x @ _exact_weight(state["w_gate"], case).t()
        up = x @ _exact_weight(state["w_up"], case).t()
        return _exact_act(case["act"], gate * case["gm"])[0] * up * case["dm"]
    gate, up = _halves(state)
    g, u = _exact_codes(gate), _exact_codes(up)
    a, da = _exact_act(case["act"], g * case["gm"])
    d = state["dh"].double() * case["dm"]
    dgate, dup = d * u * da * case["gm"], d * a
    if op == "recompute":
        return a * u * case["dm"], dgate, dup
    h = _exact_act(case["act"], gate.double() * case["gm"])[0] * up.double() * case["dm"]
    return (h, torch.cat((dgate, dup), dim=1)) if case["packed"] else (h, dgate, dup)


# ---------------------------------------------------------------------------------------------- bytes and operations


def work(case):
    op, size = case["op"], SIZES[case["dtype"]]
    if op in ("step", "recompute"):
        rows, cols = case["rows"], case["cols"]
        n, groups = rows * cols, rows * ((cols + 31) // 32)
        codes = 2 * (n + groups)  # of gate and up, written by the one pass and read by the other
        # step: gate, up -> h; dh -> dgate, dup.  recompute: gate, up; dh -> h, dgate, dup
        return {"bytes": 6 * n * size + 2 * codes, "flops": 40 * n}
    n, k = case["n"], case["k"]
    groups = n * ((k + case["group"] - 1) // case["group"])
    weight = n * k // 2 + groups * (size + (1 if case["zeros"] else 0))
    if op == "dequantize":
        return {"bytes": weight + n * k * size, "flops": 2 * n * k}
    m, count = case["m"], 2 if op == "gate_up" else 1
    return {"bytes": count * weight + m * (k + n) * size, "flops": 2 * m * n * k * count}
