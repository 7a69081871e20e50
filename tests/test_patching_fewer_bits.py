"""patch() with the block held in fewer bits: gate and up kept in 8 bits for the backward, projections in 4 bits for
generating, on randomly initialised tiny models (no checkpoint needed)."""
import copy

import pytest
import torch

from kernel_pocs_b200 import patching
from kernel_pocs_b200.fused_mlp import check_status

transformers = pytest.importorskip("transformers")
from tests.test_patching import tiny_gemma2, tiny_qwen3, wrap_mlps  # noqa: E402

gpu = pytest.mark.gpu


def test_orchestration_on_cpu():
    model = patching.patch(tiny_qwen3(), kernels=["swiglu_ckpt8"])
    assert model._forge_patched_counts == {"swiglu_ckpt8": 2}
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        model(torch.randint(0, 512, (1, 8)))
    ids = torch.randint(0, 512, (1, 8))
    assert torch.equal(patching.unpatch(model)(ids).logits, tiny_qwen3()(ids).logits)
    assert patching.patch(tiny_gemma2(), kernels=["geglu_ckpt8"])._forge_patched_counts == {"geglu_ckpt8": 2}
    with pytest.raises(NotImplementedError, match="only supports activation='silu'"):
        patching.patch(tiny_gemma2(), kernels=["swiglu_ckpt8"])

    # 4 bits need 16-bit projections: fp32 ones are left to the next kernel, wrapped ones too
    model = patching.patch(tiny_qwen3(), kernels=["mlp_w4", "swiglu"])
    assert model._forge_patched_counts == {"swiglu": 2}
    model = patching.patch(wrap_mlps(tiny_qwen3(torch.bfloat16)), kernels=["mlp_w4", "lora_mlp"])
    assert model._forge_patched_counts == {"lora_mlp": 2}
    for make in (tiny_qwen3, tiny_gemma2):
        model = patching.patch(make(torch.bfloat16), kernels=["mlp_w4"])
        assert model._forge_patched_counts == {"mlp_w4": 2}
        with pytest.raises(RuntimeError, match="no CPU fallback"), torch.no_grad():
            model(torch.randint(0, 512, (1, 8)))


def _loss_grads(model, ids):
    model.zero_grad()
    out = model(ids, labels=ids)
    out.loss.backward()
    return out.logits.detach(), torch.cat([p.grad.float().flatten() for p in model.parameters() if p.grad is not None])


@gpu
@pytest.mark.parametrize("make,plain,ckpt", [(tiny_qwen3, "swiglu", "swiglu_ckpt8"), (tiny_gemma2, "geglu", "geglu_ckpt8")])
def test_8_bit_checkpoints_in_a_model(make, plain, ckpt):
    ids = torch.randint(0, 512, (2, 48), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    model = make(torch.bfloat16, "cuda")
    logits, grads = _loss_grads(patching.patch(model, kernels=[plain]), ids)
    patching.unpatch(model)
    logits8, grads8 = _loss_grads(patching.patch(model, kernels=[ckpt]), ids)
    assert torch.equal(logits8, logits)                      # the forward does not see the codes
    # a kept value is off by at most half a step, 1/127 of its group's largest magnitude at worst: about 1 % of a
    # standard deviation rms.  Two layers of two such tensors: 3 % of the gradient, a cosine of 1 - 0.03^2 / 2
    cos = torch.nn.functional.cosine_similarity(grads8.double(), grads.double(), dim=0)
    assert float(cos) > 0.9995


@gpu
@pytest.mark.parametrize("make", [tiny_qwen3, tiny_gemma2])
def test_lora_block_with_8_bit_checkpoints_in_a_model(make):
    ids = torch.randint(0, 512, (2, 48), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    model = wrap_mlps(make()).to(device="cuda", dtype=torch.bfloat16)
    logits, grads = _loss_grads(patching.patch(model, kernels=["lora_mlp_fused"]), ids)
    patching.unpatch(model)
    patching.patch(model, kernels=["lora_mlp_fused_ckpt8"])
    assert model._forge_patched_counts == {"lora_mlp_fused_ckpt8": 2}
    logits8, grads8 = _loss_grads(model, ids)
    assert torch.equal(logits8, logits)
    cos = torch.nn.functional.cosine_similarity(grads8.double(), grads.double(), dim=0)
    assert float(cos) > 0.9995
    check_status()


@gpu
@pytest.mark.parametrize("make", [tiny_qwen3, tiny_gemma2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_4_bit_projections_in_a_model_that_generates(make, dtype):
    """A prompt (16-bit path) and then tokens one at a time (4-bit kernels), against the unpatched model whose weights
    are the values the codes stand for."""
    model = make(dtype, "cuda").eval()
    rounded = copy.deepcopy(model)
    from kernel_pocs_b200.w4 import quantize_w4

    for m in rounded.modules():
        if type(m).__name__ in ("Qwen3MLP", "Gemma2MLP"):
            for proj in (m.gate_proj, m.up_proj, m.down_proj):
                proj.weight.data.copy_(quantize_w4(proj.weight).dequantize())
    patching.patch(model, kernels=["mlp_w4"])
    ids = torch.randint(0, 512, (2, 60), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    with torch.no_grad():
        past = past_r = None
        for part in (ids, *(torch.full((2, 1), t, device="cuda") for t in (3, 77, 400))):
            out = model(part, past_key_values=past, use_cache=True)
            ref = rounded(part, past_key_values=past_r, use_cache=True)
            past, past_r = out.past_key_values, ref.past_key_values
            a, b = out.logits.double().flatten(), ref.logits.double().flatten()
            assert bool(torch.isfinite(a).all())
            assert float(torch.nn.functional.cosine_similarity(a, b, dim=0)) > 0.999
            assert float((a - b).abs().max()) < 1.0
    check_status()
    with pytest.raises(RuntimeError, match="forward only"):
        model(ids)
    patching.unpatch(model)
    assert model(ids).logits.requires_grad


@gpu
def test_patched_on_the_host_and_moved():
    model = patching.patch(tiny_qwen3(torch.bfloat16), kernels=["mlp_w4"]).to("cuda").eval()
    direct = patching.patch(tiny_qwen3(torch.bfloat16, "cuda"), kernels=["mlp_w4"]).eval()
    ids = torch.randint(0, 512, (1, 5), device="cuda")
    with torch.no_grad():
        assert torch.equal(model(ids).logits, direct(ids).logits)
