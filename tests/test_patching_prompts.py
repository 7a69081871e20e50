"""A model with 4-bit projections that reads prompts of more tokens than the 4-bit kernels are for, then generates."""
import copy

import pytest
import torch

from kernel_pocs_b200 import patching, w4
from kernel_pocs_b200.fused_mlp import check_status

transformers = pytest.importorskip("transformers")
from tests.test_patching import tiny_gemma2, tiny_qwen3  # noqa: E402

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("make", [tiny_qwen3, tiny_gemma2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch", [2, 5, 10])
def test_prompts_on_both_sides_of_the_limits(make, dtype, batch):
    """120 tokens take the 4-bit kernels, 300 those of gate and up and a written-out down projection, 600 written-out weights
    throughout; against the unpatched model whose weights are the values the codes stand for."""
    tokens = batch * 60
    assert (tokens > w4.GATE_UP_ROWS) == (batch == 10) and (tokens > w4.LINEAR_ROWS) == (batch != 2)
    model = make(dtype, "cuda").eval()
    rounded = copy.deepcopy(model)
    for m in rounded.modules():
        if type(m).__name__ in ("Qwen3MLP", "Gemma2MLP"):
            for proj in (m.gate_proj, m.up_proj, m.down_proj):
                proj.weight.data.copy_(w4.quantize_w4(proj.weight).dequantize())
    patching.patch(model, kernels=["mlp_w4"])
    ids = torch.randint(0, 512, (batch, 60), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    with torch.no_grad():
        past = past_r = None
        for part in (ids, *(torch.full((batch, 1), t, device="cuda") for t in (3, 77))):
            out = model(part, past_key_values=past, use_cache=True)
            ref = rounded(part, past_key_values=past_r, use_cache=True)
            past, past_r = out.past_key_values, ref.past_key_values
            a, b = out.logits.double().flatten(), ref.logits.double().flatten()
            assert bool(torch.isfinite(a).all())
            # two models in 16 bits that round in different places
            assert float(torch.nn.functional.cosine_similarity(a, b, dim=0)) > 0.999
            assert float((a - b).abs().max()) < 1.0
    check_status()
