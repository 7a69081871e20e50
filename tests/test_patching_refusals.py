"""What patch() and the patched blocks refuse, and that a refusal leaves the model as it was."""
import pytest
import torch

from kernel_pocs_b200 import patching

transformers = pytest.importorskip("transformers")
from tests.test_patching import tiny_gemma2, tiny_qwen3  # noqa: E402

gpu = pytest.mark.gpu


def _freeze_all_but(model, name):
    for n, p in model.named_parameters():
        p.requires_grad_(name in n)
    return model


@pytest.mark.parametrize("make", [tiny_qwen3, tiny_gemma2])
@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj"])
def test_4_bit_projections_do_not_train(make, name):
    """With nothing trainable before an MLP its input wants no gradient, but its weights would get none either."""
    model = patching.patch(_freeze_all_but(make(torch.bfloat16), name), kernels=["mlp_w4"])
    ids = torch.randint(0, 512, (1, 8))
    with pytest.raises(RuntimeError, match="forward only"):
        model(ids)
    with pytest.raises(RuntimeError, match="no CPU fallback"), torch.no_grad():
        model(ids)
    _freeze_all_but(model, "nothing")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        model(ids)


@gpu
def test_frozen_4_bit_projections_run_with_gradients_enabled():
    model = patching.patch(_freeze_all_but(tiny_qwen3(torch.bfloat16, "cuda"), "lm_head"), kernels=["mlp_w4"])
    ids = torch.randint(0, 512, (1, 8), device="cuda")
    model(ids, labels=ids).loss.backward()
    assert all((p.grad is not None) == p.requires_grad for p in model.parameters())
    for p in model.model.layers[0].mlp.parameters():
        p.requires_grad_()
    with pytest.raises(RuntimeError, match="forward only"):
        model(ids)


@pytest.mark.parametrize("make", [tiny_qwen3, tiny_gemma2])
def test_a_patch_that_fails_leaves_the_model_as_it_was(make):
    """The second layer cannot be quantised: nothing of the first one stays behind, and the model can be patched anew."""
    model = make(torch.bfloat16)
    mlp = model.model.layers[1].mlp
    with torch.no_grad():
        kept = mlp.down_proj.weight[3, 5].clone()
        mlp.down_proj.weight[3, 5] = float("nan")
    with pytest.raises(ValueError, match="not finite"):
        patching.patch(model, kernels=["mlp_w4"])
    assert all("forward" not in vars(layer.mlp) for layer in model.model.layers)
    assert not hasattr(model, "_forge_originals") and not getattr(model, "_forge_patched", False)
    with torch.no_grad():
        mlp.down_proj.weight[3, 5] = kept
    assert patching.patch(model, kernels=["mlp_w4"])._forge_patched_counts == {"mlp_w4": 2}
