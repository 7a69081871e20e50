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
