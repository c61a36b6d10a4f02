"""The option saved_activations where the fused LoRA-MLP is asked for it."""
import pytest
import torch

pytest.importorskip("transformers")


@pytest.mark.parametrize("arch", ["qwen3", "gemma2"])
def test_lora_mlp_refuses_what_it_does_not_do(arch):
    """The fused LoRA-MLP saves gate and up as they are: asked for 8 bits it
    names the kernels that keep them; another value is an error, as in those."""
    from test_patch_adapters import build

    from forge.patching import FORWARD_MAKERS

    m, _ = build(arch, "mlp")
    with pytest.raises(ValueError, match="saved_activations must be"):
        FORWARD_MAKERS["lora_mlp"](m, {"saved_activations": "4bit"})
    with pytest.raises(NotImplementedError, match="'swiglu' or 'geglu'"):
        FORWARD_MAKERS["lora_mlp"](m, {"saved_activations": "8bit"})
    FORWARD_MAKERS["lora_mlp"](m, {"saved_activations": None})
    # those take the same module
    FORWARD_MAKERS["swiglu" if arch == "qwen3" else "geglu"](m, {"saved_activations": "8bit"})


@pytest.mark.gpu
def test_8_bits_of_a_lora_mlp_through_the_swiglu_adapter():
    import copy

    from test_patch_adapters import _run, build

    from forge.patching import FORWARD_MAKERS

    m, _ = build("qwen3", "mlp", dtype=torch.bfloat16, device="cuda")
    plain = copy.deepcopy(m)
    m.forward = FORWARD_MAKERS["swiglu"](m, {"saved_activations": "8bit"})
    x, dy = (torch.randn(2, 37, 512, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    got, want = _run(m, x, (), "mlp", dy), _run(plain, x, (), "mlp", dy)
    # 16-bit products and activations on one side, 1/127 of a group's largest at most on gate and up on the other
    for a, b in zip((got[0], got[1], *got[2]), (want[0], want[1], *want[2])):
        assert (a.float() - b.float()).norm() <= 2e-2 * b.float().norm()
