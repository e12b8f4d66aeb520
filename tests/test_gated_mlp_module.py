"""What ``GatedMLP`` takes as its configuration and projections (CPU only)."""
import pytest
import torch
import torch.nn as nn

from tokenfactory_amd import Fp8Linear, GatedMLP


class Config:
    hidden_size = 256
    intermediate_size = 17408
    quantization_config = {"quant_method": "fp8", "weight_block_size": [128, 128]}


def config(**kw):
    return type("C", (Config,), kw)()


@pytest.mark.parametrize("tp", [16, 32])
def test_a_share_that_cuts_a_block_of_the_weights_is_refused(tp):
    """17408 / 16 = 1088 = 8.5 blocks: rank 1's rows 0 to 127 have two scales each."""
    with pytest.raises(NotImplementedError, match="128"):
        GatedMLP(config(tp_size=tp))


def test_whole_blocks_and_unshared_widths_are_taken():
    assert GatedMLP(config(tp_size=8)).down_proj.weight.shape == (256, 2176)
    assert GatedMLP(config(intermediate_size=1088)).up_proj.weight.shape == (1088, 256)
    assert GatedMLP(config(intermediate_size=1088, tp_size=1)).up_proj.weight.shape == (1088, 256)


def altered(mlp, how):
    proj = mlp.up_proj
    if how == "hook":
        proj.register_forward_hook(lambda m, i, o: o)
    elif how == "pre-hook":
        proj.register_forward_pre_hook(lambda m, i: i)
    elif how == "forward":
        proj.forward = lambda x: x
    elif how == "subclass":
        mlp.up_proj = type("Adapted", (Fp8Linear,), {})(256, 512)
    elif how == "other module":
        mlp.up_proj = nn.Linear(256, 512, bias=False)
    elif how == "bias":
        mlp.up_proj = Fp8Linear(256, 512, bias=True)
    elif how == "blocks":
        mlp.up_proj = Fp8Linear(256, 512, block_size=(64, 64))
    return mlp


@pytest.mark.parametrize("how", ["hook", "pre-hook", "forward", "subclass", "other module", "bias",
                                 "blocks"])
def test_a_projection_that_does_more_is_not_passed_by(how):
    """The block reads the weights and calls no module."""
    mlp = altered(GatedMLP(config(intermediate_size=512)), how)
    with pytest.raises(NotImplementedError, match="up_proj"):
        mlp(torch.zeros((2, 256), dtype=torch.bfloat16))


def test_plain_projections_are_read():
    mlp = GatedMLP(config(intermediate_size=512))
    handle = mlp.gate_proj.register_forward_hook(lambda m, i, o: o)
    handle.remove()
    with pytest.raises(ValueError):     # (the tensors lie on the CPU)
        mlp(torch.zeros((2, 256), dtype=torch.bfloat16))


def test_a_loaders_parameter_class_is_read():
    """A weight is read where it lies, whatever class of parameter holds it."""
    mlp = GatedMLP(config(intermediate_size=512))
    loaded = type("Loaded", (nn.Parameter,), {})
    mlp.up_proj.weight = loaded(mlp.up_proj.weight.data, requires_grad=False)
    with pytest.raises(ValueError):     # (the tensors lie on the CPU)
        mlp(torch.zeros((2, 256), dtype=torch.bfloat16))
