"""What ``GatedMLP`` takes as its configuration and projections (CPU only)."""
import pytest

from tokenfactory_amd import GatedMLP


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
