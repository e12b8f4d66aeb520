"""``Fp8Linear`` on rows that come quantised with a scale per 128 columns."""
import pytest
import torch

from oracle import block_fp8 as ob
from tokenfactory_amd import Fp8Linear, add_rms_norm, block_scaled_linear


def rows(m, k, device="cpu"):
    return (torch.zeros((m, k), dtype=torch.float8_e4m3fn, device=device),
            torch.ones((m, -(-k // 128)), device=device))


def test_refusals():
    q, s = rows(4, 256)
    with pytest.raises(NotImplementedError, match="128 x 128"):
        Fp8Linear(256, 64, block_size=(64, 128))(q, x_scale=s)
    with pytest.raises(ValueError, match="amax"):
        Fp8Linear(256, 64)(q, torch.zeros((1,), dtype=torch.int32), s)
    with pytest.raises(ValueError):     # (the tensors lie on the CPU)
        Fp8Linear(256, 64)(q, x_scale=s)


@pytest.mark.gpu
@pytest.mark.parametrize("m,bias", [(1, False), (7, True), (40, False), (300, True)])
def test_a_projection_of_a_quantised_norm(gpu, m, bias):
    """The hand-over of a norm's result to a module's projection."""
    print(f"[fp8 linear] quantised rows m={m}", flush=True)
    g = torch.Generator().manual_seed(m)
    lin = Fp8Linear(400, 200, bias=bias).to(gpu)
    lin.quantize_from(torch.randn((200, 400), generator=g).to(gpu))
    if bias:
        lin.bias.copy_(torch.randn((200,), generator=g).to(gpu))
    x = torch.randn((m, 400), generator=g).to(torch.bfloat16).to(gpu)
    (q, s), _ = add_rms_norm(x, None, torch.ones(400, device=gpu), quantize=True)
    out = lin(q, x_scale=s)
    assert torch.equal(out, block_scaled_linear(q, lin.weight, lin.weight_scale_inv, lin.bias,
                                                x_scale=s))
    ref, bound = ob.product(ob.dequantize(q.cpu(), s.cpu()),
                            ob.dequantize_weight(lin.weight.cpu(), lin.weight_scale_inv.cpu()))
    ref = ref if not bias else ref + lin.bias.double().cpu()
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= 2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * bound + 2.0 ** -22 * ref.abs()).all())
    with pytest.raises(ValueError):
        lin(q)                          # scales go with quantised rows
    with pytest.raises(ValueError):
        lin(x, x_scale=s)
