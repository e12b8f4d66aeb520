"""The block-scaled operators and norms record no gradients: operands that ask for one
are refused while autograd records, instead of results that are cut off from them."""
import pytest
import torch

from tokenfactory_amd import add_rms_norm, block_scaled_linear, gated_mlp, quantize_blocks


def ones(*shape, grad=False, dtype=torch.float32):
    return torch.ones(shape, dtype=dtype, requires_grad=grad)


def fp8(*shape):
    return torch.zeros(shape, dtype=torch.float8_e4m3fn)


def calls(device):
    """(name, a call whose operand of that name asks for a gradient)"""
    put = lambda t: t.detach().to(device).requires_grad_(t.requires_grad)
    x = lambda g=False: put(ones(4, 256, grad=g, dtype=torch.bfloat16))
    w, s = fp8(128, 256).to(device), put(ones(1, 2))
    d, ds = fp8(256, 128).to(device), put(ones(2, 1))
    v = lambda g=False: put(ones(256, grad=g))
    sg = put(ones(1, 2, grad=True))
    bias = put(ones(128, grad=True, dtype=torch.bfloat16))
    return {
        "quantize x": lambda: quantize_blocks(x(True)),
        "linear x": lambda: block_scaled_linear(x(True), w, s),
        "linear bias": lambda: block_scaled_linear(x(), w, s, bias),
        "linear scales": lambda: block_scaled_linear(x(), w, sg),
        "mlp x": lambda: gated_mlp(x(True), w, s, w, s, d, ds),
        "mlp scales": lambda: gated_mlp(x(), w, s, w, sg, d, ds),
        "norm x": lambda: add_rms_norm(x(True), None, v()),
        "norm residual": lambda: add_rms_norm(x(), x(True), v()),
        "norm weight": lambda: add_rms_norm(x(), x(), v(True)),
        "norm post_weight": lambda: add_rms_norm(x(), x(), v(), post_weight=v(True)),
        "norm gate": lambda: add_rms_norm(x(), x(), v(), gate=v(True)),
        "norm in place": lambda: add_rms_norm(x(), x(True), v(), inplace=True),
    }


@pytest.mark.parametrize("name", calls("cpu"))
def test_refused_while_autograd_records(name):
    with pytest.raises(NotImplementedError, match="gradient"):
        calls("cpu")[name]()
    with torch.no_grad(), pytest.raises(ValueError):      # (the tensors lie on the CPU)
        calls("cpu")[name]()


@pytest.mark.gpu
@pytest.mark.parametrize("name", calls("cpu"))
def test_runs_where_autograd_does_not(gpu, name):
    print(f"[no gradients] {name}", flush=True)
    call = calls(gpu)[name]
    with pytest.raises(NotImplementedError, match="gradient"):
        call()
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            call()


@pytest.mark.gpu
def test_autograd_sees_a_residual_summed_in_place(gpu):
    """A backward pass that needs the values that were there says so."""
    leaf = torch.ones((4, 256), device=gpu, requires_grad=True)
    residual = leaf * 2.0
    loss = (residual * residual).sum()            # keeps residual for its backward pass
    x = torch.ones((4, 256), dtype=torch.bfloat16, device=gpu)
    with torch.no_grad():
        _, r = add_rms_norm(x, residual, None, inplace=True)
    assert r is residual and float(residual.detach()[0, 0]) == 3.0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
