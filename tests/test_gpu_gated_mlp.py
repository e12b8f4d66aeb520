"""``gated_mlp`` and ``GatedMLP`` against the float64 oracle.

The hidden activations are rounded to e4m3 from fp32 sums.  The oracle rounds them
from exact sums and says for each of them what the products' arithmetic may make of
it: mostly nothing, a step of e4m3 for those next to a border.  The outputs may
differ by those steps through the down weight, the last product's own arithmetic
and one bf16 rounding.  In the norm: a product off by d moves a value of spacing p
by p with probability d / p, sqrt(d p) in the mean square; with d = 1e-4 and p = 1/8
3.5e-3, and 2.3e-3 for the bf16 rounding: 4.2e-3 together.
"""
import pytest
import torch

from oracle import block_fp8 as ob
from tests.test_gpu_block_fp8 import make_weight, make_x
from tokenfactory_amd import Fp8Linear, GatedMLP, gated_mlp, quantize_blocks

pytestmark = pytest.mark.gpu


def make_mlp(hidden, inter, n, seed, device):
    ws = [make_weight(r, k, seed + i) for i, (r, k) in
          enumerate(((inter, hidden), (inter, hidden), (n, inter)))]
    # sums of some units: silu's curved part
    ws = [(q, s * (4.0 / k ** 0.5)) for (q, s), k in zip(ws, (hidden, hidden, inter))]
    return ws, [t.to(device) for pair in ws for t in pair]


def check(gpu, m, hidden, inter, n=None, quantized=False, dtype=torch.bfloat16, seed=0):
    n = n or hidden
    print(f"[mlp] m={m} {hidden} -> {inter} -> {n} quantized={quantized} {dtype}", flush=True)
    x = make_x(m, hidden, seed + m, dtype)
    host, dev = make_mlp(hidden, inter, n, seed + inter, gpu)
    q, s = ob.quantize(x)
    if quantized:
        out = gated_mlp(q.to(gpu), *dev, x_scale=s.to(gpu))
    else:
        out = gated_mlp(x.to(gpu), *dev)
    assert out.shape == (m, n) and out.dtype == torch.bfloat16
    compare(out.double().cpu(), ob.dequantize(q, s), host)
    return out


def compare(out, x, host):
    wg, wu, wd = (ob.dequantize_weight(*p) for p in host)
    h, off = ob.gated_hidden(x, wg, wu)
    ref, bound = ob.product(h, wd)
    bound = 2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * (bound + off @ wd.abs().t()) \
        + 2.0 ** -22 * ref.abs()
    err = (out - ref).abs()
    assert bool((err <= bound).all()), f"{int((err > bound).sum())} of {err.numel()} outside, " \
        f"worst {(err / bound.clamp(min=1e-300)).max().item():.2f} of the bound"
    assert float(err.norm()) <= 4.2e-3 * float(ref.norm())


# One row to several tiles of rows; widths that end inside a block and a tile.
@pytest.mark.parametrize("m,hidden,inter", [
    (1, 16, 16), (1, 256, 1024), (1, 5120, 640), (1, 512, 8192), (2, 272, 400),
    (4, 1024, 4112), (7, 512, 8192), (16, 512, 1040), (17, 1024, 512),
    (48, 640, 1152), (64, 384, 272), (65, 256, 2176), (130, 1040, 384), (200, 512, 528),
    (333, 1024, 2176), (520, 256, 640), (1100, 256, 512)])
@pytest.mark.parametrize("quantized", [False, True])
def test_gated_mlp(gpu, m, hidden, inter, quantized):
    check(gpu, m, hidden, inter, quantized=quantized)


def test_other_output_width_fp32_input_and_leading_dims(gpu):
    check(gpu, 9, 256, 384, n=77)
    check(gpu, 260, 256, 384, n=513, dtype=torch.float32)
    x = make_x(12, 256, 5).to(gpu)
    _, dev = make_mlp(256, 384, 256, 6, gpu)
    want = gated_mlp(x, *dev)
    assert torch.equal(gated_mlp(x.view(3, 4, 256), *dev), want.view(3, 4, 256))
    assert gated_mlp(x[:0], *dev).shape == (0, 256)


@pytest.mark.parametrize("m", [1500, 3000, 6000])
def test_large_tiles(gpu, m):
    """The tiles of long prompts: rows spread over all of them (23 divides no tile)."""
    hidden, inter = 512, 4096
    print(f"[mlp] large m={m} {hidden} -> {inter}", flush=True)
    host, dev = make_mlp(hidden, inter, hidden, 3, gpu)
    x = make_x(m, hidden, m)
    out = gated_mlp(x.to(gpu), *dev)
    rows = sorted(set(range(0, m, 23)) | {m - 1})
    compare(out[rows].double().cpu(), ob.dequantize(*ob.quantize(x[rows])), host)


def test_padding_rows_and_odd_values_stay_with_their_rows(gpu):
    for m in (40, 300):
        x = make_x(m, 384, 8).to(gpu)
        _, dev = make_mlp(384, 640, 384, 9, gpu)
        want = gated_mlp(x, *dev)
        y = x.clone()
        y[5], y[11, 3], y[m - 1, 380] = 0.0, float("nan"), float("inf")
        got = gated_mlp(y, *dev)
        keep = [i for i in range(m) if i not in (5, 11, m - 1)]
        assert torch.equal(got[keep], want[keep])
        assert not got[5].any() and bool(torch.isnan(got[[11, m - 1]]).all())


def test_large_gates_saturate_silu(gpu):
    """silu far from zero: 0 below, the value itself above, no overflow."""
    hidden = inter = 128
    eye = torch.eye(128)
    q = (eye * 448).to(torch.float8_e4m3fn)
    one = torch.full((1, 1), 1 / 448)
    x = torch.zeros((2, hidden))
    x[0, :4] = torch.tensor([448.0, -448.0, 224.0, -224.0])
    x[1, :2] = torch.tensor([-3e30, 3e30])
    out = gated_mlp(x.to(torch.bfloat16).to(gpu), *(t.to(gpu) for t in (q, one) * 3)).cpu().float()
    want = torch.zeros((inter,))
    want[0], want[2] = 448.0 ** 2, 224.0 ** 2
    assert torch.allclose(out[0], want, rtol=2 ** -4, atol=1e-3)
    assert float(out[1, 0]) == 0.0 or float(out[1, 0]) != float(out[1, 0])


@pytest.mark.parametrize("m", [1, 40, 400])
def test_captured_and_replayed(gpu, m):
    x = make_x(m, 512, 17).to(gpu)
    _, dev = make_mlp(512, 1040, 512, 18, gpu)
    gated_mlp(x, *dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gated_mlp(x, *dev)
    for seed in range(4):
        x.copy_(make_x(m, 512, 100 + seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gated_mlp(x, *dev)), f"replay {seed}"


def test_module_loads_a_reference_layer(gpu):
    class Config:
        hidden_size, intermediate_size = 256, 512
        quantization_config = {"quant_method": "fp8", "weight_block_size": [128, 128]}
    mlp = GatedMLP(Config()).to(gpu)
    g = torch.Generator().manual_seed(4)
    for lin in (mlp.gate_proj, mlp.up_proj, mlp.down_proj):
        assert isinstance(lin, Fp8Linear)
        lin.quantize_from(torch.randn((lin.out_features, lin.in_features), generator=g).to(gpu) / 16)
    x = make_x(33, 256, 6).to(gpu)
    out = mlp(x)
    q, s = quantize_blocks(x)
    assert torch.equal(mlp(q, s), out)
    h = torch.nn.functional.silu(x.float() @ mlp.gate_proj.dequantize_weight(torch.float32).t())
    h = h * (x.float() @ mlp.up_proj.dequantize_weight(torch.float32).t())
    plain = h @ mlp.down_proj.dequantize_weight(torch.float32).t()
    # against the unquantised block: e4m3 roundings of x and h, 2^-4 at most each
    assert float((out.float() - plain).norm() / plain.norm()) < 0.1
    with pytest.raises(ValueError):
        gated_mlp(x, *[t for lin in (mlp.gate_proj, mlp.down_proj, mlp.down_proj)
                       for t in (lin.weight, lin.weight_scale_inv)])


@pytest.mark.parametrize("m", [4, 30, 300])
def test_nothing_behind_quantised_rows_is_used(gpu, m):
    q, s = ob.quantize(make_x(m, 400, 50))
    _, dev = make_mlp(400, 272, 96, 51, gpu)
    want = gated_mlp(q.to(gpu), *dev, x_scale=s.to(gpu))
    buf = torch.full((m, 640), 0x7F, dtype=torch.uint8, device=gpu)
    rows = buf[:, 16:416]
    rows.copy_(q.view(torch.uint8))
    assert torch.equal(gated_mlp(rows.view(torch.float8_e4m3fn), *dev, x_scale=s.to(gpu)), want)
