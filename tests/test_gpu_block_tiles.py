"""Every tile of the block-scaled products against the float64 oracle, which runs on
the GPU here: each shape of ``csrc/block_plan.h``, whole tiles, tiles split along K
and both in one launch, the gate and up products fused or left as partials, with and
without the wide operands.  ``test_block_plan.py`` says (without a GPU) that these
sizes reach all of them.  The tolerances are those of ``test_gpu_block_fp8.py`` and
``test_gpu_gated_mlp.py``.
"""
import pytest
import torch

from oracle import block_fp8 as ob
from tokenfactory_amd import block_scaled_linear, gated_mlp

pytestmark = pytest.mark.gpu

# rows, columns, K
LINEAR = [
    (17, 100, 272), (17, 100, 1040), (48, 5120, 2176), (1345, 644, 400), (1027, 131, 1936),
    (1675, 2326, 8864), (1220, 1545, 912), (641, 899, 6736), (2497, 1540, 9104), (17, 100, 128),
    (19, 100, 912), (7229, 2051, 912), (2314, 1667, 2064), (900, 1281, 8496), (8193, 769, 128),
    (5470, 259, 9488), (7214, 6660, 656), (12305, 769, 128), (1933, 2049, 12960),
    (5006, 3079, 1168),
    # a verify step's and a prompt's projections, the down products of a decode batch
    (77, 2592, 5120), (48, 5120, 17408), (1900, 12288, 5120)]
# rows, hidden, intermediate
GATED = [
    (17, 1296, 8208), (17, 528, 96), (33, 1952, 8224), (33, 1040, 2704), (17, 128, 96),
    (769, 2064, 528), (65, 528, 96), (1345, 2320, 272), (673, 1168, 272), (65, 144, 96),
    (1352, 2448, 288), (1793, 656, 1040), (4107, 12816, 656), (65, 656, 96), (6150, 6432, 272),
    (1203, 6416, 544), (65, 128, 96), (5453, 14944, 656), (2711, 6592, 656), (3654, 128, 1552),
    (2311, 19472, 2448), (2700, 7968, 656)]
# A 27B layer's block and one rank's share of it: sampled rows.
LAYER = [(48, 5120, 17408), (65, 5120, 17408), (100, 5120, 17408), (200, 5120, 17408),
         (1024, 5120, 17408), (8192, 5120, 17408), (64, 5120, 2176), (128, 5120, 2176),
         (333, 5120, 2176)]


def rows_of(m, cols, seed, gpu):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randn((m, cols), generator=g, device=gpu)
    return (x * torch.exp(torch.randn((cols,), generator=g, device=gpu))).to(torch.bfloat16)


def weight(n, k, seed, gpu):
    """e4m3 values and fp32 scales that make sums of some units."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    q = (100 * torch.randn((n, k), generator=g, device=gpu)).clamp(-448, 448)
    s = torch.rand((-(-n // 128), -(-k // 128)), generator=g, device=gpu) + 0.5
    return q.to(torch.float8_e4m3fn), s * (0.02 / k ** 0.5)


def close(out, ref, bound, norm):
    err = (out.double() - ref).abs()
    bound = 2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * bound + 2.0 ** -22 * ref.abs()
    assert bool((err <= bound).all()), f"{int((err > bound).sum())} of {err.numel()} outside, " \
        f"worst {(err / bound.clamp(min=1e-300)).max().item():.2f} of the bound"
    assert float(err.norm()) <= norm * float(ref.norm())


@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear(gpu, m, n, k):
    print(f"[tiles] linear m={m} n={n} k={k}", flush=True)
    x, (w, ws) = rows_of(m, k, m + k, gpu), weight(n, k, n, gpu)
    q, s = ob.quantize(x)
    out = block_scaled_linear(q, w, ws, x_scale=s)
    close(out, *ob.product(ob.dequantize(q, s), ob.dequantize_weight(w, ws)), 2.5e-3)
    assert torch.equal(block_scaled_linear(x, w, ws), out)


def check_gated(gpu, m, hidden, inter, n, rows):
    x = rows_of(m, hidden, m + inter, gpu)
    mats = [weight(r, c, i, gpu) for i, (r, c) in enumerate(
        ((inter, hidden), (inter, hidden), (n, inter)))]
    q, s = ob.quantize(x)
    out = gated_mlp(q, *(t for pair in mats for t in pair), x_scale=s)
    wg, wu, wd = (ob.dequantize_weight(*p) for p in mats)
    h, off = ob.gated_hidden(ob.dequantize(q[rows], s[rows]), wg, wu)
    ref, bound = ob.product(h, wd)
    close(out[rows], ref, bound + off @ wd.abs().t(), 4.2e-3)


@pytest.mark.parametrize("m,hidden,inter", GATED)
def test_gated(gpu, m, hidden, inter):
    print(f"[tiles] gated m={m} {hidden} / {inter}", flush=True)
    check_gated(gpu, m, hidden, inter, 100, torch.arange(m, device=gpu))


@pytest.mark.parametrize("m,hidden,inter", LAYER)
def test_layer(gpu, m, hidden, inter):
    """Rows spread over the tiles (no step divides a tile) and the last."""
    print(f"[tiles] layer m={m} {hidden} / {inter}", flush=True)
    rows = sorted({*range(0, m, max(1, m // 50) | 1), m - 1})
    check_gated(gpu, m, hidden, inter, hidden, torch.tensor(rows, device=gpu))
