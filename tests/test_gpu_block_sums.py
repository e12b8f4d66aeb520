"""How the block-scaled products add: exactly (fp32) up to the documented numbers of
rows, within the documented cut of the fp8 MFMA above.

Terms that cancel show it: 448 * 448 - 448 * 448 beside products of 1.  In fp32 every
partial sum is a whole number below 2^24, so the small products are all that is left;
cut 13 bits below 2^17 they are gone.  Both pairs of large terms stand in each group of
eight, so that no order of the columns inside a group of 128 separates them."""
import pytest
import torch

from tokenfactory_amd import block_scaled_linear, gated_mlp

pytestmark = pytest.mark.gpu
K = 256


def cancelling(rows, gpu):
    """x, its scales, one weight row: in each group of 8 columns two products of 448^2
    that cancel and six of 1, so that a row's sum is 6 K / 8."""
    x = torch.ones((rows, K // 8, 8))
    x[:, :, :2] = 448.0
    w = torch.ones((1, K // 8, 8))
    w[:, :, 0], w[:, :, 1] = 448.0, -448.0
    one = torch.ones((rows, K // 128), device=gpu).t().contiguous().t()
    e4m3 = lambda t: t.view(-1, K).to(torch.float8_e4m3fn).to(gpu)
    return e4m3(x), one, e4m3(w)


@pytest.mark.parametrize("m", [1, 2, 5, 16])
def test_few_rows_add_in_fp32(gpu, m):
    x, xs, w = cancelling(m, gpu)
    out = block_scaled_linear(x, w.expand(40, K).contiguous(), torch.ones((1, 2), device=gpu),
                              x_scale=xs)
    assert bool((out == 6.0 * K / 8).all())


@pytest.mark.parametrize("m", [17, 64, 65, 300])
def test_more_rows_stay_within_the_cut(gpu, m):
    x, xs, w = cancelling(m, gpu)
    out = block_scaled_linear(x, w.expand(40, K).contiguous(), torch.ones((1, 2), device=gpu),
                              x_scale=xs)
    # 2^-10 of 448^2 for each of the K / 8 groups, and one rounding to bf16
    bound = 2.0 ** -10 * 448.0 ** 2 * K / 8
    assert bool(((out.float() - 6.0 * K / 8).abs() <= (1 + 2.0 ** -8) * bound + 1.0).all())


@pytest.mark.parametrize("m", [1, 16, 17, 40, 64])
@pytest.mark.parametrize("inter", [128, 2176])
def test_gate_and_up_add_in_fp32_up_to_64_rows(gpu, m, inter):
    """h = silu(192 / 64) * 192 / 64 in every column, a block's largest, so e4m3 takes
    it as 448 and its scale as h / 448; down takes one column, a power of two away."""
    x, xs, w = cancelling(m, gpu)
    gate = w.expand(inter, K).contiguous()
    scale = torch.full((-(-inter // 128), 2), 1.0 / 64, device=gpu)
    down = torch.zeros((16, inter), device=gpu)
    down[:, 5] = 1.0
    out = gated_mlp(x, gate, scale, gate, scale, down.to(torch.float8_e4m3fn),
                    torch.ones((1, inter // 128), device=gpu), x_scale=xs)
    v = torch.tensor(3.0, dtype=torch.float64)
    h = float(v / (1 + torch.exp(-v)) * v)
    # h: some ten roundings of 2^-24, its scale one; the output one of bf16
    assert bool(((out.double() - h).abs() <= (2.0 ** -8 + 2.0 ** -19) * h).all())
