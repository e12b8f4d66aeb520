"""``quantize_blocks`` and ``block_scaled_linear`` against the float64 oracle.

* Quantisation: the same scales and the same e4m3 bytes (both are rounded as torch
  rounds them, so they are equal, not close).
* Product: what ``oracle.block_fp8.product`` allows the MFMA and the fp32 sums, and one
  rounding to bf16 (2^-8).  In the norm the losses of the MFMA average out: the bf16
  rounding alone is 2^-8 / sqrt(3) of the values at most, 2.3e-3.
"""
import math

import pytest
import torch

from oracle import block_fp8 as ob
from oracle.fp8_linear import quantize_weight_blocks
from tokenfactory_amd import block_scaled_linear, quantize_blocks

pytestmark = pytest.mark.gpu


def make_x(rows, cols, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * torch.exp(torch.randn((cols,), generator=g))
    return x.to(dtype)


def make_weight(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((n, k), generator=g) * (torch.rand((n, 1), generator=g) + 0.05)
    return quantize_weight_blocks(w)


def same_bytes(got, want):
    nan = torch.isnan(want.float())
    assert torch.equal(torch.isnan(got.float()), nan)
    diff = (got.view(torch.uint8) != want.view(torch.uint8)) & ~nan
    assert not diff.any(), f"{int(diff.sum())} of {diff.numel()} e4m3 bytes differ"


def check_quant(x):
    q, s = quantize_blocks(x)
    wq, wsc = ob.quantize(x.cpu())
    assert q.shape == x.shape and s.shape == wsc.shape and s.dtype == torch.float32
    gs = s.cpu()
    assert torch.equal(torch.isnan(gs), torch.isnan(wsc))
    assert torch.equal(gs[~torch.isnan(wsc)], wsc[~torch.isnan(wsc)])
    same_bytes(q.cpu(), wq)
    return q, s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 6144), (5, 200), (17, 1000), (64, 136),
                                       (333, 2560), (2, 16384)])
def test_quantize_is_bit_exact(gpu, rows, cols, dtype):
    print(f"[quant] {rows} x {cols} {dtype}", flush=True)
    check_quant(make_x(rows, cols, rows + cols, dtype).to(gpu))


def test_quantize_special_values(gpu):
    print("[quant] special values", flush=True)
    x = make_x(20, 384, 1, torch.float32)
    x[3] = 0.0
    x[4, :128] = 1e-30                  # below the smallest scale's range
    x[5, 130] = 3e38
    x[6, 7] = float("inf")
    x[7, 200] = float("nan")
    x[8, 300] = -float("inf")
    x[9, 0] = -0.0
    x[10, :128] = torch.arange(128) * 1e-3
    check_quant(x.to(gpu))
    check_quant(x.to(torch.bfloat16).to(gpu))


def test_quantize_strided_and_misaligned_rows(gpu):
    print("[quant] strides", flush=True)
    x = make_x(9, 272, 2).to(gpu)
    wide = torch.zeros((9, 400), dtype=torch.bfloat16, device=gpu)
    want_q, want_s = check_quant(x)
    for view in (wide[:, :272], wide[:, 8:280], wide[:, 3:275]):
        view.copy_(x)
        q, s = quantize_blocks(view)
        same_bytes(q, want_q)
        assert torch.equal(s, want_s)
    t = x.t().contiguous().t()          # columns far apart
    same_bytes(quantize_blocks(t)[0], want_q)
    same_bytes(quantize_blocks(x[:1].expand(9, 272))[0][4:5], want_q[:1])


def check_linear(gpu, m, n, k, bias=False, quantized=False, dtype=torch.bfloat16, seed=0):
    print(f"[linear] m={m} n={n} k={k} bias={bias} quantized={quantized} {dtype}", flush=True)
    x = make_x(m, k, seed + m, dtype)
    w, ws = make_weight(n, k, seed + n)
    b = torch.randn(n, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16) if bias \
        else None
    q, s = ob.quantize(x)
    args = (w.to(gpu), ws.to(gpu), None if b is None else b.to(gpu))
    if quantized:
        out = block_scaled_linear(q.to(gpu), *args, x_scale=s.to(gpu))
    else:
        out = block_scaled_linear(x.to(gpu), *args)
    assert out.shape == (m, n) and out.dtype == torch.bfloat16
    dev = gpu if m * n * k > 1e9 else "cpu"
    ref, bound = ob.product(ob.dequantize(q, s).to(dev), ob.dequantize_weight(w, ws).to(dev))
    if b is not None:
        ref = ref + b.double().to(dev)
    err = (out.double().to(dev) - ref).abs()
    bound = 2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * bound + 2.0 ** -22 * ref.abs()
    assert float(err.norm()) <= 2.5e-3 * float(ref.norm())
    assert bool((err <= bound).all()), f"{int((err > bound).sum())} of {err.numel()} outside, " \
        f"worst {(err / bound.clamp(min=1e-300)).max().item():.2f} of the bound"
    return out


# One row to many, tiles cut in every dimension (every tile shape: test_gpu_block_tiles.py).
@pytest.mark.parametrize("m,n,k", [
    (1, 64, 16), (1, 1, 48), (1, 5120, 6144), (1, 40, 17408), (1, 33, 36864), (2, 130, 272),
    (4, 100, 8192), (5, 77, 9008), (16, 48, 12800), (16, 640, 256), (17, 2592, 5120),
    (33, 129, 128), (48, 5120, 1024), (64, 257, 1040), (65, 512, 384), (100, 2592, 1536),
    (129, 384, 2064), (300, 5120, 640), (700, 513, 400), (1030, 1024, 256), (1900, 12288, 640),
    (2100, 640, 512), (4097, 5120, 256), (8192, 2048, 384)])
@pytest.mark.parametrize("quantized", [False, True])
def test_linear(gpu, m, n, k, quantized):
    check_linear(gpu, m, n, k, bias=n % 3 == 0, quantized=quantized)


# More tiles than CUs, the last of them split along K (256 whole of 264, 512 of 539).
@pytest.mark.parametrize("m,n,k", [(1300, 6139, 4096), (1290, 12300, 4000)])
def test_last_round_of_tiles_split(gpu, m, n, k):
    check_linear(gpu, m, n, k, bias=True, quantized=True)


def test_linear_fp32_input_and_leading_dims(gpu):
    check_linear(gpu, 23, 200, 400, dtype=torch.float32)
    x = make_x(24, 400, 5).to(gpu)
    w, ws = (t.to(gpu) for t in make_weight(200, 400, 6))
    want = block_scaled_linear(x, w, ws)
    assert torch.equal(block_scaled_linear(x.view(2, 3, 4, 400), w, ws), want.view(2, 3, 4, 200))
    assert torch.equal(block_scaled_linear(x[0], w, ws), block_scaled_linear(x[:1], w, ws)[0])
    assert block_scaled_linear(x[:0], w, ws).shape == (0, 200)


def test_rows_do_not_depend_on_each_other(gpu):
    """A row's result is the same in any batch that runs the same tiles, and a NaN or
    infinite value stays with its row."""
    x = make_x(80, 1024, 8).to(gpu)
    w, ws = (t.to(gpu) for t in make_weight(384, 1024, 9))
    want = block_scaled_linear(x, w, ws)
    y = x.clone()
    y[7, 100], y[30, 1000], y[79, 0] = float("nan"), float("inf"), -float("inf")
    got = block_scaled_linear(y, w, ws)
    bad = [7, 30, 79]
    good = [i for i in range(80) if i not in bad]
    assert torch.equal(got[good], want[good])
    assert bool(torch.isnan(got[bad]).all())


@pytest.mark.parametrize("m", [3, 200])
def test_nan_weight_stays_with_its_column(gpu, m):
    x = make_x(m, 400, 11).to(gpu)
    w, ws = (t.to(gpu) for t in make_weight(300, 400, 12))
    want = block_scaled_linear(x, w, ws)
    w.view(torch.uint8)[77, 390] = 0x7f
    got = block_scaled_linear(x, w, ws)
    assert bool(torch.isnan(got[:, 77]).all())
    keep = [i for i in range(300) if i != 77]
    assert torch.equal(got[:, keep], want[:, keep])


@pytest.mark.parametrize("m", [5, 150])
def test_linear_strides(gpu, m):
    """Rows of x, its scales, the weight and the weight's scales as they lie."""
    n, k = 260, 512
    q, s = quantize_blocks(make_x(m, k, 13).to(gpu))
    w, ws = (t.to(gpu) for t in make_weight(n, k, 14))
    want = block_scaled_linear(q, w, ws, x_scale=s)
    wide = torch.empty((m, k + 64), dtype=torch.uint8, device=gpu).fill_(0x7f)
    wide[:, 16:16 + k] = q.view(torch.uint8)
    qv = wide.view(torch.float8_e4m3fn)[:, 16:16 + k]
    ww = torch.empty((n, k + 32), dtype=torch.uint8, device=gpu).fill_(0x7f)
    ww[:, :k] = w.view(torch.uint8)
    wv = ww.view(torch.float8_e4m3fn)[:, :k]
    assert torch.equal(block_scaled_linear(qv, wv, ws.t().contiguous().t(),
                                           x_scale=s.contiguous()), want)
    big = torch.full((s.shape[1], m + 9), float("nan"), device=gpu).t()
    big[:m] = s
    assert torch.equal(block_scaled_linear(q, w, ws, x_scale=big[:m]), want)
    with pytest.raises(ValueError):
        block_scaled_linear(q, w, ws, x_scale=s[:, :1])
    with pytest.raises(ValueError):
        block_scaled_linear(q, w, ws)
    with pytest.raises(ValueError):
        block_scaled_linear(q, w.t(), ws, x_scale=s)
    with pytest.raises(NotImplementedError):
        block_scaled_linear(make_x(3, 24, 1).to(gpu), w[:, :24], ws[:, :1])


def test_linear_is_deterministic_and_runs_on_other_streams(gpu):
    x = make_x(40, 2048, 15).to(gpu)
    w, ws = (t.to(gpu) for t in make_weight(512, 2048, 16))
    want = block_scaled_linear(x, w, ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = [block_scaled_linear(x, w, ws, stream=s) for _ in range(3)]
    with torch.cuda.stream(s):
        outs += [block_scaled_linear(x, w, ws) for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_captured_and_replayed(gpu, m):
    x = make_x(m, 1040, 17).to(gpu)
    w, ws = (t.to(gpu) for t in make_weight(640, 1040, 18))
    block_scaled_linear(x, w, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block_scaled_linear(x, w, ws)
    for seed in range(4):
        x.copy_(make_x(m, 1040, 100 + seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, block_scaled_linear(x, w, ws)), f"replay {seed}"


def test_two_graphs_and_eager_calls_share_no_scratch(gpu):
    x = make_x(20, 4096, 19).to(gpu)
    w, ws = (t.to(gpu) for t in make_weight(256, 4096, 20))
    want = block_scaled_linear(x, w, ws)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block_scaled_linear(x, w, ws))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = block_scaled_linear(x, w, ws)
        torch.cuda.synchronize()
        assert torch.equal(eager, want) and all(torch.equal(o, want) for o in outs)


def test_scales_far_apart_do_not_lose_small_blocks(gpu):
    """A block of large values in a row does not cost the other blocks precision."""
    x = make_x(4, 256, 21, torch.float32)
    x[:, :128] *= 1e6
    x[:, 128:] *= 1e-6
    q, s = quantize_blocks(x.to(gpu))
    back = ob.dequantize(q.cpu(), s.cpu())
    rel = ((back - x.double()).norm(dim=1) / x.double().norm(dim=1))
    small = (back[:, 128:] - x[:, 128:].double()).norm(dim=1) / x[:, 128:].double().norm(dim=1)
    # one rounding of e4m3: 2^-4 of a normal value (and of the block's largest / 448 below)
    assert float(rel.max()) <= 2 ** -4 and float(small.max()) <= 2 ** -4
    assert not math.isnan(float(small.max()))


def test_a_copy_of_the_rows_is_made_on_the_calls_stream(gpu):
    """Leading dims that no view flattens: the copy must not run on the current stream,
    which the given one does not wait for."""
    w, ws = (t.to(gpu) for t in make_weight(128, 256, 30))
    base = make_x(64 * 256, 32, 31).to(gpu).view(64, 256, 32)
    x = base.transpose(1, 2)                       # [64, 32, 256]
    want = block_scaled_linear(x.reshape(-1, 256), w, ws).view(64, 32, 128)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    big = torch.zeros(1 << 28, device=gpu)
    for _ in range(40):                            # keeps the current stream busy meanwhile
        big.add_(1.0)
    got = block_scaled_linear(x, w, ws, stream=s)
    with torch.cuda.stream(s):
        same = torch.equal(got, want)              # (waits for the call's stream only)
    assert same
    with pytest.raises(ValueError):
        block_scaled_linear(x[..., :0], w[:, :0], ws[:, :0])


@pytest.mark.parametrize("m", [1, 16, 40, 300])
def test_nothing_behind_quantised_rows_is_used(gpu, m):
    """Rows of a width that ends inside a block, in a wider buffer of NaNs."""
    k = 1040
    q, s = ob.quantize(make_x(m, k, 40))
    w, ws = (t.to(gpu) for t in make_weight(192, k, 41))
    want = block_scaled_linear(q.to(gpu), w, ws, x_scale=s.to(gpu))
    buf = torch.full((m, k + 240), 0x7F, dtype=torch.uint8, device=gpu)
    rows = buf[:, :k]
    rows.copy_(q.view(torch.uint8))
    got = block_scaled_linear(rows.view(torch.float8_e4m3fn), w, ws, x_scale=s.to(gpu))
    assert torch.equal(got, want)
    assert bool((buf[:, k:] == 0x7F).all())
