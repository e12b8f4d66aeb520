"""``add_rms_norm`` against the float64 oracle.

fp32 arithmetic: a mean square over up to 16384 columns is summed 16 values per
thread at a time and then over lanes and waves (a relative error of at most some 40
roundings of 2^-24), rms and the products add a few more: 2^-18 of the value covers
y, 2^-20 of the terms' sizes r.  Each result is rounded once to its type (bf16
2^-8, e4m3 2^-4 of a normal value and half a step of 2^-9 scales below).
"""
import itertools

import pytest
import torch

from oracle import block_fp8 as ob
from tests.test_gpu_block_fp8 import make_x
from tokenfactory_amd import add_rms_norm

pytestmark = pytest.mark.gpu
EPS = 1e-6
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def weights(cols, seed, dtype=torch.float32):
    return (1.0 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(seed))).to(dtype)


def make_gate(kind, rows, cols, dtype=torch.bfloat16):
    if kind is None:
        return None
    shape = {"row": (rows, 1), "col": (cols,), "full": (rows, cols), "one": (1, 1),
             "row0": (1, cols)}[kind]
    return torch.rand(shape, generator=torch.Generator().manual_seed(9)).to(dtype)


def check(gpu, x, residual, weight, post=None, gate=None, scale=1.0, quantize=False, **kw):
    put = lambda t: None if t is None else t.to(gpu)
    y, r = add_rms_norm(put(x), put(residual), put(weight), EPS, post_weight=put(post),
                        gate=put(gate), residual_scale=scale, quantize=quantize, **kw)
    compare(y, r, x, residual, weight, post, gate, scale, quantize)
    return y, r


def compare(y, r, x, residual, weight, post, gate, scale, quantize):
    ry, rr, size = ob.add_rms_norm(x, residual, weight, EPS, post, gate, scale)
    rt = (x if residual is None else residual).dtype
    assert r.dtype == rt and r.shape == x.shape
    err = (r.double().cpu() - rr).abs()
    assert bool((err <= ROUND[rt] * rr.abs() + 2.0 ** -20 * size).all()), err.max()
    if weight is None:
        assert y is None
        return
    # r's own error reaches y through 1 / rms(r)
    carry = 2.0 ** -20 * size / torch.sqrt((rr * rr).mean(dim=1, keepdim=True) + EPS) \
        * weight.double().abs()
    slack = 2.0 ** -18 * ry.abs() + carry
    if not quantize:
        assert y.dtype == x.dtype and y.shape == x.shape
        err = (y.double().cpu() - ry).abs()
        assert bool((err <= ROUND[x.dtype] * ry.abs() + slack).all()), err.max()
        return
    q, s = (t.cpu() for t in y)
    sb = ob.blocks(slack).amax(dim=2)
    ws = ob.blocks(ry).abs().amax(dim=2).clamp(min=1e-12) / 448
    assert s.shape == ws.shape and bool(((s.double() - ws).abs() <= sb / 448 + 2.0 ** -23 * ws).all())
    full = s.double().repeat_interleave(128, dim=1)[:, : x.shape[1]]
    err = (ob.dequantize(q, s) - ry).abs()
    bound = torch.maximum(2.0 ** -4 * (ry.abs() + slack), 2.0 ** -10 * full) + slack \
        + 2.0 ** -22 * ry.abs()
    assert bool((err <= bound).all()), (err - bound).max()


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 5120), (3, 136), (7, 1000), (48, 5120),
                                       (50, 2560), (2, 8200), (5, 16384), (600, 256)])
def test_residual_sum_and_norm(gpu, rows, cols, quantize):
    print(f"[norm] {rows} x {cols} quantize={quantize}", flush=True)
    x = make_x(rows, cols, rows + cols)
    check(gpu, x, make_x(rows, cols, 1) * 3, weights(cols, 2), quantize=quantize)


@pytest.mark.parametrize("residual,post,gate,scale", itertools.product(
    [None, torch.bfloat16, torch.float32], [False, True], [None, "row", "col", "full", "one", "row0"],
    [1.0, 0.25]))
def test_every_form(gpu, residual, post, gate, scale):
    rows, cols = 13, 648
    print(f"[norm] residual={residual} post={post} gate={gate} scale={scale}", flush=True)
    x = make_x(rows, cols, 3)
    r = None if residual is None else (make_x(rows, cols, 4, torch.float32) * 3).to(residual)
    p = weights(cols, 5, torch.bfloat16) if post else None
    g = make_gate(gate, rows, cols)
    for quantize in (False, True):
        check(gpu, x, r, weights(cols, 6), p, g, scale, quantize)
    check(gpu, x, r, None, p, g, scale)


@pytest.mark.parametrize("xt,gt,wt", itertools.product([torch.bfloat16, torch.float32], repeat=3))
def test_types(gpu, xt, gt, wt):
    x = make_x(6, 264, 7, torch.float32).to(xt)
    check(gpu, x, make_x(6, 264, 8, torch.float32), weights(264, 9, wt), weights(264, 1, wt),
          make_gate("full", 6, 264, gt), 0.5)
    check(gpu, x, None, weights(264, 9, wt), None, make_gate("row", 6, 264, gt), 2.0, True)


def test_plain_norm_returns_x_as_residual(gpu):
    x = make_x(5, 512, 2).to(gpu)
    y, r = add_rms_norm(x, None, weights(512, 1).to(gpu), EPS)
    assert r is x
    compare(y, r, x.cpu(), None, weights(512, 1), None, None, 1.0, False)
    y, r = add_rms_norm(x, None, None, EPS)
    assert y is None and r is x


def test_in_place_and_empty(gpu):
    x, res = make_x(9, 640, 2), make_x(9, 640, 3)
    w = weights(640, 4)
    want_y, want_r = add_rms_norm(x.to(gpu), res.to(gpu), w.to(gpu), EPS)
    buf = torch.full((9, 800), 7.0, dtype=torch.bfloat16, device=gpu)
    view = buf[:, 80:720]
    view.copy_(res)
    y, r = add_rms_norm(x.to(gpu), view, w.to(gpu), EPS, inplace=True)
    assert r is view and torch.equal(view, want_r) and torch.equal(y, want_y)
    assert bool((buf[:, :80] == 7).all()) and bool((buf[:, 720:] == 7).all())
    same = x.to(gpu)
    y, r = add_rms_norm(same, same, w.to(gpu), EPS, inplace=True)   # x + x over x
    compare(y, r, x, x, w, None, None, 1.0, False)
    for bad in (None, buf[:, 3:643], x[:1].to(gpu).expand(9, 640)):
        with pytest.raises(ValueError):
            add_rms_norm(x.to(gpu), bad, w.to(gpu), EPS, inplace=True)
    (q, s), r = add_rms_norm(same[:0], same[:0], w.to(gpu), EPS, quantize=True)
    assert q.shape == (0, 640) and s.shape == (0, 5) and r.shape == (0, 640)


def test_strides(gpu):
    x, res, w = make_x(6, 256, 2), make_x(6, 256, 3), weights(256, 4)
    g = make_gate("full", 6, 256)
    want = add_rms_norm(x.to(gpu), res.to(gpu), w.to(gpu), EPS, gate=g.to(gpu))
    wide = torch.zeros((3, 6, 300), dtype=torch.bfloat16, device=gpu)
    for off in (0, 8, 5):
        views = [wide[i, :, off:off + 256] for i in range(3)]
        for v, t in zip(views, (x, res, g)):
            v.copy_(t)
        got = add_rms_norm(views[0], views[1], w.to(gpu), EPS, gate=views[2])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ww = torch.zeros(512, device=gpu)
    ww[::2] = w.to(gpu)
    got = add_rms_norm(x.t().contiguous().to(gpu).t(), res.to(gpu), ww[::2], EPS, gate=g.to(gpu))
    assert torch.equal(got[0], want[0])


def test_odd_values_stay_with_their_rows(gpu):
    x, res, w = make_x(8, 384, 2).to(gpu), make_x(8, 384, 3).to(gpu), weights(384, 4).to(gpu)
    (wq, wsc), wr = add_rms_norm(x, res, w, EPS, quantize=True)
    y = x.clone()
    y[2, 5], y[6, 300] = float("nan"), float("inf")
    (q, s), r = add_rms_norm(y, res, w, EPS, quantize=True)
    keep = [0, 1, 3, 4, 5, 7]
    assert torch.equal(q[keep].view(torch.uint8), wq[keep].view(torch.uint8))
    assert torch.equal(s[keep], wsc[keep]) and torch.equal(r[keep], wr[keep])
    assert bool(torch.isnan(s[2]).all())
    zeros, _ = add_rms_norm(torch.zeros_like(x), None, w, EPS)
    assert not zeros.any()


def test_refusals(gpu):
    x, w = make_x(4, 256, 1).to(gpu), weights(256, 2).to(gpu)
    with pytest.raises(ValueError):
        add_rms_norm(x, x[:3], w)
    with pytest.raises(ValueError):
        add_rms_norm(x, None, w[:128])
    with pytest.raises(ValueError):
        add_rms_norm(x, None, None, quantize=True)
    with pytest.raises(ValueError):
        add_rms_norm(x.half(), None, w)
    with pytest.raises(ValueError):
        add_rms_norm(x[:, :252], None, w[:252])
    with pytest.raises(NotImplementedError):
        add_rms_norm(torch.zeros((1, 16392), device=gpu), None, torch.ones(16392, device=gpu))
    with pytest.raises(RuntimeError):
        add_rms_norm(x, None, w, gate=torch.ones((3, 1), device=gpu))


def test_in_place_refuses_operands_that_it_would_overwrite(gpu):
    x, w = make_x(4, 256, 1).to(gpu), weights(256, 2, torch.bfloat16).to(gpu)
    buf = make_x(6, 512, 3).to(gpu)
    r = buf[:4, :256]
    for kw in (dict(x=buf[1:5, :256]), dict(gate=buf[0, :256]), dict(gate=r[:, :1]),
               dict(post_weight=buf[1, :256]), dict(weight=buf[2, :256])):
        a = dict(x=x, weight=w)
        a.update(kw)
        keep = buf.clone()
        with pytest.raises(ValueError):
            add_rms_norm(a.pop("x"), r, a.pop("weight"), EPS, inplace=True, **a)
        assert torch.equal(buf, keep)
    gate = buf[:4, 256:]                     # other columns of the same rows
    want = add_rms_norm(x, r, w, EPS, gate=gate)
    got = add_rms_norm(x, r, w, EPS, gate=gate, inplace=True)
    assert torch.equal(got[0], want[0]) and torch.equal(r, want[1])


def test_weights_that_lie_unaligned(gpu):
    x = make_x(5, 264, 1).to(gpu)
    flat = weights(600, 2).to(gpu)
    for off in (1, 3, 265):
        w, p = flat[off:off + 264], flat[off + 2:off + 266]
        want = add_rms_norm(x, x, w.clone(), EPS, post_weight=p.clone())
        got = add_rms_norm(x, x, w, EPS, post_weight=p)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
