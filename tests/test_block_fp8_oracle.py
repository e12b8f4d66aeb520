"""The block-scaled FP8 oracle against closed forms, and the refusals of the operators'
entry points (CPU only: nothing is launched)."""
import ctypes
import types

import pytest
import torch

from oracle import block_fp8 as ob
from tokenfactory_amd import (GatedMLP, _native, add_rms_norm, block_scaled_linear, gated_mlp,
                              quantize_blocks)
from tokenfactory_amd.add_norm import _clash

INVALID, UNSUPPORTED = _native.TF_ERR_INVALID, _native.TF_ERR_UNSUPPORTED
BF16, FP8, FP32 = _native.TF_DTYPE_BF16, _native.TF_DTYPE_FP8_E4M3, _native.TF_DTYPE_FP32


def test_round_e4m3_is_the_nearest_value():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every)].unique()
    assert torch.equal(ob.round_e4m3(every), every)
    mid = (every[1:] + every[:-1]) / 2
    for v, sign in ((mid + 1e-9, 1), (mid - 1e-9, -1)):
        want = every[1:] if sign > 0 else every[:-1]
        assert torch.equal(ob.round_e4m3(v), want)
    even = ob.round_e4m3(mid)            # ties: the neighbour with an even mantissa
    bits = even.to(torch.float8_e4m3fn).view(torch.uint8)
    assert bool((bits % 2 == 0).all())


def test_quantize_closed_forms():
    x = torch.zeros((3, 200))
    x[0, 5], x[0, 7] = 448.0, -17.0      # scale 1: 17 is a tie between 16 and 18
    x[0, 130] = 3.0
    x[1] = 1e-20
    q, s = ob.quantize(x)
    assert s.shape == (3, 2) and float(s[0, 0]) == 1.0 and float(s[0, 1]) == float(
        torch.tensor(3.0) / 448)
    assert float(q[0, 5]) == 448.0 and float(q[0, 7]) == -16.0 and float(q[0, 130]) == 448.0
    assert bool((s[2] == torch.tensor(1e-12) / 448).all()) and not q[2].float().any()
    back = ob.dequantize(q, s)
    assert float(back[0, 130]) == pytest.approx(3.0, rel=2 ** -24)


def test_gated_hidden_bounds_hold_the_neighbouring_roundings():
    g = torch.Generator().manual_seed(3)
    x = torch.randn((5, 64), generator=g, dtype=torch.float64)
    wg, wu = (torch.randn((200, 64), generator=g, dtype=torch.float64) for _ in range(2))
    h, off = ob.gated_hidden(x, wg, wu)
    assert h.shape == off.shape == (5, 200) and bool((off >= 0).all())
    moved, _ = ob.gated_hidden(x, wg * (1 + 2.0 ** -18), wu * (1 - 2.0 ** -18))
    assert bool(((moved - h).abs() <= off + 1e-12).all())


@pytest.mark.parametrize("rows,cols,dtype,xs,qs,ss,code", [
    (4, 130, BF16, 136, 136, 4, INVALID),       # cols not a multiple of 8
    (4, 0, BF16, 8, 8, 4, INVALID),
    (-1, 128, BF16, 128, 128, 4, INVALID),
    (4, 128, FP8, 128, 128, 4, UNSUPPORTED),
    (4, 128, BF16, 120, 128, 4, INVALID),       # rows overlap
    (4, 128, BF16, 132, 128, 4, INVALID),       # rows misaligned
    (4, 128, BF16, 128, 128, 3, INVALID),       # scales overlap
    (4, 1 << 25, BF16, 1 << 25, 1 << 25, 4, UNSUPPORTED),
])
def test_quant_refusals(rows, cols, dtype, xs, qs, ss, code):
    lib = _native.load()
    assert lib.tf_block_quant(16, dtype, rows, cols, xs, 16, qs, 16, ss, None) == code
    assert lib.tf_attn_last_error()


def test_quant_null_and_empty():
    lib = _native.load()
    assert lib.tf_block_quant(None, BF16, 4, 128, 128, 16, 128, 16, 4, None) == INVALID
    assert lib.tf_block_quant(8, BF16, 4, 128, 128, 16, 128, 16, 4, None) == INVALID
    assert lib.tf_block_quant(None, BF16, 0, 128, 128, None, 128, None, 0, None) == 0


def _mat(n, k, **kw):
    f = dict(w=16, w_row_stride=k, w_scale=16, w_scale_row_stride=-(-k // 128),
             w_scale_col_stride=1, bias=None, n=n, out=16, out_row_stride=n)
    f.update(kw)
    return _native.Fp8Mat(**f)


def _linear(m=4, k=256, n=64, x=16, x_dtype=BF16, xs=256, sc=None, ss=0, ws=256, ws_bytes=1 << 30,
            **kw):
    lib = _native.load()
    mat = _mat(n, k, **kw)
    return lib.tf_block_linear(x, x_dtype, xs, sc, ss, ctypes.byref(mat), m, k, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(k=250), INVALID),                      # not a multiple of 16
    (dict(n=0), INVALID),
    (dict(m=-1), INVALID),
    (dict(x=None), INVALID),
    (dict(x=24), INVALID),                       # misaligned
    (dict(xs=128), INVALID),
    (dict(x_dtype=5), UNSUPPORTED),
    (dict(w=None), INVALID),
    (dict(w_scale=None), INVALID),
    (dict(w=8), INVALID),
    (dict(w_row_stride=264), INVALID),
    (dict(w_scale_col_stride=-1), INVALID),
    (dict(out=None), INVALID),
    (dict(out_row_stride=63), INVALID),
    (dict(ws=None), INVALID),
    (dict(ws=260), INVALID),
    (dict(ws_bytes=100), INVALID),
    (dict(x_dtype=FP8, sc=None, ss=4), INVALID),  # quantised without scales
    (dict(x_dtype=FP8, sc=16, ss=3), INVALID),
    (dict(x_dtype=FP8, sc=16, ss=4, k=208, xs=192), INVALID),   # rows overlap
    (dict(m=1 << 23, n=1 << 23), UNSUPPORTED),
])
def test_linear_refusals(kw, code):
    assert _linear(**kw) == code
    assert _native.load().tf_attn_last_error()


def test_empty_products_touch_nothing():
    assert _linear(m=0, x=None, ws=None, ws_bytes=0) == 0
    lib = _native.load()
    assert lib.tf_block_linear_workspace_bytes(0, 64, 256, BF16) == 0
    assert lib.tf_gated_mlp_workspace_bytes(0, 256, 512, 256, BF16) == 0
    mats = (_native.Fp8Mat * 3)(*[_mat(n, k) for n, k in ((512, 256), (512, 256), (256, 512))])
    assert lib.tf_gated_mlp(None, BF16, 256, None, 0, mats, 0, 256, 512, None, 0, None) == 0


@pytest.mark.parametrize("change,code", [
    (dict(hidden=250), INVALID), (dict(inter=500), INVALID),
    (dict(up=(496, 256)), INVALID), (dict(ws_bytes=64), INVALID), (dict(mats=None), INVALID),
    (dict(down=(0, 512)), INVALID),
    (dict(x_dtype=9), UNSUPPORTED),
])
def test_mlp_refusals(change, code):
    a = dict(hidden=256, inter=512, up=(512, 256), down=(256, 512), ws_bytes=1 << 30, x_dtype=BF16)
    a.update(change)
    mats = (_native.Fp8Mat * 3)(_mat(512, 256), _mat(*a["up"]), _mat(*a["down"]))
    lib = _native.load()
    assert lib.tf_gated_mlp(16, a["x_dtype"], 256, None, 0, a.get("mats", mats), 4, a["hidden"],
                            a["inter"], 256, a["ws_bytes"], None) == code


def test_workspaces_cover_the_quantised_rows():
    lib = _native.load()
    for m, k in ((1, 256), (77, 5120), (8192, 1040)):
        kp, kb = -(-k // 128) * 128, -(-k // 128)
        own = lib.tf_block_linear_workspace_bytes(m, 640, k, BF16)
        given = lib.tf_block_linear_workspace_bytes(m, 640, k, FP8)
        padded = m * kp if k % 128 and m > 16 else 0     # a copy with zeros behind its rows
        assert own >= given + 4 * m * kb + m * kp - padded and given >= padded
        assert lib.tf_gated_mlp_workspace_bytes(m, k, 640, k, FP8) >= m * 640 + 4 * m * 5
    assert lib.tf_block_linear_workspace_bytes(4, 64, 100, BF16) == INVALID
    assert lib.tf_gated_mlp_workspace_bytes(4, 128, 100, 128, BF16) == INVALID


def _norm(**kw):
    a = dict(x=16, x_dtype=BF16, xs=256, r=16, r_dtype=BF16, rs=256, g=None, g_dtype=0, gs=0,
             gcol=0, post=None, post_dtype=0, w=16, w_dtype=FP32, rows=4, cols=256, ro=16, ros=256,
             y=16, y_dtype=BF16, ys=256, sc=None, ss=0)
    a.update(kw)
    return _native.load().tf_add_rms_norm(
        a["x"], a["x_dtype"], a["xs"], a["r"], a["r_dtype"], a["rs"], a["g"], a["g_dtype"], a["gs"],
        a["gcol"], a["post"], a["post_dtype"], a["w"], a["w_dtype"], 1e-6, 1.0, a["rows"],
        a["cols"], a["ro"], a["ros"], a["y"], a["y_dtype"], a["ys"], a["sc"], a["ss"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), INVALID), (dict(y=None, ro=None), INVALID), (dict(w=None), INVALID),
    (dict(cols=252), INVALID), (dict(cols=16392, xs=16392), UNSUPPORTED), (dict(rows=-1), INVALID),
    (dict(xs=128), INVALID), (dict(x=8), INVALID), (dict(x_dtype=FP8), UNSUPPORTED),
    (dict(r_dtype=7), UNSUPPORTED), (dict(rs=0), INVALID), (dict(ros=248), INVALID),
    (dict(y_dtype=7), UNSUPPORTED), (dict(ys=132), INVALID), (dict(y_dtype=FP8), INVALID),
    (dict(y_dtype=FP8, sc=16, ss=3), INVALID), (dict(g=16, g_dtype=FP8), UNSUPPORTED),
    (dict(g=16, g_dtype=BF16, gs=128, gcol=1), INVALID),
    (dict(g=17, g_dtype=BF16, gs=1), INVALID), (dict(post=8, post_dtype=FP32), INVALID),
])
def test_norm_refusals(kw, code):
    assert _norm(**kw) == code
    assert _native.load().tf_attn_last_error()


def test_norm_of_no_rows_touches_nothing():
    assert _norm(rows=0, x=None, y=None, ro=None) == 0


def test_python_refuses_cpu_tensors_and_mismatches():
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    w = torch.zeros((128, 256), dtype=torch.float8_e4m3fn)
    s = torch.ones((1, 2))
    d, ds = torch.zeros((256, 128), dtype=torch.float8_e4m3fn), torch.ones((2, 1))
    with pytest.raises(ValueError):
        quantize_blocks(x)
    with pytest.raises(ValueError):
        block_scaled_linear(x, w, s)
    with pytest.raises(ValueError):
        gated_mlp(x, w, s, w, s, d, ds)
    with pytest.raises(ValueError):
        add_rms_norm(x, None, torch.ones(256))


class _Config:
    hidden_size = 256
    intermediate_size = 512
    quantization_config = {"quant_method": "fp8", "weight_block_size": [128, 128]}


def test_module_holds_the_reference_parameters():
    mlp = GatedMLP(_Config())
    assert {k: tuple(v.shape) for k, v in mlp.state_dict().items()} == {
        "gate_proj.weight": (512, 256), "gate_proj.weight_scale_inv": (4, 2),
        "up_proj.weight": (512, 256), "up_proj.weight_scale_inv": (4, 2),
        "down_proj.weight": (256, 512), "down_proj.weight_scale_inv": (2, 4)}
    share = type("C", (_Config,), {"tp_size": 4})
    assert GatedMLP(share()).down_proj.weight.shape == (256, 128)


@pytest.mark.parametrize("change", [
    dict(quantization_config=None),
    dict(quantization_config={"quant_method": "fp8", "weight_block_size": [64, 128]}),
    dict(hidden_act="gelu"), dict(intermediate_size=520, tp_size=5)])
def test_module_refusals(change):
    with pytest.raises(NotImplementedError):
        GatedMLP(type("C", (_Config,), change)())


def test_more_than_a_launch_holds_is_refused():
    """2^32 threads: a thread per 8 columns (norm, quantisation), 128 per 32 x 64 outputs."""
    lib = _native.load()
    assert _norm(rows=1 << 22, cols=8192, xs=8192, rs=8192, ros=8192, ys=8192) == UNSUPPORTED
    assert lib.tf_block_quant(16, BF16, 1 << 24, 1 << 20, 1 << 20, 16, 1 << 20, 16, 1 << 24,
                              None) == UNSUPPORTED
    assert lib.tf_block_linear_workspace_bytes(1 << 20, 1 << 17, 256, BF16) == UNSUPPORTED
    assert lib.tf_gated_mlp_workspace_bytes(1 << 20, 256, 1 << 17, 256, BF16) == UNSUPPORTED


def test_a_stream_of_another_device_is_refused():
    stream = types.SimpleNamespace(device=torch.device("cuda", 1))
    with pytest.raises(ValueError):
        with _native.launching(torch.device("cuda", 0), stream):
            pass


def test_operands_that_an_in_place_sum_would_overwrite():
    buf = torch.zeros((8, 64), dtype=torch.bfloat16)
    r = buf[1:5, 16:32]
    same = buf[1:5, 16:32]
    other = torch.zeros_like(r)
    assert not any(_clash(r, t) for t in (None, same, other, other[0], other[:, :1]))
    # other columns of the same rows, in either order, and rows before or after
    assert not any(_clash(r, t) for t in (buf[1:5, 32:48], buf[1:5, :16], buf[0:1, 16:32], buf[5]))
    for t in (buf[2:6, 16:32], buf[0:4, 16:32], buf[1:5, 24:40], buf[1:5, 8:24], buf[2, 16:32],
              buf[1:5, 16:17], r.view(torch.uint8)[:, :16], buf[0:8:2, 16:32], buf[1:2, 16:32]):
        assert _clash(r, t)
