"""Calls that the block-scaled products and ``add_rms_norm`` refuse, and neighbours that
they take (CPU only: nothing is launched)."""
import ctypes

import torch

from tokenfactory_amd import _native
from tokenfactory_amd.add_norm import _clash

FP8 = _native.TF_DTYPE_FP8_E4M3
M, K = 1 << 24, 4112        # 2^24 rows of 264 16-byte pieces: 2^32.04 threads


def mat(n, k):
    return _native.Fp8Mat(w=16, w_row_stride=k, w_scale=16, w_scale_row_stride=-(-k // 128),
                          w_scale_col_stride=1, bias=None, n=n, out=16, out_row_stride=n)


def test_more_padded_rows_than_a_launch_holds_are_refused():
    lib = _native.load()
    rc = lib.tf_block_linear(16, FP8, K, 16, M, ctypes.byref(mat(16, K)), M, K, 256, 1 << 50, None)
    assert rc == _native.TF_ERR_UNSUPPORTED and b"too large" in lib.tf_attn_last_error()
    mats = (_native.Fp8Mat * 3)(mat(16, K), mat(16, K), mat(16, 16))
    rc = lib.tf_gated_mlp(16, FP8, K, 16, M, mats, M, K, 16, 256, 1 << 50, None)
    assert rc == _native.TF_ERR_UNSUPPORTED and b"too large" in lib.tf_attn_last_error()


def test_one_row_in_place_goes_by_its_elements():
    """The stride of a single row says nothing: a decode step's row may be the residual
    under another view, and a row of stride 0 is compared like any other."""
    r = torch.zeros((8, 512))[:1, :256]
    same = r[0].view(1, 256)
    assert same.stride() != r.stride() and same.data_ptr() == r.data_ptr()
    assert not _clash(r, same)
    flat = torch.zeros(1024)
    row = lambda at, stride: torch.as_strided(flat, (1, 256), (stride, 1), at)
    for a in (0, 1, 256, 512):
        for b in (0, 1, 256, 512):
            assert not _clash(row(64, a), row(64, b))
            assert not _clash(row(64, a), row(320, b)) and not _clash(row(320, a), row(64, b))
            assert _clash(row(64, a), row(72, b)) and _clash(row(72, a), row(64, b))
    assert _clash(row(64, 256), torch.as_strided(flat, (1, 256), (512, 2), 64))
