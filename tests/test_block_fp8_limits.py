"""Sizes that the block-scaled products refuse (CPU only: nothing is launched)."""
import ctypes

from tokenfactory_amd import _native

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
