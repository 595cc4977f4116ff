"""8-bit operators: sizes that no launch takes (2^32 threads and more) are refused as sizes, by the native checks, before anything is launched.  No GPU is needed."""
import ctypes as C

import pytest

FAR = 1 << 32


# a wavefront per 512 columns, four to a workgroup: 2^26 rows of up to 512 columns; with 2^30 columns 32 rows
@pytest.mark.parametrize("n,W", [(1 << 26, 1), ((1 << 31) - 1, 128), (1 << 25, 513), (1 << 5, 1 << 30), ((1 << 31) + 4, 8)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_rows(n, W, dtype):
    from jacobiforcing_amd import _native as N
    L = N.layers()
    for scale in (0, 1):
        assert L.jl_quantize_fp8(4096, dtype, n, FAR, W, 4096, FAR, 4096, FAR, scale, None) == -1
        assert L.jl_gated_act_fp8(4096, dtype, n, FAR, 0, -1, W, 2, 0.0, 1.0, 0.0, 4096, FAR, 4096, FAR, scale, None) == -1


# four rows to 256 threads up to 1024 columns, then 256 threads for a row, beyond 8192 columns 1024
@pytest.mark.parametrize("n,W", [(1 << 26, 1), (1 << 26, 1024), (1 << 24, 1025), (1 << 24, 8192), (1 << 22, 8193), (1 << 22, 33000), ((1 << 31) + 4, 8)])
def test_norms(n, W):
    from jacobiforcing_amd import _native as N
    L = N.layers()
    for dtype in (0, 1):
        for scale in (0, 1):
            assert L.jl_add_rmsnorm_fp8(4096, dtype, FAR, None, 0, 0, None, 0, 1e-6, n, W, 4096, FAR, 4096, FAR, scale, None) == -1


# 512 threads for 16 rows of w (few rows of x); tiles of 128 x 128; rows of scales at no whole word, which go straight from memory
@pytest.mark.parametrize("change", [dict(N=1, O=1 << 27), dict(N=1, O=1 << 30), dict(N=1 << 21, O=1 << 18), dict(N=1 << 21, O=1 << 18, scale_type=1), dict(N=16, O=1 << 29, x_scale=4097)], ids=str)
def test_products(change):
    from jacobiforcing_amd import _native as N
    p = N.Fp8Product(**{**dict(x=4096, x_scale=4096, w=4096, w_scale=4096, N=4, x_ld=256, x_scale_ld=1 << 21, w_ld=256, w_scale_ld=2, K=256, O=256, scale_type=0), **change})
    assert N.layers().jl_linear_fp8(C.byref(p), None, 0, 4096, 1 << 30, 0, 4096, None) == -1


@pytest.mark.parametrize("change", [dict(N=16, O=1 << 30, x_scale=4097), dict(N=1 << 21, O=1 << 20, scale_type=1)], ids=str)
def test_gated_products(change):
    from jacobiforcing_amd import _native as N
    p = N.Fp8Product(**{**dict(x=4096, x_scale=4096, w=4096, w_scale=4096, N=4, x_ld=256, x_scale_ld=1 << 21, w_ld=256, w_scale_ld=2, K=256, O=256, scale_type=0), **change})
    assert N.layers().jl_linear_gated_fp8(C.byref(p), 2, 0.0, 1.0, 0.0, 4096, 1 << 30, 4096, 1 << 22, None) == -1
