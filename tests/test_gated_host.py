"""Host side of the gated and MXFP4 entry points: sizes, workspaces and refusals, without a device."""
import ctypes as C

import pytest

from tenzor_b200 import _lib


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def workspace(fn, *args):
    need = C.c_size_t(12345)
    return fn(*args, C.byref(need)), need.value


@pytest.mark.parametrize("rows,cols,want", [(0, 64, 0), (1, 32, 512), (128, 128, 512), (129, 128, 1024), (128, 160, 1024),
                                            (300, 4096, 3 * 32 * 512), (-1, 64, 0), (5, 0, 0), (1 << 22, 8192, (1 << 15) * 64 * 512)])
def test_scale_bytes(L, rows, cols, want):
    assert L.tz_mxfp4_scale_bytes(rows, cols) == want


def test_linear_workspace(L):
    f = L.tz_linear_mxfp4_workspace
    assert workspace(f, 1, 4096, 4096) == (_lib.TZ_OK, 0)  # x is quantised inside the kernel
    assert workspace(f, 16, 8192, 64) == (_lib.TZ_OK, 0)
    for m, k in ((17, 4096), (16, 8224), (1000, 384), (1 << 20, 8192)):
        codes = (m * k // 2 + 255) // 256 * 256
        scales = ((m + 127) // 128 * ((k + 127) // 128) * 512 + 255) // 256 * 256
        assert workspace(f, m, k, 64) == (_lib.TZ_OK, codes + scales)
    assert workspace(f, 0, 64, 64) == (_lib.TZ_OK, 0)
    for bad in ((-1, 64, 64), (4, 0, 64), (4, 48, 64), (4, 64, -8), (4, 1 << 25, 64), ((1 << 30) + 1, 64, 64)):
        assert workspace(f, *bad)[0] == _lib.TZ_EINVAL, bad
    assert f(4, 64, 64, None) == _lib.TZ_EINVAL


def test_python_layout_matches_the_library(L):
    from tenzor_b200 import ops
    for rows, cols in ((17, 32), (100, 4096), (129, 160), (70000, 384)):
        off, size = ops._mx_layout(rows, cols)
        assert off % 256 == 0 and off >= rows * cols // 2
        assert size - off == L.tz_mxfp4_scale_bytes(rows, cols)
        assert workspace(L.tz_linear_mxfp4_workspace, rows, cols, 8)[1] == (size + 255) // 256 * 256


@pytest.mark.parametrize("t,d,f", [(0, 64, 72), (1, 8, 8), (77, 384, 1000), (18106, 384, 1536), (8192, 4096, 8192), (1 << 20, 64, 64)])
@pytest.mark.parametrize("sms", [1, 2, 148])
def test_backward_workspace(L, sms, t, d, f):
    rc, need = workspace(L.tz_gated_linear_backward_workspace, sms, t, d, f)
    assert rc == _lib.TZ_OK and need >= 2 * t * f * 2
    # dg and du, and at most 16 partial sums of whole row tiles
    rows = (t + 255) // 256 * 256 + 2 * ((f + 255) // 256 * 256)
    assert need <= 2 * (t * f * 2 + 256) + 16 * rows * d * 4 + 512


def test_backward_workspace_refusals(L):
    f = L.tz_gated_linear_backward_workspace
    for bad in ((0, 4, 64, 64), (148, -1, 64, 64), (148, 4, 60, 64), (148, 4, 64, 12), (148, 4, 0, 64), (148, 4, 64, 1 << 25)):
        assert workspace(f, *bad)[0] == _lib.TZ_EINVAL, bad
    assert f(148, 4, 64, 64, None) == _lib.TZ_EINVAL


def test_null_contexts_are_refused(L):
    E = _lib.TZ_EINVAL
    assert L.tz_gated_linear(None, None, 64, None, None, None, 4, 64, 64, 9, 1, None) == E
    assert L.tz_gated_linear_backward(None, None, 64, None, None, None, 64, None, None, None, None, 0, 4, 64, 64, 9, 1, None) == E
    assert L.tz_quantize_mxfp4(None, None, 64, 0, None, None, 4, 64, None) == E
    assert L.tz_dequantize_mxfp4(None, None, None, None, 0, 4, 64, None) == E
    assert L.tz_pack_gated_mxfp4(None, None, None, 0, None, None, 16, 64, None) == E
    assert L.tz_gemm_mxfp4(None, None, None, None, None, None, None, 0, 4, 64, 64, None) == E
    assert L.tz_linear_mxfp4(None, None, 64, 0, None, None, None, None, 0, None, 0, 4, 64, 64, None) == E
    assert L.tz_gated_linear_mxfp4(None, None, 64, 1, None, None, None, 9, None, 0, 4, 64, 64, None) == E
    assert "null" in L.tz_get_last_error().decode()
