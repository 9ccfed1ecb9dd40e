"""CPU: what the 4-bit calls refuse at their limits, before any GPU work, and that the size of a workspace is refused with the call."""
import pytest

from tests.test_mx4 import LINEAR


@pytest.mark.parametrize("x_dtype, rows, n, k, code", [
    (0, 4, 0, 64, -1), (0, 4, (1 << 22) + 1, 64, -3), (0, 4, 16, (1 << 22) + 1, -3), (0, 4, 16, 0, -1), (0, -1, 16, 64, -1), (4, 4, 16, 64, -1),
    (7, 4, 16, 64, -1), (0, 1 << 36, 128, 32, -3), (0, 1 << 32, 1 << 22, 32, -3), (5, 1 << 36, 128, 32, -3), (0, 1 << 41, 128, 32, -3),
    (0, 1 << 22, 1 << 22, 32, -3)])
def test_linear_and_its_workspace_refuse_the_same(x_dtype, rows, n, k, code):
    from yololite_amd import _lib

    L = _lib.lib()
    change = dict(x_dtype=x_dtype, x_scales=1 << 20, rows=rows, n=n, k=k, x_stride=k, y_stride=n, work_bytes=1 << 62)
    assert L.yl_mx4_linear(*(LINEAR | change).values()) == code and b"mx4_linear" in L.yl_last_error()
    assert L.yl_mx4_linear_workspace_bytes(x_dtype, rows, n, k) == -1


@pytest.mark.parametrize("x_dtype", [0, 1, 5])
@pytest.mark.parametrize("rows, n, k", [(5_000_000, 64, 64), (65, 1 << 22, 32), (1, 1 << 22, 1 << 22), (1 << 28, 64, 64)])
def test_sizes_that_have_a_workspace(x_dtype, rows, n, k):
    """Many rows, many columns: 65536 groups of 64 and more on either side are no limit."""
    from yololite_amd import _lib

    assert _lib.lib().yl_mx4_linear_workspace_bytes(x_dtype, rows, n, k) >= 0


@pytest.mark.parametrize("rows, cols", [(1 << 30, 1), (1 << 30, 32), ((1 << 29) + 1, 64), (1 << 14, 1 << 22), (1 << 34, 32)])
def test_quantize_takes_fewer_than_2_to_the_30_blocks(rows, cols):
    """Four threads to a block: a launch of 2^32 would be cut off."""
    from yololite_amd import _lib

    L = _lib.lib()
    at = 1 << 20
    assert L.yl_mx4_quantize(at, 0, rows, cols, cols, at, at, None) == -3 and b"mx4_quantize" in L.yl_last_error()
    assert L.yl_mx4_dequantize(at, at, rows, cols, at, 0, cols, None) == -3 and b"mx4_dequantize" in L.yl_last_error()
