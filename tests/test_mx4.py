"""CPU: the MX4 restatement against hand-derived values; refusals of the MX4 entry points (argument checks come before any GPU work)."""
import ctypes

import numpy as np
import pytest
import torch

from tests import mx4_ref


def test_restatement_on_hand_derived_blocks():
    x = np.zeros((1, 40))
    # largest magnitude 5 = 2^2 * 1.25: scale 2^0; ties 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5 go to the even code
    x[0, :10] = [5.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -5.0, -0.26, 0.0]
    x[0, 32:36] = [7.9, 1.0, -6.1, 0.3]  # saturates at 6
    code, byte = mx4_ref.quantize(x)
    assert byte.tolist() == [[127, 127]]
    assert code[0, 0, :10].tolist() == [6, 0, 2, 2, 4, 4, 6, 14, 9, 0]
    assert code[0, 1, :4].tolist() == [7, 2, 15, 1]
    assert mx4_ref.rounded(x)[0, [0, 2, 7, 32, 34]].tolist() == [4.0, 1.0, -4.0, 6.0, -6.0]
    assert mx4_ref.unpack(mx4_ref.pack(code)).tolist() == code.tolist()


def test_restatement_at_the_ends_of_the_range():
    x = np.array([[2.0 ** -149] + [0.0] * 31, [2.0 ** -124] + [2.0 ** -128] * 31, [np.inf] + [1.0] * 31, [3.0e38] + [1.0] * 31])
    code, byte = mx4_ref.quantize(x)
    assert byte[:, 0].tolist() == [0, 1, 255, 252]
    r = mx4_ref.rounded(x)
    assert r[0, 0] == 0.0 and r[1, 0] == 2.0 ** -124 and r[1, 1] == 0.0  # 2^-128 is a quarter of 2^-126: the tie goes to 0
    assert np.isnan(r[2]).all() and r[3, 0] == 3 * 2.0 ** 126


def _ptr(n):
    """An aligned host address: the calls below are refused before anything is read."""
    return (n << 12) + 4096


@pytest.mark.parametrize("change, code", [
    (dict(x_dtype=3), -1), (dict(x=None), -1), (dict(codes=None), -1), (dict(codes=_ptr(3) + 8), -1), (dict(cols=0), -1),
    (dict(rows=-1), -1), (dict(stride=63), -1), (dict(cols=(1 << 22) + 1, stride=1 << 23), -3), (dict(rows=1 << 41), -3)])
def test_quantize_refusals(change, code):
    from yololite_amd import _lib

    a = dict(x=_ptr(1), x_dtype=0, rows=4, cols=64, stride=64, codes=_ptr(3), scales=_ptr(4), stream=None) | change
    L = _lib.lib()
    assert L.yl_mx4_quantize(*a.values()) == code and b"mx4_quantize" in L.yl_last_error()
    a = dict(codes=a["codes"], scales=a["scales"], rows=a["rows"], cols=a["cols"], y=a["x"], y_dtype=a["x_dtype"], stride=a["stride"],
             stream=None)
    assert L.yl_mx4_dequantize(*a.values()) == code and b"mx4_dequantize" in L.yl_last_error()


LINEAR = dict(x=_ptr(1), x_scales=None, x_dtype=0, rows=40, x_stride=64, w_codes=_ptr(2), w_scales=_ptr(3), n=16, k=64, bias=None, act=0,
              res=None, res_stride=0, y=_ptr(5), y_dtype=0, y_stride=16, work=_ptr(6), work_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change, code", [
    (dict(x_dtype=4), -1), (dict(x_dtype=5), -1), (dict(y_dtype=5), -1), (dict(x=None), -1), (dict(w_codes=None), -1), (dict(y=None), -1),
    (dict(w_scales=None), -1), (dict(w_codes=_ptr(2) + 4), -1), (dict(work=None), -1), (dict(work_bytes=8), -1), (dict(work=_ptr(6) + 8), -1),
    (dict(n=0), -1), (dict(k=0), -1), (dict(rows=-3), -1), (dict(x_stride=32), -1), (dict(y_stride=8), -1),
    (dict(res=_ptr(7), res_stride=8), -1), (dict(n=1 << 23), -3), (dict(k=1 << 23, x_stride=1 << 23), -3)])
def test_linear_refusals(change, code):
    from yololite_amd import _lib

    L = _lib.lib()
    assert L.yl_mx4_linear(*(LINEAR | change).values()) == code and b"mx4_linear" in L.yl_last_error()


def test_nothing_to_do_is_no_error():
    from yololite_amd import _lib

    L = _lib.lib()
    assert L.yl_mx4_linear(*(LINEAR | dict(rows=0, x=None, y=None, work=None, work_bytes=0)).values()) == 0
    assert L.yl_mx4_quantize(None, 0, 0, 64, 64, None, None, None) == 0
    assert L.yl_mx4_linear_workspace_bytes(0, 0, 16, 64) == 0 and L.yl_mx4_linear_workspace_bytes(5, 9, 16, 64) == 0
    assert L.yl_mx4_linear_workspace_bytes(0, 100, 16, 64) >= 100 * 34 and L.yl_mx4_linear_workspace_bytes(0, -1, 16, 64) == -1


def test_python_face_refuses_without_a_gpu_tensor():
    import yololite_amd as ya

    assert ctypes.sizeof(ctypes.c_void_p) == 8
    with pytest.raises(RuntimeError, match="GPU only"):
        ya.mx4_quantize(torch.zeros(2, 32))
    w = ya.Mx4Tensor(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 32)
    with pytest.raises(RuntimeError, match="GPU only"):
        ya.mx4_linear(torch.zeros(2, 32), w)
