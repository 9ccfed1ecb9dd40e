"""GPU: 4-bit products of more than 65535 groups of 64 rows and columns.  Tolerances as in test_gpu_mx4.py."""
import pytest
import torch

from tests import mx4_ref
from tests.test_gpu_mx4 import _check_product, _np, _ya

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("rows, n, k", [(4_400_000, 16, 32), (2_400_000, 130, 100), (80, 1 << 22, 32), (4_194_240, 64, 64), (4_194_241, 64, 64)])
def test_many_rows_and_columns(gpu_device, rows, n, k, packed):
    """Against the definition for some rows (or columns), the first and last and those around the 32768th group of 64."""
    ya = _ya()
    g = torch.Generator(device=gpu_device).manual_seed(rows % 1000 + n)
    x = torch.randn(rows, k, generator=g, device=gpu_device).bfloat16()
    w = torch.randn(n, k, generator=g, device=gpu_device)
    b = torch.randn(n, generator=g, device=gpu_device)
    y = ya.mx4_linear(ya.mx4_quantize(x) if packed else x, ya.mx4_quantize(w), bias=b, act=True)
    some = lambda m: torch.tensor(sorted({i for i in (0, 1, 64 * 32768 - 1, 64 * 32768, 64 * 32768 + 63, m // 2, m - 130, m - 1) if 0 <= i < m}),
                                  device=gpu_device)
    r = some(rows) if rows > n else torch.arange(rows, device=gpu_device)
    c = some(n) if n > rows else torch.arange(n, device=gpu_device)
    _check_product(y[r][:, c], mx4_ref.rounded(_np(x[r])), mx4_ref.rounded(_np(w[c])), b[c], True, None)
    assert bool(torch.isfinite(y).all())


def test_more_than_2_to_the_31_groups_of_eight_columns(gpu_device):
    """One column of values that 4 bits hold: what comes back is what went in."""
    ya = _ya()
    rows = (1 << 29) + 70_001
    g = torch.Generator(device=gpu_device).manual_seed(3)
    part = torch.randint(2, 4, (1_000_003, 1), generator=g, device=gpu_device) * 2.0 ** torch.randint(-20, 20, (1_000_003, 1), generator=g, device=gpu_device)
    part = (part * (torch.randint(0, 2, (1_000_003, 1), generator=g, device=gpu_device) * 2 - 1)).bfloat16()
    x = part.repeat(rows // 1_000_003 + 1, 1)[:rows]
    t = ya.mx4_quantize(x)
    assert t.codes.shape == (rows, 16)
    assert torch.equal(ya.mx4_dequantize(t), x)
