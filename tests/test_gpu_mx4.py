"""GPU: MX4 quantisation is exact to the bit; products against 64-bit arithmetic on the same 4-bit values.

Tolerance of a product: the operands are exact, their products too (2 x 2 significant bits and powers of two), so the fp32
accumulation of k terms is off by at most k 2^-24 sum |x w| (each addition by half a step of a partial sum no larger than that), and
the result's rounding adds eps / 2 of it.  SiLU has slope at most 1.1; computed as v / (1 + 2^(-v log2 e)) in fp32 it adds the error of
the exponent, |v| 2^-24 for the product and as much for the constant, and 2^-23 each for the exponential and the reciprocal, 2^-24
for the sum and the product (under 4 2^-23); where the exponential overflows (v < -88) it is 0 instead of less than 2^-120.  The bias
and the residual add one fp32 rounding each of what they are added to."""
import numpy as np
import pytest
import torch

from tests import mx4_ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _ya():
    import yololite_amd as ya

    return ya


def _np(t):
    return t.double().cpu().numpy()


def _check_quantize(x):
    ya = _ya()
    t = ya.mx4_quantize(x)
    cols = x.shape[-1]
    code, byte = mx4_ref.quantize(_np(x).reshape(-1, cols))
    assert t.cols == cols and t.codes.shape == (*x.shape[:-1], -(-cols // 32) * 16) and t.scales.shape == (*x.shape[:-1], -(-cols // 32))
    got_b = t.scales.cpu().numpy().reshape(byte.shape)
    assert np.array_equal(got_b, byte)
    got_c = mx4_ref.unpack(t.codes.cpu().numpy().reshape(code.shape[0], -1))
    some = byte != 255  # the codes of a block that reads as NaN say nothing
    assert np.array_equal(got_c[some], code[some])
    want = mx4_ref.values(code, byte, cols).reshape(x.shape)
    for dt in (torch.bfloat16, torch.float32):
        y = ya.mx4_dequantize(t, dt)
        assert y.dtype == dt and np.array_equal(_np(y), want, equal_nan=True)
    return t


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 31), (3, 32), (5, 33), (17, 64), (2, 1000), (129, 96), (1, 768), (64, 40)])
def test_quantize_sizes(gpu_device, rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 1000 + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    _check_quantize(x.to(TYPES[dtype]).to(gpu_device))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantize_ties_and_saturation(gpu_device, dtype):
    """Every multiple of 1/8 up to 7.875 in a block whose scale is 1, and the same scaled over the type's exponents."""
    base = torch.arange(64, dtype=torch.float64) / 8
    rows = []
    for e in range(-12, 12):
        for lo in range(0, 64, 30):
            v = torch.zeros(32, dtype=torch.float64)
            part = base[lo: lo + 30]
            v[: len(part)] = part
            v[31] = 4.0
            rows += [v * 2.0 ** e, -v * 2.0 ** e]
    _check_quantize(torch.stack(rows).to(TYPES[dtype]).to(gpu_device))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_quantize_ends_of_the_range(gpu_device, dtype):
    """Scales at both ends of the byte: subnormal values, the largest finite ones, zeros of both signs."""
    rows = []
    for e in list(range(-149, -110)) + list(range(115, 128)):
        v = torch.zeros(32, dtype=torch.float64)
        v[:8] = torch.tensor([1.0, 1.5, 1.75, 0.5, 0.25, -0.75, -1.25, 0.125])
        rows.append(v * 2.0 ** e)
    x = torch.stack(rows).to(TYPES[dtype])
    x[:, 9] = -0.0
    x = torch.cat((x, torch.zeros(2, 32, dtype=x.dtype)))
    _check_quantize(x.to(gpu_device))


def test_quantize_infinities_and_nan(gpu_device):
    x = torch.randn(6, 96, generator=torch.Generator().manual_seed(1))
    x[0, 5], x[1, 40], x[2, 95], x[3, 64], x[4, 0] = float("inf"), float("-inf"), float("nan"), -float("nan"), 3.4e38
    for dt in TYPES.values():
        _check_quantize(x.to(dt).to(gpu_device))


def test_quantize_views(gpu_device):
    """Strides, offsets that leave 16 bytes, transposed and expanded tensors, leading dimensions."""
    x = torch.randn(40, 130, generator=torch.Generator().manual_seed(2)).to(gpu_device)
    for v in (x[:, 1:98], x[3:, :64], x[::2, 2:66], x.t(), x[:1].expand(5, 130), x.view(4, 10, 130), x[:, :64].bfloat16()[:, 1:]):
        _check_quantize(v)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_dequantize_every_code(gpu_device, dtype):
    """All codes under all scales; fp16 rounds and overflows as a conversion does."""
    code = np.tile(np.arange(16), (256, 2)).reshape(256, 1, 32)
    byte = np.arange(256).reshape(256, 1)
    t = _ya().Mx4Tensor(torch.from_numpy(mx4_ref.pack(code)).to(gpu_device), torch.from_numpy(byte.astype(np.uint8)).to(gpu_device), 32)
    want = torch.from_numpy(mx4_ref.values(code, byte, 32)).to(TYPES[dtype])
    got = _ya().mx4_dequantize(t, TYPES[dtype]).cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~want.isnan()], want[~want.isnan()])


def _linear_case(dev, rows, n, k, dtype, bias, act, res, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed + rows + 7 * n + 13 * k)
    x = (torch.randn(rows, k, generator=g) * torch.exp(spread * torch.randn(1, k, generator=g))).to(TYPES[dtype])
    w = torch.randn(n, k, generator=g) * k ** -0.5 * torch.exp(spread * torch.randn(n, 1, generator=g))
    b = torch.randn(n, generator=g) if bias else None
    r = torch.randn(rows, n, generator=g).to(TYPES[dtype]) if res else None
    return x.to(dev), w.to(dev), None if b is None else b.to(dev), None if r is None else r.to(dev)


def _check_product(y, xq, wq, b, act, r):
    """xq, wq: the 4-bit values in 64 bits."""
    k = xq.shape[1]
    z = xq @ wq.T
    tol = k * 2.0 ** -24 * (np.abs(xq) @ np.abs(wq).T)
    if b is not None:
        z = z + _np(b)
        tol += 2.0 ** -24 * np.abs(z)
    if act:
        v = z
        with np.errstate(over="ignore"):
            z = v / (1 + np.exp(-v))
        tol = 1.1 * tol + (4 * 2.0 ** -23 + 2 * np.abs(v) * 2.0 ** -24) * np.abs(z) + 2.0 ** -120
    if r is not None:
        z = z + _np(r)
        tol += 2.0 ** -24 * np.abs(z)
    tol += torch.finfo(y.dtype).eps / 2 * (np.abs(z) + tol) + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    bad = np.abs(_np(y) - z) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(_np(y) - z).max(), tol.min())


@pytest.mark.parametrize("rows, n, k", [
    (1, 1, 1), (1, 16, 32), (1, 17, 33), (1, 768, 768), (2, 40, 129), (7, 5, 1000), (16, 16, 128), (16, 1040, 512), (17, 33, 640),
    (31, 256, 2048), (33, 130, 96), (48, 64, 4096), (65, 129, 161), (127, 128, 128), (128, 128, 512), (129, 257, 513), (200, 96, 31),
    (256, 256, 256), (300, 520, 1000), (513, 384, 768), (1030, 260, 544)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_linear_sizes(gpu_device, rows, n, k, dtype):
    ya = _ya()
    x, w, b, r = _linear_case(gpu_device, rows, n, k, dtype, rows % 2, False, n % 2)
    y = ya.mx4_linear(x, ya.mx4_quantize(w), bias=b, res=r)
    assert y.shape == (rows, n) and y.dtype == TYPES[dtype]
    _check_product(y, mx4_ref.rounded(_np(x)), mx4_ref.rounded(_np(w)), b, False, r)


@pytest.mark.parametrize("rows, n, k", [(1, 16400, 1056), (9, 16385, 1100), (2, 300, 60000), (16, 4100, 4128), (70, 4100, 160), (300, 96, 4000)])
@pytest.mark.parametrize("packed", [False, True])
def test_linear_of_few_rows_with_large_weights(gpu_device, rows, n, k, packed):
    ya = _ya()
    x, w, b, r = _linear_case(gpu_device, rows, n, k, "bf16", True, False, True)
    y = ya.mx4_linear(ya.mx4_quantize(x) if packed else x, ya.mx4_quantize(w), bias=b, res=r)
    _check_product(y, mx4_ref.rounded(_np(x)), mx4_ref.rounded(_np(w)), b, False, r)


@pytest.mark.parametrize("rows, n, k", [(1, 72, 160), (40, 200, 288), (400, 304, 416), (2048, 512, 256)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bias, act, res", [(0, 0, 0), (1, 1, 0), (0, 1, 1), (1, 0, 1), (1, 1, 1)])
def test_linear_epilogues(gpu_device, rows, n, k, dtype, bias, act, res):
    ya = _ya()
    x, w, b, r = _linear_case(gpu_device, rows, n, k, dtype, bias, act, res, seed=5)
    y = ya.mx4_linear(x, ya.mx4_quantize(w), bias=b, act=act, res=r)
    _check_product(y, mx4_ref.rounded(_np(x)), mx4_ref.rounded(_np(w)), b, act, r)


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_linear_of_a_quantized_operand_is_the_same(gpu_device, rows):
    ya = _ya()
    x, w, b, _ = _linear_case(gpu_device, rows, 200, 352, "bf16", 1, 1, 0)
    wq = ya.mx4_quantize(w)
    assert torch.equal(ya.mx4_linear(x, wq, bias=b, act=True), ya.mx4_linear(ya.mx4_quantize(x), wq, bias=b, act=True))
    y = ya.mx4_linear(ya.mx4_quantize(x.view(rows, 1, 352)), wq, dtype=torch.float32)
    assert y.shape == (rows, 1, 200) and y.dtype == torch.float32


@pytest.mark.parametrize("rows", [1, 20, 400])
def test_linear_range_and_nan(gpu_device, rows):
    """Scales far from one on both sides cancel; a NaN block makes NaN of its row (or column) and of nothing else."""
    ya = _ya()
    x, w, _, _ = _linear_case(gpu_device, rows, 144, 288, "fp32", 0, 0, 0, spread=0.3)
    y = ya.mx4_linear(x * 2.0 ** 100, ya.mx4_quantize(w * 2.0 ** -100))
    assert torch.equal(y, ya.mx4_linear(x, ya.mx4_quantize(w)))
    x2, w2 = x.clone(), w.clone()
    x2[rows // 2, 287], w2[143, 3] = float("nan"), float("inf")
    z = ya.mx4_linear(x2, ya.mx4_quantize(w2))
    want = torch.zeros_like(z, dtype=torch.bool)
    want[rows // 2], want[:, 143] = True, True
    assert torch.equal(z.isnan(), want) and torch.equal(z[~want], y[~want])


@pytest.mark.parametrize("rows", [1, 9, 300])
def test_linear_views_and_surroundings(gpu_device, rows):
    """Strided activations and residual; nothing outside y is written; the result does not depend on where the operands lie."""
    from yololite_amd import _lib

    ya = _ya()
    x, w, b, r = _linear_case(gpu_device, rows, 90, 200, "bf16", 1, 1, 1)
    wq = ya.mx4_quantize(w)
    want = ya.mx4_linear(x, wq, bias=b, act=True, res=r)
    wide = torch.randn(rows, 333, device=gpu_device).bfloat16()
    wide[:, 5:205], wide[:, 211:301] = x, r
    assert torch.equal(ya.mx4_linear(wide[:, 5:205], wq, bias=b, act=True, res=wide[:, 211:301]), want)
    assert torch.equal(ya.mx4_linear(x.t().contiguous().t(), wq, bias=b, act=True, res=r), want)
    # the C entry with a strided y that is its own residual
    L = _lib.lib()
    y = torch.full((rows + 2, 101), 7.0, device=gpu_device).bfloat16()
    y[1:-1, 3:93] = r
    nbytes = L.yl_mx4_linear_workspace_bytes(0, rows, 90, 200)
    work = torch.empty(nbytes, dtype=torch.uint8, device=gpu_device)
    at = y[1:, 3:].data_ptr()
    rc = L.yl_mx4_linear(x.data_ptr(), None, 0, rows, 200, wq.codes.data_ptr(), wq.scales.data_ptr(), 90, 200, b.data_ptr(), 1, at, 101, at,
                         0, 101, work.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(y[1:-1, 3:93], want)
    y[1:-1, 3:93] = 7.0
    assert bool((y == 7.0).all())


def test_linear_refusals(gpu_device):
    ya = _ya()
    x, w, b, r = _linear_case(gpu_device, 4, 16, 64, "bf16", 1, 0, 1)
    wq = ya.mx4_quantize(w)
    for bad in (dict(x=x[:, :32]), dict(bias=b[:8]), dict(res=r.float()), dict(res=r[:2]), dict(x=x.double()), dict(dtype=torch.float64),
                dict(x=x.cpu()), dict(bias=b.cpu()), dict(x=x.float().requires_grad_()),
                dict(w=ya.Mx4Tensor(wq.codes, wq.scales[:, :1], 64)), dict(w=ya.Mx4Tensor(wq.codes, wq.scales, 65)),
                dict(w=ya.Mx4Tensor(wq.codes.int(), wq.scales, 64)), dict(w=ya.Mx4Tensor(wq.codes[None], wq.scales[None], 64))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ya.mx4_linear(**(dict(x=x, w=wq, bias=b, res=r) | bad))
    assert ya.mx4_linear(x[:0], wq, bias=b).shape == (0, 16) and ya.mx4_quantize(x[:0]).codes.shape == (0, 32)


@pytest.mark.parametrize("rows", [1, 40, 600])
def test_streams_and_graphs(gpu_device, rows):
    """On a side stream; captured, with other work between the replays and new inputs for each."""
    ya = _ya()
    x, w, b, r = _linear_case(gpu_device, rows, 272, 416, "bf16", 1, 1, 1)
    wq = ya.mx4_quantize(w)
    inputs = [x, -x, x.flip(0) * 3]
    want = [ya.mx4_linear(v, wq, bias=b, act=True, res=r) for v in inputs]
    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ya.mx4_linear(x, wq, bias=b, act=True, res=r)
    side.synchronize()
    assert torch.equal(got, want[0])
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ya.mx4_linear(static, wq, bias=b, act=True, res=r)
        back = ya.mx4_dequantize(ya.mx4_quantize(static))
    for k in (0, 1, 2, 1):
        static.copy_(inputs[k])
        graph.replay()
        ya.mx4_linear(inputs[(k + 1) % 3], wq)  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out, want[k]) and torch.equal(back, ya.mx4_dequantize(ya.mx4_quantize(inputs[k])))
