"""GPU: block selection is equal to the 64-bit restatement's; attention against 64-bit softmax over the same blocks.

Tolerance of an output: a score's fp32 sum of dk products is off by at most dk 2^-24 sum |q k| scale, its scaling by 2 2^-24 of that;
a softmax weight then by twice that much, relatively (its own score and the sum's), plus 4 2^-23 for the exponentials and 2 n 2^-24 for
the two sums over n keys; weights are rounded to the tensors' type before the product with v: eps / 2 each (fp16: and half of its
smallest step, 2^-25, under its normal range), and so are a block's results before they are joined: eps / 2 of a weighted mean of |v|
(and 2^-25 in fp16).  All of these weigh |v|.  The result's rounding adds eps / 2 of it."""
import numpy as np
import pytest
import torch

from tests import block_ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _ya():
    import yololite_amd as ya

    return ya


def _np(t):
    return t.double().cpu().numpy()


def _inputs(dev, b, nq, nk, heads, kv, dk, dv, dtype="bf16", seed=0):
    g = torch.Generator().manual_seed(seed + nq + 3 * nk + 5 * dk)

    def field(n, h, d):  # neighbours alike, as on a map
        part = torch.randn(b, n // 24 + 1, h, d, generator=g).repeat_interleave(24, 1)[:, :n]
        return (0.8 * part + 0.6 * torch.randn(b, n, h, d, generator=g)).to(TYPES[dtype]).to(dev)

    return field(nq, heads, dk), field(nk, kv, dk), torch.randn(b, nk, kv, dv, generator=g).to(TYPES[dtype]).to(dev)


def _np_mask(mask):
    return None if mask is None else mask.cpu().numpy().astype(bool)


def _check_select(q, k, block, topk, mask=None):
    got = _ya().block_select(q, k, block=block, topk=topk, mask=mask)
    assert got.dtype == torch.int32
    want = block_ref.select(_np(q), _np(k), block, topk, _np_mask(mask))
    assert np.array_equal(got.cpu().numpy(), want), np.argwhere(got.cpu().numpy() != want)[:5]
    return got


def _check_attend(q, k, v, picked, block, mask=None, scale=None, rows=None):
    got = _ya().block_attention(q, k, v, picked, block=block, mask=mask, scale=scale)
    assert got.dtype == q.dtype and got.shape == (*q.shape[:3], v.shape[3])
    qn, pn, gn = _np(q), picked.cpu().numpy(), _np(got)
    if rows is not None:  # a sample of the queries of a long map
        qn, pn, gn = qn[:, rows], pn[:, :, rows], gn[:, rows]
    m = _np_mask(mask)
    kn, vn = _np(k), _np(v)
    if m is not None:  # what a masked key or value holds does not matter
        kn[~m], vn[~m] = 0, 0
    want, mass, work = block_ref.attend(qn, kn, vn, pn, block, m, scale)
    dk, n = q.shape[3], picked.shape[3] * block
    eps = torch.finfo(q.dtype).eps
    rel = 2 * (dk + 2) * 2.0 ** -24 * work + 4 * 2.0 ** -23 + 2 * n * 2.0 ** -24 + 2 * eps / 2
    tol = rel * mass + 2.0 ** -25 * (n * (np.abs(vn).max() if vn.size else 0) + 1) * (q.dtype == torch.float16)
    tol += eps / 2 * (np.abs(want) + tol) + 1e-30
    assert (np.abs(gn - want) <= tol).all(), (np.abs(gn - want) / tol).max()
    return got


SHAPES = [  # b, nq, nk, heads, kv, dk, dv, block, topk
    (1, 1, 1, 1, 1, 8, 8, 32, 1), (1, 1, 31, 1, 1, 32, 64, 32, 4), (2, 1, 33, 2, 1, 16, 32, 32, 1), (1, 1, 1000, 8, 8, 64, 64, 64, 4),
    (3, 1, 700, 4, 2, 128, 128, 128, 3), (2, 5, 129, 6, 6, 32, 64, 64, 2), (1, 17, 64, 3, 3, 32, 64, 64, 8), (2, 100, 100, 2, 2, 32, 64, 32, 2),
    (1, 65, 513, 8, 2, 64, 64, 64, 4), (1, 130, 300, 12, 1, 40, 24, 32, 5), (2, 400, 400, 2, 2, 32, 64, 64, 3), (1, 333, 260, 16, 1, 128, 96, 128, 2),
    (1, 257, 2100, 1, 1, 80, 128, 32, 16), (1, 70, 4200, 2, 1, 24, 56, 32, 64), (4, 63, 96, 5, 5, 8, 120, 32, 3), (1, 260, 515, 2, 1, 64, 32, 128, 4)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_sizes(gpu_device, shape, dtype):
    *sizes, block, topk = shape
    q, k, v = _inputs(gpu_device, *sizes, dtype=dtype)
    picked = _check_select(q, k, block, topk)
    _check_attend(q, k, v, picked, block)


@pytest.mark.parametrize("shape", SHAPES[2:], ids=lambda s: "x".join(map(str, s)))
def test_masks(gpu_device, shape):
    """Padded maps, holes, a whole image masked; infinities and NaN where nothing may be read."""
    *sizes, block, topk = shape
    b, nq, nk = sizes[:3]
    q, k, v = _inputs(gpu_device, *sizes, seed=9)
    g = torch.Generator().manual_seed(nk)
    mask = torch.rand(b, nk, generator=g) < 0.7
    mask[0, nk - nk // 3:] = False
    if nk > 2 * block:
        mask[0, block: 2 * block] = False
    if b > 1:
        mask[-1] = False
    mask = mask.to(gpu_device)
    k[~mask], v[~mask] = float("nan"), float("inf")
    for m in (mask, mask.to(torch.uint8) * 255):
        picked = _check_select(q, k, block, topk, m)
        out = _check_attend(q, k, v, picked, block, m)
    if b > 1:
        assert bool((picked[-1] == -1).all()) and bool((out[-1] == 0).all())


def test_no_keys(gpu_device):
    q, k, v = _inputs(gpu_device, 2, 3, 0, 2, 1, 32, 64)
    picked = _check_select(q, k, 64, 2)
    assert bool((picked == -1).all())
    assert bool((_check_attend(q, k, v, picked, 64) == 0).all())
    q, k, v = _inputs(gpu_device, 2, 0, 50, 2, 1, 32, 64)
    assert _ya().block_attention(q, k, v, _ya().block_select(q, k)).shape == (2, 0, 2, 64)


@pytest.mark.parametrize("nq", [1, 3, 90])
def test_ties_go_to_the_lower_index(gpu_device, nq):
    """Blocks alike (all of them; in pairs), scores of zero of both signs, queries of zeros."""
    b, kv, dk, block, nb = 2, 2, 32, 32, 21
    q, _, v = _inputs(gpu_device, b, nq, nb * block, 2, kv, dk, 64)
    one = torch.randn(b, 1, kv, dk, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu_device)
    same = one.expand(b, nb * block, kv, dk)
    assert _check_select(q, same, block, 5)[0, 0, 0].tolist() == [0, 1, 2, 3, 4]
    pairs = torch.randn(b, (nb + 1) // 2, kv, dk, generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu_device)
    pairs = pairs.repeat_interleave(2, 1)[:, :nb].repeat_interleave(block, 1)
    for topk in (1, 4, 7, nb, nb + 3):
        _check_select(q, pairs, block, topk)
    q[:, ::2] = 0
    _check_select(q, -pairs, block, 6)


@pytest.mark.parametrize("nq", [1, 70])
def test_scores_next_to_each_other(gpu_device, nq):
    """Blocks whose means differ in the last bit of one dim of one key: far below fp32's resolution of a score."""
    b, kv, dk, block, nb = 1, 1, 64, 64, 40
    q = torch.randn(b, nq, 1, dk, generator=torch.Generator().manual_seed(3)).bfloat16().to(gpu_device)
    k = (torch.randn(1, 1, 1, dk, generator=torch.Generator().manual_seed(4)).bfloat16().repeat(1, nb * block, 1, 1)).to(gpu_device)
    at = torch.arange(nb, device=gpu_device) * block
    k[0, at, 0, 5] = (1e-4 * (torch.arange(nb, device=gpu_device) * 7 % nb + 1)).bfloat16()
    for topk in (1, 8, 39):
        _check_select(q, k, block, topk)


def test_scores_that_are_not_finite(gpu_device):
    q, k, v = _inputs(gpu_device, 1, 40, 400, 2, 1, 32, 64)
    k[0, 70, 0, 3], k[0, 200, 0, 0] = float("nan"), float("inf")
    q[0, 5, 0, 1] = float("nan")
    _check_select(q, k, 32, 12)  # of 13 blocks


@pytest.mark.parametrize("heads, kv", [(1, 1), (6, 6), (8, 2), (16, 1), (20, 1), (6, 2)])
@pytest.mark.parametrize("nq, nk", [(1, 900), (50, 900), (900, 900)])
def test_head_layouts(gpu_device, heads, kv, nq, nk):
    q, k, v = _inputs(gpu_device, 1, nq, nk, heads, kv, 32, 64, seed=4)
    picked = _check_select(q, k, 64, 4)
    _check_attend(q, k, v, picked, 64, rows=np.arange(0, nq, 7))


@pytest.mark.parametrize("nq", [3, 37])
@pytest.mark.parametrize("nb", [257, 512, 513, 1024, 1025, 2049, 4096])
def test_many_blocks(gpu_device, nb, nq):
    """Few queries and more over hundreds and thousands of blocks: ordinary scores, masked blocks, ties across the whole range,
    scores that are not finite."""
    nk = nb * 32 - 5
    q, k, _ = _inputs(gpu_device, 2, nq, nk, 4, 2, 40, 8, seed=nb)
    _check_select(q, k, 32, 64)
    mask = (torch.rand(2, nk, generator=torch.Generator().manual_seed(nb)) < 0.6).to(gpu_device)
    mask[0, nk // 3: nk // 2] = False
    mask[1, 32 * 9:] = False
    bad = k.clone()
    bad[~mask] = float("nan")
    _check_select(q, bad, 32, 11, mask)
    few = k[:, :: 32 * 64].repeat_interleave(32 * 64, 1)[:, :nk]  # 64 neighbours alike, and whole waves of them
    _check_select(q, few, 32, 7)
    _check_select(q, k[:, :1].expand(2, nk, 2, 40), 32, 64)
    k[0, nk // 2, 0, 3], k[0, nk - 1, 1, 0], q[1, 1, 0, 1], q[1, nq - 1] = float("nan"), float("inf"), float("nan"), 0
    _check_select(q, k, 32, 5)


def test_any_list_of_blocks(gpu_device):
    """Random order, blocks named twice, indices that name no block, empty lists, one block for every query."""
    q, k, v = _inputs(gpu_device, 2, 150, 600, 4, 2, 64, 64, seed=11)
    g = torch.Generator().manual_seed(0)
    picked = torch.randint(-3, 14, (2, 2, 150, 9), generator=g).int()
    picked[0, 0, 7], picked[1, 1, 3], picked[0, 1, 50:120] = -1, 4, 9
    picked[1, 0, 0, 0], picked[1, 0, 0, 1] = 2 ** 31 - 1, -2 ** 31
    picked = picked.to(gpu_device)
    out = _check_attend(q, k, v, picked, 64)
    assert bool((out[0, 7, :2] == 0).all())
    perm = picked[..., torch.randperm(9, generator=g).to(gpu_device)]
    again = _ya().block_attention(q, k, v, perm, block=64)
    _check_attend(q, k, v, perm, 64)
    assert torch.allclose(again.float(), out.float(), atol=0.05)
    one = picked[:, :, :1, :1].clone()
    _check_attend(q[:, :1], k, v, one, 64)


def test_scales_and_large_scores(gpu_device):
    q, k, v = _inputs(gpu_device, 1, 80, 300, 2, 2, 32, 64)
    picked = _check_select(q, k, 64, 3)
    for scale in (0.0, 1.0, -0.5):
        _check_attend(q, k, v, picked, 64, scale=scale)
    _check_attend(q * 8, k * 8, v, picked, 64, scale=1.0)  # scores of thousands: one key takes all
    lowest = torch.finfo(torch.bfloat16).min
    v2 = v.clone()
    v2[0, 10:20] = lowest
    got = _ya().block_attention(q, k, v2, picked, block=64)
    assert not bool(got.isnan().any())


def test_strides(gpu_device):
    """A packed q | k | v map as the network stores it, heads in front of tokens, views that need a copy, broadcast keys."""
    b, n, heads, dk, dv = 2, 140, 3, 32, 64
    g = torch.Generator().manual_seed(6)
    qkv = torch.randn(b, n, heads, 2 * dk + dv, generator=g).bfloat16().to(gpu_device)
    q, k, v = qkv[..., :dk], qkv[..., dk: 2 * dk], qkv[..., 2 * dk:]
    picked = _check_select(q, k, 32, 3)
    want = _check_attend(q, k, v, picked, 32)
    ya = _ya()
    flip = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]
    assert torch.equal(ya.block_attention(*flip, picked, block=32), want)
    odd = torch.zeros(b, n, heads, dk + 3, device=gpu_device, dtype=torch.bfloat16)
    odd[..., 1: dk + 1] = q
    assert torch.equal(ya.block_attention(odd[..., 1: dk + 1], k, v, picked, block=32), want)
    assert torch.equal(ya.block_select(odd[..., 1: dk + 1], k, block=32, topk=3), picked)
    wide = torch.zeros(b, n, 40, device=gpu_device, dtype=torch.bool)
    wide[..., 3] = True
    assert torch.equal(ya.block_attention(q, k, v, picked, block=32, mask=wide[..., 3]), want)
    _check_attend(q, k[:1].expand(b, n, heads, dk), v[:, :, :1].expand(b, n, heads, dv), picked, 32)


def test_long_maps(gpu_device):
    """More than 2048 blocks; keys and values behind a 2^31-byte offset, reached through their strides."""
    q, k, v = _inputs(gpu_device, 1, 2, 32 * 2500 + 5, 1, 1, 32, 32)
    _check_attend(q, k, v, _check_select(q, k, 32, 16), 32)
    room = torch.zeros((1 << 30) + 8192, dtype=torch.bfloat16, device=gpu_device)
    far = room.as_strided((2, 64, 1, 32), (1 << 30, 32, 32, 1))
    q, k, v = _inputs(gpu_device, 2, 40, 64, 1, 1, 32, 32)
    far.copy_(k)
    picked = _check_select(q, far, 32, 1)
    _check_attend(q, far, v, picked, 32)
    far.copy_(v)
    _check_attend(q, k, far, picked, 32)


@pytest.mark.parametrize("nq, topk, block", [(1, 1, 64), (1, 3, 64), (3, 64, 128), (90, 1, 32), (90, 5, 64), (200, 64, 128)])
@pytest.mark.parametrize("exponent", [127, 90, -60, -100])
def test_ends_of_the_range_of_values(gpu_device, nq, topk, block, exponent):
    """Every value next to the largest (or tiny): no sum on the way leaves the range."""
    q, k, v = _inputs(gpu_device, 1, nq, 64 * 128 if topk == 64 else 300, 2, 1, 32, 32)
    v = (v.sign() * (2 - 2.0 ** -7) * 2.0 ** (exponent / 2) * 2.0 ** (exponent - exponent / 2)).bfloat16()
    v[..., 3] = v[..., 3].abs()
    v[..., 4:] = torch.where(torch.rand(v[..., 4:].shape, generator=torch.Generator().manual_seed(1)).to(gpu_device) < 0.9, v[..., 4:], 0)
    picked = _check_select(q, k, block, topk)
    out = _check_attend(q, k, v, picked, block)
    assert torch.equal(out[..., 3], v[0, 0, 0, 3].expand_as(out[..., 3]))


def test_queries_far_apart(gpu_device):
    """Queries and keys whose token strides do not fit 24 bits, with one and with several heads."""
    room = torch.zeros((40 << 24) + 4096, dtype=torch.bfloat16, device=gpu_device)
    for heads in (1, 2):
        q, k, v = _inputs(gpu_device, 1, 40, 130, heads, 1, 32, 32, seed=heads)
        far = room.as_strided((1, 40, heads, 32), (8, 1 << 24, 40, 1))
        far.copy_(q)
        picked = _check_select(far, k, 32, 2)
        _check_attend(far, k, v, picked, 32)
        _check_attend(far[:, :3], k, v, picked[:, :, :3], 32)


def test_refusals(gpu_device):
    ya = _ya()
    q, k, v = _inputs(gpu_device, 1, 10, 100, 4, 2, 32, 64)
    picked = ya.block_select(q, k, block=64, topk=2)
    mask = torch.ones(1, 100, dtype=torch.bool, device=gpu_device)
    for bad in (dict(q=q.float()), dict(k=k.half()), dict(q=q[0]), dict(q=q[:, :, :3]), dict(k=k[..., :16]), dict(mask=mask.int()),
                dict(mask=mask[:, :50]), dict(block=48), dict(q=q.cpu()), dict(q=q.clone().requires_grad_())):
        with pytest.raises((ValueError, TypeError, RuntimeError, NotImplementedError)):
            ya.block_select(**(dict(q=q, k=k, block=64, topk=2) | bad))
        with pytest.raises((ValueError, TypeError, RuntimeError, NotImplementedError)):
            ya.block_attention(**(dict(q=q, k=k, v=v, picked=picked, block=64) | bad))
    for bad in (dict(v=v[:, :50]), dict(v=v.half()), dict(picked=picked.long()), dict(picked=picked[:, :1]), dict(v=v[..., :60])):
        with pytest.raises((ValueError, TypeError, RuntimeError, NotImplementedError)):
            ya.block_attention(**(dict(q=q, k=k, v=v, picked=picked, block=64) | bad))
    for topk in (0, 65):
        with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
            ya.block_select(q, k, topk=topk)


@pytest.mark.parametrize("nq, nk", [(1, 2000), (300, 900)])
def test_streams_and_graphs(gpu_device, nq, nk):
    """On a side stream; captured, with other work between the replays and new inputs for each; two graphs on two streams at once."""
    ya = _ya()

    def both(q, k, v, mask):
        picked = ya.block_select(q, k, block=64, topk=4, mask=mask)
        return picked, ya.block_attention(q, k, v, picked, block=64, mask=mask)

    q, k, v = _inputs(gpu_device, 2, nq, nk, 4, 2, 64, 64)
    mask = torch.rand(2, nk, generator=torch.Generator().manual_seed(0)).to(gpu_device) < 0.8
    inputs = [(q, k, v), (-q, k.flip(1), v * 2), (q * 0.5, -k, v.flip(1))]
    want = [both(*t, mask) for t in inputs]
    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(*inputs[0], mask)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want[0]))
    graphs, held, outs = [], [], []
    for _ in range(2):
        t = [x.clone() for x in inputs[0]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(*t, mask)
        graphs.append(graph), held.append(t), outs.append(out)
    for step in ((0, 1), (1, 2), (2, 0), (2, 1)):
        for t, s in zip(held, step):
            for x, y in zip(t, inputs[s]):
                x.copy_(y)
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        both(*inputs[step[0]], mask)  # eager work beside the replays
        torch.cuda.synchronize()
        for out, s in zip(outs, step):
            assert all(torch.equal(x, y) for x, y in zip(out, want[s]))


def test_together_as_an_attention_stage(gpu_device):
    """qkv product in 4 bits, selection, attention, output product: a PSA block's attention half on a padded map, each stage
    against the restatements on that stage's own inputs."""
    from tests import mx4_ref
    from tests.test_gpu_mx4 import _check_product

    ya = _ya()
    b, n, c, heads, dk, dv = 2, 324, 192, 3, 32, 64
    g = torch.Generator().manual_seed(8)
    x = torch.randn(b, n, c, generator=g).bfloat16().to(gpu_device)
    w1 = (torch.randn(heads * (2 * dk + dv), c, generator=g) * c ** -0.5).to(gpu_device)
    w2 = (torch.randn(c, heads * dv, generator=g) * (heads * dv) ** -0.5).to(gpu_device)
    bias = torch.randn(c, generator=g).to(gpu_device)
    mask = torch.ones(b, n, dtype=torch.bool, device=gpu_device)
    mask[1, 200:] = False
    qkv = ya.mx4_linear(x, ya.mx4_quantize(w1))
    _check_product(qkv.view(b * n, -1), mx4_ref.rounded(_np(x).reshape(b * n, c)), mx4_ref.rounded(_np(w1)), None, False, None)
    q, k, v = qkv.view(b, n, heads, 2 * dk + dv).split((dk, dk, dv), -1)
    picked = _check_select(q, k, 64, 2, mask)
    o = _check_attend(q, k, v, picked, 64, mask)
    y = ya.mx4_linear(o.view(b, n, -1), ya.mx4_quantize(w2), bias=bias, res=x)
    _check_product(y.view(b * n, c), mx4_ref.rounded(_np(o).reshape(b * n, -1)), mx4_ref.rounded(_np(w2)), bias, False, x.view(b * n, c))


@pytest.mark.parametrize("b, nh, h, w, block, topk", [(2, 2, 20, 20, 64, 3), (1, 1, 7, 5, 32, 1), (3, 4, 13, 7, 32, 2), (2, 1, 40, 40, 128, 4),
                                                      (1, 2, 20, 1, 32, 1), (1, 6, 40, 40, 64, 8), (2, 1, 2, 2, 32, 2)])
def test_engine_op_on_the_networks_maps(gpu_device, b, nh, h, w, block, topk):
    """YL_OP_ATTENTION with grp != 0 on planar guarded maps: the bits of the direct calls on the same tokens, guards untouched."""
    from tests.hip_util import Mini
    from yololite_amd import _lib
    from yololite_amd.nn.lower import OP_ATTENTION

    g = torch.Generator().manual_seed(h * w)
    qkv = torch.randn(b, nh * 128, h, w, generator=g).bfloat16()
    m = Mini(b, gpu_device)
    xin, out = m.buf(h, w, nh * 128 + 16).slice(16, nh * 128), m.buf(h, w, nh * 64 + 8).slice(8, nh * 64)
    m.fill(xin, qkv.float())
    scratch = m.ar.alloc_bytes(_lib.lib().yl_attention_scratch_bytes(b, nh, h * w, block, topk))
    m.op(kind=OP_ATTENTION, name="attn", heads=nh, key_dim=32, head_dim=64, scale=32 ** -0.5, inp=xin, out=out, grp=block, topk=topk,
         scratch=scratch)
    m.run()
    assert m.eng.op_kernel(0) == "block_attention"
    got = m.read(out)
    t = qkv.to(gpu_device).view(b, nh, 128, h * w).permute(0, 3, 1, 2).contiguous()
    q, k, v = t.split((32, 32, 64), -1)
    picked = _check_select(q, k, block, topk)
    want = _check_attend(q, k, v, picked, block, rows=np.arange(0, h * w, 13))
    assert torch.equal(got, want.permute(0, 2, 3, 1).reshape(b, nh * 64, h, w).float().cpu())


def test_engine_op_refusals(gpu_device):
    from tests.hip_util import Mini
    from yololite_amd.nn.lower import OP_ATTENTION

    for change in (dict(grp=48), dict(topk=65), dict(scratch=1 << 40), dict(scratch=100), dict(scratch=-1)):
        m = Mini(1, gpu_device)
        xin, out = m.buf(20, 20, 128), m.buf(20, 20, 64)
        m.op(**(dict(kind=OP_ATTENTION, name="attn", heads=1, key_dim=32, head_dim=64, scale=1.0, inp=xin, out=out, grp=64, topk=2,
                     scratch=m.ar.alloc_bytes(1 << 20)) | change))
        with pytest.raises((RuntimeError, NotImplementedError)):
            m.run()


def test_network_with_selected_blocks(gpu_device, monkeypatch):
    """YL_PSA_TOPK through the whole network: eager and replayed graphs agree on changing inputs; with the knob unset nothing has
    changed."""
    from yololite_amd.nn import arch
    from yololite_amd.nn.engine import HipEngine
    from yololite_amd.nn.synth import synth_state_dict

    specs, _ = arch.parse_model(arch.yolo11_dict("n"))
    sd = synth_state_dict("n", 0)
    g = torch.Generator().manual_seed(5)
    xs = [torch.rand(2, 3, 640, 640, generator=g).to(gpu_device) for _ in range(2)]

    def engine():
        return HipEngine.from_model(specs, sd, 2, 640, 640, gpu_device)

    dense = engine()
    y_dense = [dense.forward(x).clone() for x in xs]
    monkeypatch.setenv("YL_PSA_TOPK", "3")
    eng = engine()
    want = [eng.forward(x).clone() for x in xs]
    assert not torch.equal(want[0], y_dense[0]) and bool(torch.isfinite(want[0]).all())
    buf, y = torch.empty_like(xs[0]), torch.empty_like(want[0])
    for k in (0, 1, 0, 1):
        buf.copy_(xs[k])
        eng.forward(buf, y=y, graph=True)
        eng.forward(xs[1 - k])  # eager work between the replays
        buf.copy_(xs[k])
        eng.forward(buf, y=y, graph=True)
        torch.cuda.synchronize()
        assert torch.equal(y, want[k])
    monkeypatch.delenv("YL_PSA_TOPK")
    assert torch.equal(engine().forward(xs[0]), y_dense[0])
