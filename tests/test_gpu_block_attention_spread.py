"""GPU: attention over selected blocks where the values of one block differ widely in size, and in several passes over its block
results.  Tolerances as in test_gpu_block_attention.py: they are relative to each channel's own sum of weights times |v|."""
import numpy as np
import pytest
import torch

from tests.test_gpu_block_attention import _check_attend, _inputs, _ya

pytestmark = pytest.mark.gpu
FORMS = [(1, 64), (90, 64), (700, 32), (700, 64), (700, 128)]  # queries, block: one launch for few queries, lists for many


@pytest.mark.parametrize("dv", [64, 96, 24])
@pytest.mark.parametrize("nq, block", FORMS)
@pytest.mark.parametrize("bits", [10, 20, 24, 30, 40, 60, 120])
def test_channels_of_different_size(gpu_device, nq, block, dv, bits):
    """Channels 2^(bits / 2) .. 2^-(bits / 2), neighbours and far apart."""
    q, k, v = _inputs(gpu_device, 1, nq, 700, 6, 3, 32, dv, seed=bits)
    size = 2.0 ** (bits // 2 - (torch.arange(dv) * 7 % dv * bits / (dv - 1)).round())
    v = (v.float() * size.to(gpu_device)).bfloat16()
    picked = _ya().block_select(q, k, block=block, topk=8)
    _check_attend(q, k, v, picked, block, rows=np.arange(0, nq, 9))


@pytest.mark.parametrize("nq, block", FORMS)
@pytest.mark.parametrize("bits", [20, 30, 45, 100])
def test_large_values_that_have_no_weight(gpu_device, nq, block, bits):
    """Keys with values 2^bits times the others', which no query looks at: their weight is 2^-140."""
    q, k, v = _inputs(gpu_device, 1, nq, 700, 6, 3, 32, 64, seed=bits)
    q[..., 0], k[..., 0] = 24.0, 0.0
    far = torch.arange(0, 700, 5, device=gpu_device)
    k[:, far, :, 0] = -24.0
    v[:, far] *= 2.0 ** bits
    picked = _ya().block_select(q, k, block=block, topk=8)
    _check_attend(q, k, v, picked, block, rows=np.arange(0, nq, 9))


@pytest.mark.parametrize("nq, block", FORMS)
def test_channels_and_keys_of_zeros(gpu_device, nq, block):
    """Channels that are zero in every key, in some blocks, and single values among zeros."""
    q, k, v = _inputs(gpu_device, 1, nq, 700, 6, 3, 32, 64, seed=2)
    v[..., ::5] = 0
    v[:, :350, :, 1] = 0
    v[..., 3] *= (torch.arange(700, device=gpu_device) % 61 == 0)[None, :, None]
    picked = _ya().block_select(q, k, block=block, topk=8)
    out = _check_attend(q, k, v, picked, block, rows=np.arange(0, nq, 9))
    assert bool((out[..., ::5] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_several_passes_over_the_block_results(gpu_device, dtype):
    """16 query heads x 64 results of width 128: 1024 queries in bf16 (512 in fp16) to a pass of 256 MiB.  The same queries in calls of one
    pass each, a call once more, and the definition for some of them."""
    nq, part = 2500, 500
    q, k, v = _inputs(gpu_device, 1, nq, 64 * 128 - 7, 16, 4, 32, 128, dtype=dtype)
    v[:, 100:200] = 0  # (some blocks' results in fp32)
    picked = _ya().block_select(q, k, block=128, topk=32)
    out = _check_attend(q, k, v, picked, 128, rows=np.array([0, 511, 512, 1023, 1024, 1500, 2047, 2048, nq - 1]))
    assert torch.equal(out, _ya().block_attention(q, k, v, picked, block=128))
    for i in range(0, nq, part):
        got = _ya().block_attention(q[:, i: i + part], k, v, picked[:, :, i: i + part].contiguous(), block=128)
        assert torch.equal(got, out[:, i: i + part])
