"""GPU: calls of the operators' Python faces that are refused where the call below would do something else."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_block_sizes_that_32_bits_do_not_hold(gpu_device):
    """2^32 + 64 is not 64."""
    import yololite_amd as ya

    q = torch.randn(1, 10, 2, 32, device=gpu_device).bfloat16()
    k = torch.randn(1, 100, 2, 32, device=gpu_device).bfloat16()
    picked = ya.block_select(q, k, block=64, topk=2)
    for bad in (dict(block=2 ** 32 + 64), dict(block=64 - 2 ** 32), dict(topk=2 ** 32 + 2), dict(topk=-1), dict(block=-64)):
        with pytest.raises(NotImplementedError):
            ya.block_select(q, k, **(dict(block=64, topk=2) | bad))
    for block in (2 ** 32 + 64, 64 - 2 ** 32, -64):
        with pytest.raises(NotImplementedError):
            ya.block_attention(q, k, k, picked, block=block)
    far = q[:, :1].expand(1, 2 ** 32 + 10, 2, 32)
    with pytest.raises(NotImplementedError):
        ya.block_select(far, k, block=64, topk=2)
    with pytest.raises(NotImplementedError):
        ya.block_attention(far, k, k, picked[:, :, :1].expand(1, 2, 2 ** 32 + 10, 2), block=64)
    with pytest.raises(NotImplementedError):
        ya.block_select(q, k[:, :1].expand(1, 2 ** 32 + 100, 2, 32), block=64, topk=2)
