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


def test_tangents_are_refused(gpu_device):
    """Forward-mode derivatives: a dual tensor loses its tangent nowhere, under no_grad neither; other tensors pass inside a dual level."""
    from torch.autograd import forward_ad

    import yololite_amd as ya

    x = torch.randn(4, 64, device=gpu_device)
    w = ya.mx4_quantize(torch.randn(16, 64, device=gpu_device))
    q = torch.randn(1, 10, 2, 32, device=gpu_device).bfloat16()
    picked = ya.block_select(q, q, block=32, topk=1)
    with forward_ad.dual_level():
        dx, dq = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(q, torch.ones_like(q))
        calls = [lambda: ya.mx4_quantize(dx), lambda: ya.mx4_linear(dx, w), lambda: ya.mx4_linear(x, w, bias=dx[0, :16]),
                 lambda: ya.mx4_linear(x, w, res=dx[:, :16]), lambda: ya.block_select(dq, q), lambda: ya.block_select(q, dq),
                 lambda: ya.block_attention(q, q, dq, picked, block=32)]
        for call in calls:
            with pytest.raises(RuntimeError, match="derivative"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="derivative"):
                call()
        inside = ya.mx4_linear(x, w), ya.block_attention(q, q, q, ya.block_select(q, q, block=32, topk=1), block=32)
        y = torch.zeros_like(x, requires_grad=True)
        with pytest.raises(RuntimeError, match="no backward"):
            ya.mx4_quantize(y)
        with torch.no_grad():
            ya.mx4_quantize(y)
    assert torch.equal(inside[0], ya.mx4_linear(x, w)) and torch.equal(inside[1], ya.block_attention(q, q, q, picked, block=32))
