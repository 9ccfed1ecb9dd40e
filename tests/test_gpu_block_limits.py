"""GPU: few queries and few blocks of very many images (all alike, by strides of 0)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nk", [60, 90])
def test_many_images(gpu_device, nk):
    """2^24 images of two and three blocks: 2^32 threads, were they the one launch of four waves to an image that fewer images are."""
    import yololite_amd as ya

    g = torch.Generator().manual_seed(nk)
    batch = (1 << 24) + 5
    q, k = (torch.randn(1, n, 1, 8, generator=g).bfloat16().to(gpu_device) for n in (1, nk))
    one = ya.block_select(q, k, block=32, topk=2)
    many = ya.block_select(q.expand(batch, -1, -1, -1), k.expand(batch, -1, -1, -1), block=32, topk=2)
    assert many.shape == (batch, 1, 1, 2) and bool((many == one).all())
