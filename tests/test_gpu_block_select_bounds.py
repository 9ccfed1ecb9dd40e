"""GPU: the selection equals the 64-bit one where the scores in fewer bits say least: query heads that cancel, keys and queries whose
squares are below fp32's range, values that two bf16 hold worst.  The restatement sorts 64-bit scores; nothing is rounded but its sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _select64(q, k, block, topk):
    """(b, kv, nq, topk) from the definition, on the CPU in 64 bits."""
    q, k = q.double().cpu(), k.double().cpu()
    b, nq, heads, dk = q.shape
    nk, kv = k.shape[1:3]
    nb = -(-nk // block)
    mean = torch.stack([k[:, j * block: (j + 1) * block].mean(1) for j in range(nb)], 2)  # (b, kv, nb, dk)
    score = torch.matmul(q.view(b, nq, kv, heads // kv, dk).sum(3).permute(0, 2, 1, 3).contiguous(), mean.transpose(2, 3).contiguous())
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :topk]
    return torch.nn.functional.pad(order.sort(-1).values, (0, topk - order.shape[-1]), value=-1)


def _check(q, k, block, topk):
    import yololite_amd as ya

    got = ya.block_select(q, k, block=block, topk=topk).cpu().long()
    wrong = (got != _select64(q, k, block, topk)).any(-1)
    assert not bool(wrong.any()), f"{int(wrong.sum())} of {wrong.numel()} queries"


# blocks and queries for each way the scores are made: a wave up to 64, 128, 256 blocks, four and eight waves
WAYS = [(60, 300), (100, 300), (200, 300), (200, 32768), (400, 300), (400, 9000), (1000, 300), (2000, 100), (4000, 60)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("nb, nq", WAYS)
def test_heads_that_cancel(gpu_device, nb, nq, dtype):
    """Heads a, s, -a, t with |s|, |t| = 2^-14 .. 2^-24 of |a|: the sum is s + t, what fp32 makes of it on the way is not."""
    g = torch.Generator().manual_seed(nb + nq)
    dk, block = 64, 32
    k = torch.randn(1, nb * block, 1, dk, generator=g).to(TYPES[dtype])
    a = 16 * torch.randn(1, nq, 1, dk, generator=g)
    ratio = 2.0 ** -torch.linspace(14, 24, nq).view(1, nq, 1, 1)
    s, t = (16 * ratio * torch.randn(1, nq, 1, dk, generator=g) for _ in range(2))
    q = torch.cat((a, s, -a, t), 2).to(TYPES[dtype])
    _check(q.to(gpu_device), k.to(gpu_device), block, 8)


@pytest.mark.parametrize("heads", [2, 3, 7])
def test_other_numbers_of_heads_that_cancel(gpu_device, heads):
    g = torch.Generator().manual_seed(heads)
    nq, dk = 1000, 64
    k = torch.randn(1, 100 * 32, 1, dk, generator=g).bfloat16()
    a = torch.randn(1, nq, 1, dk, generator=g).bfloat16().float()
    s = 2.0 ** -20 * torch.randn(1, nq, heads - 1, dk, generator=g)
    q = torch.cat((a, s), 2)
    q[:, :, -1] += -a[:, :, 0] * (1 + 2.0 ** -7 * (heads == 2))
    _check(q.bfloat16().to(gpu_device), k.to(gpu_device), 32, 8)


@pytest.mark.parametrize("nb", [40, 100, 250, 500, 1000])
@pytest.mark.parametrize("kexp, qexp", [(-60, 0), (-70, 0), (-78, 0), (-90, 0), (0, -78), (-78, 70), (60, -90), (-40, -40), (-62, -62)])
def test_squares_below_the_range(gpu_device, nb, kexp, qexp):
    """Blocks whose means differ in the last bits of few keys, times powers of two: the order is the same at every scale."""
    nq, dk, block = 200, 64, 64
    g = torch.Generator().manual_seed(nb)
    q = torch.randn(1, nq, 1, dk, generator=g).bfloat16()
    base = torch.randn(1, 1, 1, dk, generator=g).bfloat16()
    k = base.repeat(1, nb * block, 1, 1)
    at = torch.arange(nb) * block
    for d in (5, 9, 33):
        k[0, at, 0, d] = (base[0, 0, 0, d].float() * (1 + 2.0 ** -7 * torch.randint(-3, 4, (nb,), generator=g))).bfloat16()
        k[0, at + 1, 0, d] = (2.0 ** -10 * torch.randn(nb, generator=g)).bfloat16()
    q, k = (q.double() * 2.0 ** qexp).bfloat16(), (k.double() * 2.0 ** kexp).bfloat16()
    for topk in (1, 8, 30):
        _check(q.to(gpu_device), k.to(gpu_device), block, topk)


@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("dk", [8, 16, 64])
@pytest.mark.parametrize("nb", [40, 100, 200, 400, 600, 1500])
def test_values_that_two_bf16_hold_worst(gpu_device, nb, dk, heads):
    """Every dim of a mean 2^-17 under or over 1 + 2^-8, half way between two bf16: the lower parts are +-2^-8.  A query of 1 + 3 2^-8
    (half way, lower part -2^-8) differs by 2^-16 between the two sorts of blocks; the product of the lower parts adds 2^-16 to
    the one and takes it from the other, and what two parts leave of the mean does half as much."""
    block, nq, over = 128, 64, 20
    k = torch.full((1, nb * block, 1, dk), 1 + 2.0 ** -8)
    sign = torch.full((nb,), -1.0)
    sign[torch.randperm(nb, generator=torch.Generator().manual_seed(dk + nb))[:over]] = 1.0
    k[0, torch.arange(nb) * block, 0] += (sign * 2.0 ** -10)[:, None]
    q = torch.full((1, nq, heads, dk), 1 + 3 * 2.0 ** -8 if heads == 1 else 2.0 ** -8)
    if heads == 2:
        q[:, :, 0] = 1 + 2.0 ** -7
    q, k = q.half(), k.half()
    assert bool((k.float().view(nb, block, dk).mean(1) == (1 + 2.0 ** -8 + sign * 2.0 ** -17)[:, None]).all())
    for topk in (over - 4, over, over + 3):
        _check(q.to(gpu_device), k.to(gpu_device), block, topk)
