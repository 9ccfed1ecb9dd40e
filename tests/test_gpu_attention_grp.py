"""GPU: a dense YL_OP_ATTENTION does not read yl_op.grp."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grp", [64, 7])
def test_dense_attention_does_not_read_grp(gpu_device, grp):
    from tests.hip_util import Mini
    from yololite_amd.nn.lower import OP_ATTENTION

    qkv = torch.randn(2, 2 * 128, 20, 20, generator=torch.Generator().manual_seed(1))
    got = []
    for more in ({}, dict(grp=grp)):
        m = Mini(2, gpu_device)
        xin, out = m.buf(20, 20, 2 * 128), m.buf(20, 20, 2 * 64)
        m.fill(xin, qkv)
        m.op(kind=OP_ATTENTION, name="attn", heads=2, key_dim=32, head_dim=64, scale=32 ** -0.5, inp=xin, out=out, **more)
        m.run()
        assert m.eng.op_kernel(0) == "attention"
        got.append(m.read(out))
    assert torch.equal(*got)
