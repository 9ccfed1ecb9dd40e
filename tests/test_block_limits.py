"""CPU: sizes of the block-sparse attention whose launches would have 2^32 threads and more are refused with the size of their workspace."""
import pytest

from tests.test_block_attention import BASE, _run


@pytest.mark.parametrize("change", [dict(batch=1 << 20, heads=8, kv_heads=8, nq=128), dict(batch=1 << 22, heads=8, kv_heads=8, nq=4),
                                    dict(batch=1 << 10, heads=2, kv_heads=2, nq=1 << 19, nk=64 * 600), dict(batch=1 << 24, heads=2, kv_heads=2, nq=1, nk=64 * 40)])
def test_select(change):
    from yololite_amd import _lib

    L, a = _lib.lib(), BASE | change
    assert _run("select", change | dict(work_bytes=1 << 62)) == -3 and b"block_select" in L.yl_last_error()
    assert L.yl_block_select_workspace_bytes(*(a[x] for x in ("batch", "nq", "nk", "heads", "kv_heads", "dk", "block"))) == -1


@pytest.mark.parametrize("change", [dict(batch=1 << 20, heads=8, kv_heads=8, nq=128), dict(batch=1 << 22, heads=8, kv_heads=8, nq=4),
                                    dict(batch=1 << 20, heads=64, kv_heads=2, nq=9, topk=8, nk=640)])
def test_attention(change):
    from yololite_amd import _lib

    L, a = _lib.lib(), BASE | change
    assert _run("attention", change | dict(work_bytes=1 << 62)) == -3 and b"block_attention" in L.yl_last_error()
    assert L.yl_block_attention_workspace_bytes(*(a[x] for x in ("dtype", "batch", "nq", "nk", "heads", "kv_heads", "dk", "dv", "block", "topk"))) == -1


def test_map():
    from yololite_amd import _lib

    assert _lib.lib().yl_attention_scratch_bytes(1 << 12, 8, 1 << 15, 64, 8) == -1
    assert _lib.lib().yl_attention_scratch_bytes(8, 6, 1600, 64, 8) > 0


@pytest.mark.parametrize("sizes", [(1, 16384, 16384, 8, 2, 64, 64), (64, 6400, 6400, 6, 6, 32, 64), (1 << 10, 1, 65536, 8, 8, 64, 64), (1, 1 << 21, 262144, 32, 32, 128, 64)])
def test_sizes_that_have_a_workspace(sizes):
    from yololite_amd import _lib

    L = _lib.lib()
    batch, nq, nk, heads, kv, dk, block = sizes
    assert L.yl_block_select_workspace_bytes(*sizes) >= 0
    assert L.yl_block_attention_workspace_bytes(0, batch, nq, nk, heads, kv, dk, 64, block, 16) >= 0
