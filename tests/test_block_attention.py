"""CPU: refusals of the block-sparse attention entry points (argument checks come before any GPU work), the restatement on a small
case by hand, the struct against the compiled header."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from tests import block_ref

ROOT = Path(__file__).resolve().parent.parent


def test_restatement_by_hand():
    """Four keys in blocks of two; the query is closer to the second block's mean, whose second key is masked."""
    q = np.array([1.0, 0.0]).reshape(1, 1, 1, 2)
    k = np.array([[1.0, 0], [0, 1], [0.75, 5], [9, 9]]).reshape(1, 4, 1, 2)
    v = np.arange(4.0).reshape(1, 4, 1, 1)
    mask = np.array([[1, 1, 1, 0]])
    picked = block_ref.select(q, k, 2, 1, mask)
    assert picked.tolist() == [[[[1]]]]
    assert block_ref.attend(q, k, v, picked, 2, mask)[0].item() == 2.0
    assert block_ref.select(q, k, 2, 3).tolist() == [[[[0, 1, -1]]]]
    both = block_ref.attend(q, k, v, np.array([[[[1, 0, 1]]]]), 2, mask, scale=np.log(2.0))[0].item()
    assert abs(both - (1 * 1 + 2 ** 0.75 * 2) / (2 + 1 + 2 ** 0.75)) < 1e-12  # weights 2, 1, 2^0.75 of values 0, 1, 2
    assert block_ref.attend(q, k, v, picked, 2, mask * 0)[0].item() == 0.0


def test_heads_struct_matches_the_compiled_header(tmp_path):
    from yololite_amd import _lib

    src = tmp_path / "h.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "yl_amd.h"\nint main(void) { printf("%zu %zu %zu %zu %zu", '
                   'sizeof(yl_heads), offsetof(yl_heads, data), offsetof(yl_heads, batch), offsetof(yl_heads, token), offsetof(yl_heads, head)); }\n')
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "h")], check=True)
    got = subprocess.run([str(tmp_path / "h")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(_lib.Heads)] + [getattr(_lib.Heads, f).offset for f, _ in _lib.Heads._fields_]


def _heads(at=4096, batch=64, token=64, head=32):
    from yololite_amd import _lib

    return _lib.Heads(at, batch, token, head)


BASE = dict(dtype=0, batch=1, nq=4, nk=100, heads=4, kv_heads=2, dk=32, dv=64, block=64, topk=2, mask=None, mask_stride=0, picked=4096,
            work=8192, work_bytes=1 << 30, scale=1.0, q={}, k={}, v={}, out={})
REFUSED = [
    (dict(dtype=1), -1), (dict(dtype=4), -1), (dict(heads=3), -1), (dict(kv_heads=0), -1), (dict(nq=-1), -1), (dict(nk=-1), -1),
    (dict(batch=-2), -1), (dict(dk=36), -3), (dict(dk=136), -3), (dict(dk=0), -3), (dict(block=16), -3), (dict(block=96), -3),
    (dict(topk=0), -3), (dict(topk=65), -3), (dict(nk=64 * 4096 + 1), -3), (dict(batch=1 << 20, nq=1 << 20), -3), (dict(picked=None), -1),
    (dict(q=dict(at=4100)), -1), (dict(q=dict(at=None)), -1), (dict(q=dict(head=30)), -1), (dict(k=dict(token=-64)), -1), (dict(k=None), -1),
    (dict(k=dict(batch=20)), -1), (dict(mask=64, mask_stride=50, batch=2), -1)]


def _run(name, change):
    from yololite_amd import _lib

    a = BASE | change
    L = _lib.lib()
    ref = [ctypes.byref(_heads(**a[t])) if a[t] is not None else None for t in ("q", "k", "v", "out")]
    sizes = [a[x] for x in ("dtype", "batch", "nq", "nk", "heads", "kv_heads", "dk")]
    tail = [a["work"], a["work_bytes"], None]
    if name == "select":
        return L.yl_block_select(*ref[:2], *sizes, a["block"], a["topk"], a["mask"], a["mask_stride"], a["picked"], *tail)
    return L.yl_block_attention(*ref[:3], *sizes, a["dv"], a["block"], a["topk"], a["picked"], a["mask"], a["mask_stride"], a["scale"],
                                ref[3], *tail)


@pytest.mark.parametrize("name", ["select", "attention"])
@pytest.mark.parametrize("change, code", REFUSED)
def test_refusals(name, change, code):
    from yololite_amd import _lib

    assert _run(name, change) == code
    assert f"block_{name}".encode() in _lib.lib().yl_last_error()


@pytest.mark.parametrize("change, code", [(dict(dv=60), -3), (dict(dv=136), -3), (dict(dv=0), -3), (dict(v=None), -1), (dict(out=None), -1),
                                          (dict(v=dict(at=4104)), -1), (dict(out=dict(token=4)), -1)])
def test_attention_refusals(change, code):
    assert _run("attention", change) == code


def test_products_of_sizes_that_wrap_in_64_bits_are_refused():
    from yololite_amd import _lib

    L = _lib.lib()
    for name in ("select", "attention"):
        assert _run(name, dict(batch=1 << 22, heads=1 << 21, kv_heads=1 << 21, nq=1 << 21)) == -3
        assert _run(name, dict(batch=1 << 30, heads=1 << 30, kv_heads=1 << 30, nq=1, nk=64 * 4096)) == -3
    assert L.yl_block_attention_workspace_bytes(0, 1 << 22, 1 << 21, 100, 1 << 21, 1 << 21, 32, 64, 64, 2) == -1
    assert L.yl_attention_scratch_bytes(1 << 30, 1 << 30, 16, 64, 2) == -1


@pytest.mark.parametrize("out", [dict(token=0), dict(head=0), dict(batch=0)])
def test_broadcast_results_are_refused(out):
    assert _run("attention", dict(out=out, batch=2)) == -1


def test_workspace_refusals():
    from yololite_amd import _lib

    L = _lib.lib()
    need = L.yl_block_select_workspace_bytes(1, 4, 100, 4, 2, 32, 64)
    assert need > 0 and _run("select", dict(work_bytes=need - 1)) == -1 and _run("select", dict(work=None)) == -1
    assert _run("select", dict(work=8200)) == -1
    assert L.yl_block_select_workspace_bytes(1, 4, 100, 4, 3, 32, 64) == -1
    assert L.yl_block_attention_workspace_bytes(0, 1, 4, 100, 4, 2, 32, 62, 64, 2) == -1


def test_nothing_to_do_is_no_error():
    for name in ("select", "attention"):
        assert _run(name, dict(nq=0, q=None, k=None, picked=None, work=None, work_bytes=0)) == 0
        assert _run(name, dict(batch=0, q=None, k=None, picked=None, work=None, work_bytes=0)) == 0


def test_python_face_refuses_without_a_gpu_tensor():
    import yololite_amd as ya

    q = torch.zeros(1, 4, 2, 32, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU only"):
        ya.block_select(q, q)
    with pytest.raises(RuntimeError, match="GPU only"):
        ya.block_attention(q, q, q, torch.zeros(1, 2, 4, 1, dtype=torch.int32))


def test_lowering_takes_blocks_on_long_maps(monkeypatch):
    """YL_PSA_TOPK: the attention of maps with more blocks than it reads, with its scratch in the arena; nothing else changes."""
    from yololite_amd import _lib
    from yololite_amd.nn import arch
    from yololite_amd.nn.lower import OP_ATTENTION, OP_PSA, lower
    from yololite_amd.nn.synth import synth_state_dict

    specs, _ = arch.parse_model(arch.yolo11_dict("n"))
    sd = synth_state_dict("n", 0)
    before = lower(specs, sd, 8, 640, 640)
    monkeypatch.setenv("YL_PSA_TOPK", "7")  # a 20x20 map has seven blocks: all of them, so the dense form stays
    assert [o["kind"] for o in lower(specs, sd, 8, 640, 640).ops] == [o["kind"] for o in before.ops]
    monkeypatch.setenv("YL_PSA_TOPK", "3")
    prog = lower(specs, sd, 8, 640, 640)
    att = [o for o in prog.ops if o["kind"] == OP_ATTENTION]
    assert [(o["grp"], o["topk"]) for o in att] == [(64, 3)] and not [o for o in prog.ops if o["kind"] == OP_PSA]
    need = _lib.lib().yl_attention_scratch_bytes(8, 2, 400, 64, 3)
    assert need > 0 and att[0]["scratch"] % 256 == 0 and att[0]["scratch"] + need <= prog.ws_bytes
    assert _lib.lib().yl_attention_scratch_bytes(8, 2, 400, 48, 3) == -1 and _lib.lib().yl_attention_scratch_bytes(8, 2, 0, 64, 3) == -1
