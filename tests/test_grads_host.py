"""The gradients' C entries on the host (no GPU): the struct's layout, and refusals before anything is launched."""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from common import grads
from common.testing import raises
from dense_reader import _lib

ROOT = Path(__file__).resolve().parents[1]


def test_struct_matches_c(tmp_path):
    names = [n for n, _ in _lib.Grads._fields_]
    prints = "".join(f'printf("%zu\\n", offsetof(dr_grads, {n.rstrip("_")}));' for n in names)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "grads.h"\n'
                   f'int main(void){{printf("%zu\\n", sizeof(dr_grads));{prints}return 0;}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.Grads)] + [getattr(_lib.Grads, n).offset for n in names]
    text = (ROOT / "include" / "grads.h").read_text()
    for name in ("DR_GRADS_LIST", "DR_GRADS_LIST_BYTES"):
        assert int(re.search(rf"^#define {name} (\d+)", text, re.M).group(1)) == getattr(_lib, name)
    types = {k: int(v) for k, v in re.findall(r"^#define DR_GRADS_(F32|BF16|F16) (\d)", text, re.M)}
    assert types == {"F32": grads.TYPES[torch.float32], "BF16": grads.TYPES[torch.bfloat16], "F16": grads.TYPES[torch.float16]}


def call(ins, sizes, types, outs=None, out_types=None, **kw):
    """A dr_grads whose pointers are never read on a device."""
    n, held = len(sizes), []

    def at(kind, values):
        held.append((kind * n)(*values))
        return ctypes.addressof(held[-1])

    A = _lib.Grads(n, at(ctypes.c_void_p, ins), at(ctypes.c_int64, sizes), at(ctypes.c_int32, types))
    if outs is not None:
        A.out, A.out_types = at(ctypes.c_void_p, outs), at(ctypes.c_int32, types if out_types is None else out_types)
    A.held = held  # (as long as the call's struct)
    A.max_norm, A.norm, A.workspace, A.workspace_bytes = 1.0, 4096, 4096, 1 << 40
    for name, v in kw.items():
        setattr(A, name, v)
    return ctypes.byref(A)


@pytest.mark.parametrize("ins, sizes, types", [
    ([4096], [-1], [0]), ([4096], [(1 << 40) + 1], [0]), ([4096, 4096], [1 << 40, 1], [0, 0]), ([4096], [8], [3]),
    ([4096], [8], [-1]), ([None], [8], [0]), ([4098], [8], [0]), ([4097], [8], [1]), ([4097], [8], [2]),
])
def test_refused_lists(ins, sizes, types):
    L = _lib.lib()
    assert L.dr_grads_workspace_bytes(call(ins, sizes, types)) == -1
    assert L.dr_grads_norm(call(ins, sizes, types)) == _lib.DR_EINVAL
    assert L.dr_grads_clip(call(ins, sizes, types, ins)) == _lib.DR_EINVAL


@pytest.mark.parametrize("bad", [dict(norm=None), dict(norm=4098), dict(workspace=None), dict(workspace=4100),
                                 dict(workspace_bytes=0), dict(workspace_bytes=-8), dict(max_norm=-1.0), dict(max_norm=float("nan")),
                                 dict(count=-1), dict(count=(1 << 20) + 1)])
def test_refused_calls(bad):
    L = _lib.lib()
    if "max_norm" not in bad:
        assert L.dr_grads_norm(call([4096], [8], [0], **bad)) == _lib.DR_EINVAL
    assert L.dr_grads_clip(call([4096], [8], [0], [4096], **bad)) == _lib.DR_EINVAL


@pytest.mark.parametrize("ins, sizes, types, outs, out_types", [
    ([4096, 4096], [8, 8], [0, 0], [4096, 4096], [0, 0]),  # one tensor twice
    ([4096, 4096], [8, 8], [0, 0], [8192, 8192 + 28], [0, 0]),  # outs that share a value
    ([4096, 8192], [8, 8], [0, 0], [8192, 4096], [0, 0]),  # each other's
    ([4096, 8192], [8, 8], [0, 0], [8192 + 4, 16384], [0, 0]),  # over another's in
    ([4096, 8192], [8, 8], [0, 0], [16384, 4096 + 31 - 3], [0, 0]),
    ([4096], [8], [0], [4100], [0]),  # over its own, shifted
    ([4096], [8], [1], [4096], [0]),  # over its own, wider
    ([4096], [8], [0], [4096 + 16], [1]),  # within its own
    ([4096], [8], [0], [4096 - 4], [1]),
    ([4096, 4096 + 8, 20000], [1000, 1, 2], [1, 1, 1], [30000, 40000, 4096 + 1998], [1, 1, 1]),  # into an in that began long before
    ([4096], [8], [0], [None], [0]), ([4096], [8], [0], [8194], [0]), ([4096], [8], [0], [8192], [3]),
])
def test_refused_memory(ins, sizes, types, outs, out_types):
    assert _lib.lib().dr_grads_clip(call(ins, sizes, types, outs, out_types)) == _lib.DR_EINVAL


@pytest.mark.parametrize("given", [0, 1])
def test_norm_within_the_outs(given):
    L = _lib.lib()
    assert L.dr_grads_clip(call([8192], [8], [0], [8192], norm=8192 + 28, given=given)) == _lib.DR_EINVAL
    assert L.dr_grads_clip(call([8192], [8], [0], [16384], norm=16384, given=given)) == _lib.DR_EINVAL


def test_workspaces():
    L = _lib.lib()
    assert L.dr_grads_workspace_bytes(call([], [], [])) == 0
    assert L.dr_grads_workspace_bytes(call([4096, None, 8192], [8192, 0, 8193], [0, 0, 1])) == 8 * 3
    assert L.dr_grads_workspace_bytes(call([4096], [1 << 30], [1])) == 8 * 2048
    assert L.dr_grads_workspace_bytes(call([4096] * 300, [1] * 300, [1] * 300)) == 8 * 300


def test_null():
    L = _lib.lib()
    assert L.dr_grads_workspace_bytes(None) == -1
    assert L.dr_grads_norm(None) == L.dr_grads_clip(None) == _lib.DR_EINVAL
    A = _lib.Grads(count=1, max_norm=1.0, norm=4096)
    assert L.dr_grads_norm(ctypes.byref(A)) == _lib.DR_EINVAL
    assert L.dr_grads_clip(call([4096], [8], [0])) == _lib.DR_EINVAL  # (no outs)


def test_python_refuses_host_tensors():
    t = torch.zeros(4)
    for fn in (lambda: grads.global_norm([t]), lambda: grads.clip_([t], 1.0), lambda: grads.clipped([t], 1.0)):
        raises("host", AssertionError, fn)
    raises("nothing", ValueError, lambda: grads.global_norm([]))
