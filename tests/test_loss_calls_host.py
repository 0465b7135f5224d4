"""The losses' C entries on the host (no GPU): refusals before anything is launched, workspaces, and plans."""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from dense_reader import _lib

ROOT = Path(__file__).resolve().parents[1]


def test_backward_constant_matches_the_header():
    text = (ROOT / "include" / "moe.h").read_text()
    assert int(re.search(r"^#define DR_BALANCE_BACKWARD (\d+)", text, re.M).group(1)) == _lib.DR_BALANCE_BACKWARD


def head(**kw):
    """A dr_head_loss whose pointers are never read."""
    A = _lib.HeadLoss(rows=100, dim=64, ldx=64, ld_head=64, vocab=1000, valid=1000, ld_ids=1, k=1, temperature=1.0, ld_dx=64,
                      ld_dhead=64, workspace_bytes=1 << 62)
    for f in ("x", "head", "ids", "loss", "lse", "logits", "dx", "dhead", "workspace"):
        setattr(A, f, 4096)
    for name, v in kw.items():
        setattr(A, name, v)
    return A


def test_farthest_rows():
    """The limit on a row's distance is the header's, and holds."""
    text = (ROOT / "include" / "lm_head.h").read_text()
    assert 1 << int(re.search(r"^#define DR_LOSS_MAX_LD \(1 << (\d+)\)", text, re.M).group(1)) == _lib.DR_LOSS_MAX_LD
    for name in ("ldx", "ld_head"):
        for ld, ok in ((_lib.DR_LOSS_MAX_LD, True), (_lib.DR_LOSS_MAX_LD + 8, False)):
            assert (_lib.lib().dr_head_loss_workspace_bytes(ctypes.byref(head(**{name: ld})), 3) > 0) == ok


@pytest.mark.parametrize("rows, vals", [(8, None), (100, None), (8192, None), (8192, 4096)])
def test_no_gradient_asked_for(rows, vals):
    """Neither dx nor dhead: the workspace is the forward's alone."""
    both, ask = dict(rows=rows, vocab=128256, valid=128256, vals=vals, ld_vals=1), _lib.lib().dr_head_loss_workspace_bytes
    forward = ask(ctypes.byref(head(**both)), _lib.DR_LOSS_FORWARD)
    neither = head(**both, dx=None, dhead=None)
    assert ask(ctypes.byref(neither), _lib.DR_LOSS_FORWARD | _lib.DR_LOSS_BACKWARD) == forward > 0
    assert _lib.lib().dr_head_loss_run(ctypes.byref(neither), _lib.DR_LOSS_BACKWARD) == _lib.DR_OK  # (nothing to do)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(logits=4098), dict(kept=None), dict(kept=4098), dict(dlogits=None), dict(dlogits=4098),
    dict(ld_dlogits=31), dict(rows=0), dict(experts=33), dict(kind=2),
])
def test_balance_backward_refuses(bad):
    A = _lib.Balance(logits=4096, kept=4096, dlogits=4096, batch=2, rows=100, experts=32, width=32, ld_logits=32, ld_dlogits=32,
                     ld_ids=1, k=1)
    assert _lib.lib().dr_moe_balance_workspace_bytes(ctypes.byref(A), _lib.DR_BALANCE_BACKWARD) == 0
    for name, v in bad.items():
        setattr(A, name, v)
    assert _lib.lib().dr_moe_balance(ctypes.byref(A), _lib.DR_BALANCE_BACKWARD) == _lib.DR_EINVAL, bad


def test_balance_refuses_a_misaligned_kept():
    A = _lib.Balance(logits=4096, ids=4096, loss=4096, counts=4096, kept=4098, batch=2, rows=10, experts=32, width=32,
                     ld_logits=32, ld_ids=4, k=4)
    assert _lib.lib().dr_moe_balance(ctypes.byref(A), _lib.DR_BALANCE_LOSS) == _lib.DR_EINVAL


# Calls whose products take the large tiles, and what of their plan they are there for: (rows, vocabulary, of it valid, dim,
# teacher's entries or 0, both directions at once), {field of dr_head_loss_info: value}. No row count or size of one is a tile's
# multiple but where it says.
T256, T128 = (256, 256, 1), (128, 128, 1)
LARGE = [
    ((2100, 5003, 5000, 2056, 0, True), dict(z=T256, kept=1, dhead=T256, dhead_stages=4, dx=T256, dx_splits=3, pieces=1)),
    ((2100, 5003, 5000, 2056, 0, False), dict(dz=T256, kept=0, dhead=T256, dhead_stages=4, dx=T256, dx_splits=3, pieces=1)),
    ((2500, 5003, 4999, 4096, 16, True), dict(z=T256, kept=1, dhead=T128, dhead_stages=4, dx=T256, dx_splits=1, pieces=1)),
    ((2500, 5003, 4999, 4096, 16, False), dict(dz=T256, kept=0, dhead=T128, dhead_stages=4, dx=T256, dx_splits=1, pieces=1)),
    ((1600, 6001, 5999, 2056, 5, True), dict(z=T256, kept=1, dhead=T256, dhead_stages=4, dx=T128, dx_splits=2, pieces=1)),
    ((130, 9001, 8999, 1000, 0, True), dict(kept=1, dhead=T256, dhead_stages=4, dx=(64, 64, 2), dx_splits=5, pieces=1)),
    ((520, 9001, 8999, 2056, 0, True), dict(z=T128, kept=1, dhead=T128, dhead_stages=1, dx=T128, dx_splits=6, pieces=1)),
    ((8200, 66000, 65990, 2056, 0, True), dict(z=T256, dz=T256, kept=0, dhead=T256, dx=T256, dx_splits=1, pieces=2)),
    ((8200, 66000, 65990, 2056, 4, True), dict(z=T256, dz=T256, kept=0, dhead=T256, dx=T256, dx_splits=1, pieces=2)),
]


@pytest.mark.parametrize("call, want", LARGE)
def test_plans_of_large_calls(call, want):
    """The kernels that the GPU tests of these calls are there for are the ones they take."""
    n, v, valid, d, k, both = call
    A = head(rows=n, vocab=v, valid=valid, dim=d, ldx=d, ld_head=d, ld_dx=d, ld_dhead=d, k=max(k, 1), ld_ids=max(k, 1),
             vals=4096 if k else None, ld_vals=k)
    info = _lib.head_loss_info(A, 3 if both else _lib.DR_LOSS_BACKWARD)
    assert {f: info[f] for f in want} == want


def test_plan_refuses_what_the_call_does():
    info = _lib.HeadLossInfo()
    for bad in (dict(rows=0), dict(temperature=0.0), dict(ldx=56)):
        assert _lib.lib().dr_head_loss_plan(ctypes.byref(head(**bad)), 3, ctypes.byref(info)) == _lib.DR_EINVAL, bad
    assert _lib.lib().dr_head_loss_plan(None, 3, ctypes.byref(info)) == _lib.DR_EINVAL
    assert _lib.lib().dr_head_loss_plan(ctypes.byref(head()), 3, None) == _lib.DR_EINVAL
    forward = _lib.head_loss_info(head(dx=None, dhead=None), 3)
    assert forward["pieces"] == 0 and forward["dhead"] == forward["dx"] == (0, 0, 0) and forward["z"] != (0, 0, 0)


def test_info_struct_matches_c(tmp_path):
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    names = [name for name, _ in _lib.HeadLossInfo._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "lm_head.h"\nint main(void){'
                   'printf("%zu\\n", sizeof(dr_head_loss_info));'
                   + "".join(f'printf("%zu\\n", offsetof(dr_head_loss_info, {n}));' for n in names) + "return 0;}\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.HeadLossInfo)] + [getattr(_lib.HeadLossInfo, n).offset for n in names]
