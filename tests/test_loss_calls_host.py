"""The losses' C entries on the host (no GPU): refusals before anything is launched, workspaces, and plans."""

import ctypes
import re
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
