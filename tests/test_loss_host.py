"""The losses' bindings on the host (no GPU): struct layouts, constants, and every refusal before anything is launched."""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from common.testing import raises
from dense_reader import _lib
from lm_head_topk import head_loss
from moe import balance

ROOT = Path(__file__).resolve().parents[1]


def test_loss_structs_match_c(tmp_path):
    src = tmp_path / "layout.c"
    fields = [("dr_head_loss", _lib.HeadLoss), ("dr_balance", _lib.Balance)]
    prints = "".join(f'printf("%zu\\n", sizeof({c}));' + "".join(
        f'printf("%zu\\n", offsetof({c}, {name}));' for name, _ in t._fields_) for c, t in fields)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "lm_head.h"\n#include "moe.h"\n'
                   f"int main(void){{{prints}return 0;}}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for _, t in fields for v in [ctypes.sizeof(t)] + [getattr(t, name).offset for name, _ in t._fields_]]
    assert got == want


def test_loss_constants_match_the_headers():
    text = "".join((ROOT / "include" / h).read_text() for h in ("lm_head.h", "moe.h"))
    defs = {k: int(v) for k, v in re.findall(r"^#define\s+(DR_\w+)\s+(\d+)\b", text, re.M)}
    for name in ("DR_LOSS_FORWARD", "DR_LOSS_BACKWARD", "DR_LOSS_MAX_K", "DR_BALANCE_LOSS", "DR_BALANCE_GRAD"):
        assert defs[name] == getattr(_lib, name), name


def _head(**kw):
    """A dr_head_loss whose pointers are never read (every call here is refused, or only asks for the workspace)."""
    A = _lib.HeadLoss()
    for f in ("x", "head", "ids", "loss", "lse", "logits", "dx", "dhead", "workspace"):
        setattr(A, f, 4096)
    A.rows, A.dim, A.ldx, A.ld_head, A.vocab, A.valid = 100, 64, 64, 64, 1000, 1000
    A.ld_ids = A.k = 1
    A.temperature, A.ld_dx, A.ld_dhead, A.workspace_bytes = 1.0, 64, 64, 1 << 40
    for name, v in kw.items():
        setattr(A, name, v)
    return A


@pytest.mark.parametrize("bad", [
    dict(rows=0), dict(rows=-1), dict(dim=0), dict(dim=60), dict(ldx=56), dict(ldx=68), dict(ld_head=56), dict(vocab=0),
    dict(valid=0), dict(valid=1001), dict(k=0), dict(k=2), dict(k=65, vals=4096, ld_ids=65, ld_vals=65),
    dict(vals=4096, k=4, ld_ids=3, ld_vals=4), dict(vals=4096, k=4, ld_ids=4, ld_vals=3), dict(temperature=0.0),
    dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=2.0),
])
def test_head_loss_refuses_sizes(bad):
    A = _head(**bad)
    for what in (1, 2, 3):
        assert _lib.lib().dr_head_loss_workspace_bytes(ctypes.byref(A), what) == -1, bad
        assert _lib.lib().dr_head_loss_run(ctypes.byref(A), what) == _lib.DR_EINVAL, bad


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(x=4104), dict(head=None), dict(head=4104), dict(ids=None), dict(ids=4098), dict(loss=None),
    dict(lse=None), dict(logits=None), dict(workspace=None), dict(workspace=4100), dict(workspace_bytes=100), dict(dx=4100),
    dict(ld_dx=60), dict(ld_dx=66), dict(dhead=4100), dict(ld_dhead=60),
])
def test_head_loss_refuses_pointers(bad):
    assert _lib.lib().dr_head_loss_run(ctypes.byref(_head(**bad)), 3) == _lib.DR_EINVAL, bad


def test_head_loss_refuses_what_it_does_not_know():
    for what in (0, 4, -1):
        assert _lib.lib().dr_head_loss_run(ctypes.byref(_head()), what) == _lib.DR_EINVAL
    assert _lib.lib().dr_head_loss_run(None, 1) == _lib.DR_EINVAL
    assert _lib.lib().dr_head_loss_workspace_bytes(None, 1) == -1
    assert _lib.lib().dr_head_loss_workspace_bytes(ctypes.byref(_head()), 1) > 0


@pytest.mark.parametrize("t", [2.0**-21, 1e-39, 1e-50])
def test_head_loss_refuses_temperatures_without_an_inverse(t):
    A = _head(vals=4096, k=4, ld_ids=4, ld_vals=4, temperature=t)
    for what in (1, 2, 3):
        assert _lib.lib().dr_head_loss_run(ctypes.byref(A), what) == _lib.DR_EINVAL, t
    A.temperature = 2.0**-20
    assert _lib.lib().dr_head_loss_workspace_bytes(ctypes.byref(A), 3) > 0


def test_head_loss_refuses_more_tiles_than_a_launch_holds():
    """A launch holds fewer than 2^32 lanes: more rows and tokens than that are refused before any of its kernels runs."""
    ask = _lib.lib().dr_head_loss_workspace_bytes
    for rows, valid, ok in ((1 << 20, 1 << 18, True), (1 << 19, 1 << 23, False), (1 << 20, 1 << 20, False), (64, 1 << 28, True)):
        A = _head(rows=rows, dim=8, ldx=8, ld_head=8, ld_dx=8, ld_dhead=8, vocab=valid, valid=valid, workspace_bytes=1 << 62)
        assert (ask(ctypes.byref(A), 1) > 0) == ok, (rows, valid)
        if not ok:
            assert _lib.lib().dr_head_loss_run(ctypes.byref(A), 1) == _lib.DR_EINVAL, (rows, valid)


def test_head_loss_workspace_keeps_no_logits():
    """The backward's workspace holds a piece of the logits' gradient, never all of it: with eight times the vocabulary it
    stays the same; nor does the forward's hold the logits."""
    big = dict(rows=65536, dim=4096, ldx=4096, ld_head=4096, ld_dx=4096, ld_dhead=4096)
    sizes = [_lib.lib().dr_head_loss_workspace_bytes(ctypes.byref(_head(**big, vocab=v, valid=v)), 2)
             for v in (128256, 8 * 128256)]
    assert sizes[1] < 1.2 * sizes[0] and sizes[0] < 65536 * 128256 * 2 / 4, sizes
    fwd = _lib.lib().dr_head_loss_workspace_bytes(ctypes.byref(_head(**big, vocab=128256, valid=128256)), 1)
    assert fwd < 65536 * 128256 * 4 / 16, fwd
    both = [_lib.lib().dr_head_loss_workspace_bytes(ctypes.byref(_head(**big, vocab=v, valid=v)), 3) for v in (8192, 128256)]
    kept = 65536 * 8192 * 4  # (one piece: 2 GiB)
    assert kept < both[0] < 2 * kept and both[1] < sizes[0] + 1.1 * fwd, both


def _balance(**kw):
    A = _lib.Balance()
    for f in ("logits", "ids", "loss", "counts", "dlogits", "workspace"):
        setattr(A, f, 4096)
    A.batch, A.rows, A.experts, A.width, A.ld_logits, A.ld_dlogits, A.ld_ids, A.k = 2, 100, 32, 32, 32, 32, 4, 4
    A.workspace_bytes = 1 << 40
    for name, v in kw.items():
        setattr(A, name, v)
    return A


@pytest.mark.parametrize("bad", [
    dict(batch=0), dict(batch=65537), dict(rows=0), dict(rows=1 << 30), dict(experts=0), dict(experts=1025, width=1025,
    ld_logits=1025, ld_dlogits=1025), dict(experts=33), dict(width=33), dict(k=0), dict(k=5), dict(k=17, ld_ids=17),
    dict(kind=2), dict(kind=-1), dict(batch=1, rows=1 << 27, k=16, ld_ids=16),
])
def test_balance_refuses_sizes(bad):
    A = _balance(**bad)
    for what in (1, 2):
        assert _lib.lib().dr_moe_balance_workspace_bytes(ctypes.byref(A), what) == -1, bad
        assert _lib.lib().dr_moe_balance(ctypes.byref(A), what) == _lib.DR_EINVAL, bad


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(logits=4098), dict(ids=None), dict(ids=4097), dict(ids32=1, ids=4098), dict(loss=None),
    dict(counts=None), dict(dlogits=None), dict(ld_dlogits=31), dict(workspace=None), dict(workspace=4100),
    dict(workspace_bytes=16),
])
def test_balance_refuses_pointers(bad):
    assert _lib.lib().dr_moe_balance(ctypes.byref(_balance(**bad)), 2) == _lib.DR_EINVAL, bad


def test_balance_refuses_what_it_does_not_know():
    for what in (0, 4, -1):
        assert _lib.lib().dr_moe_balance(ctypes.byref(_balance()), what) == _lib.DR_EINVAL
    assert _lib.lib().dr_moe_balance(None, 1) == _lib.DR_EINVAL


def test_host_tensors_are_refused():
    """There is no path on the host: tensors that are not on the GPU are refused before anything else happens."""
    x, h = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(128, 64, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64)
    for fn in (head_loss.token_loss, head_loss.token_loss_grads):
        raises(f"{fn.__name__} on the host", AssertionError, lambda: fn(x, h, t))
    v, i = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)
    for fn in (head_loss.distill_loss, head_loss.distill_loss_grads):
        raises(f"{fn.__name__} on the host", AssertionError, lambda: fn(x, h, v, i))
    lg, ids = torch.zeros(4, 32), torch.zeros(4, 2, dtype=torch.int16)
    for fn in (balance.balance_loss, balance.balance_loss_grads):
        raises(f"{fn.__name__} on the host", AssertionError, lambda: fn(lg, ids, 2))
