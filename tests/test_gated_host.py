"""The gated block's C entries on the host (no GPU): struct layouts, refusals before anything is launched, workspaces, plans, and
the emitted code of its kernel's K loops."""

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from dense_reader import _lib
from test_loss_barriers import barriers_left
from test_loss_isa import extra_waits, k_loops

ROOT = Path(__file__).resolve().parents[1]
FORWARD, BACKWARD = _lib.DR_GATED_FORWARD, _lib.DR_GATED_BACKWARD


def test_structs_match_c(tmp_path):
    fields = [("dr_gated", _lib.Gated), ("dr_gated_info", _lib.GatedInfo)]
    prints = "".join(f'printf("%zu\\n", sizeof({c}));' + "".join(
        f'printf("%zu\\n", offsetof({c}, {name}));' for name, _ in t._fields_) for c, t in fields)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "gated.h"\nint main(void){{{prints}return 0;}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [v for _, t in fields for v in [ctypes.sizeof(t)] + [getattr(t, name).offset for name, _ in t._fields_]]


def test_constants_match_the_header():
    text = (ROOT / "include" / "gated.h").read_text()
    for name in ("DR_GATED_FORWARD", "DR_GATED_BACKWARD"):
        assert int(re.search(rf"^#define {name} (\d+)", text, re.M).group(1)) == getattr(_lib, name)
    assert 1 << int(re.search(r"^#define DR_GATED_MAX_LD \(1 << (\d+)\)", text, re.M).group(1)) == _lib.DR_GATED_MAX_LD


def call(rows=100, dim=64, width=96, **kw):
    """A dr_gated whose pointers are never read."""
    A = _lib.Gated(rows=rows, dim=dim, width=width, ldx=dim, ld_gate=dim, ld_up=dim, ld_h=width, ld_dh=width, ld_dx=dim,
                   ld_dgate=dim, ld_dup=dim, workspace_bytes=1 << 62)
    for f in ("x", "gate", "up", "h", "kept", "dh", "dx", "dgate", "dup", "workspace"):
        setattr(A, f, 4096)
    for name, v in kw.items():
        setattr(A, name, v)
    return ctypes.byref(A)


@pytest.mark.parametrize("bad", [
    dict(rows=0), dict(rows=-1), dict(rows=(1 << 20) + 1), dict(dim=0), dict(dim=60), dict(dim=(1 << 17) + 8), dict(width=0),
    dict(width=90), dict(width=(1 << 20) + 8), dict(act=2), dict(act=-1), dict(ldx=56), dict(ldx=68), dict(ld_gate=56),
    dict(ld_up=66), dict(ldx=(1 << 21) + 8), dict(ld_gate=(1 << 21) + 8), dict(ld_up=(1 << 21) + 8),
    dict(rows=1 << 20, width=1 << 20),
])
def test_refused_sizes(bad):
    L = _lib.lib()
    for what in (FORWARD, BACKWARD):
        assert L.dr_gated_workspace_bytes(call(**bad), what) == -1
        assert L.dr_gated_run(call(**bad), what) == _lib.DR_EINVAL
        info = _lib.GatedInfo()
        assert L.dr_gated_plan(call(**bad), what, ctypes.byref(info)) == _lib.DR_EINVAL
    assert L.dr_gated_kept_bytes(call(**bad)) == -1


@pytest.mark.parametrize("what, bad", [(w, {p: v}) for w, names in (
    (FORWARD, ("x", "gate", "up", "h")), (BACKWARD, ("x", "gate", "up", "dh", "workspace"))) for p in names for v in (None, 4104)]
    + [(FORWARD, dict(kept=4104)), (FORWARD, dict(ld_h=88)), (FORWARD, dict(ld_h=97)), (BACKWARD, dict(ld_dh=88)),
       (BACKWARD, dict(ld_dx=56)), (BACKWARD, dict(ld_dgate=68)), (BACKWARD, dict(ld_dup=0)), (BACKWARD, dict(dx=4104)),
       (BACKWARD, dict(dgate=4104)), (BACKWARD, dict(dup=4104)), (BACKWARD, dict(kept=4104)), (BACKWARD, dict(workspace=4096 + 128)),
       (BACKWARD, dict(workspace_bytes=0)), (0, {}), (3, {}), (4, {})])
def test_refused_calls(what, bad):
    assert _lib.lib().dr_gated_run(call(**bad), what) == _lib.DR_EINVAL


def test_null():
    L = _lib.lib()
    assert L.dr_gated_run(None, FORWARD) == _lib.DR_EINVAL and L.dr_gated_kept_bytes(None) == -1
    assert L.dr_gated_workspace_bytes(None, BACKWARD) == -1 and L.dr_gated_plan(call(), FORWARD, None) == _lib.DR_EINVAL


def test_workspaces():
    L = _lib.lib()
    assert L.dr_gated_kept_bytes(call(100, 64, 264)) == 3 * 2 * 100 * 512
    assert L.dr_gated_workspace_bytes(call(), FORWARD) == 0
    neither = call(dx=None, dgate=None, dup=None, workspace=None, workspace_bytes=0)
    assert L.dr_gated_workspace_bytes(neither, BACKWARD) == 0
    assert L.dr_gated_run(neither, BACKWARD) == _lib.DR_OK  # (nothing to do)
    need = L.dr_gated_workspace_bytes(call(dx=None), BACKWARD)
    assert need == 2 * 100 * 512  # dg and du
    assert L.dr_gated_run(call(workspace_bytes=need - 1, dx=None), BACKWARD) == _lib.DR_EINVAL


# Calls whose products take each of the tiles, and what of their plan they are there for: (rows, dim, width), {field of dr_gated_info: value};
# the GPU's tests run them
T256, T192, T128 = (256, 256, 1), (192, 256, 1), (128, 128, 1)
TILES = [
    ((1, 64, 64), dict(act=(32, 32, 4), dweight=T128, dweight_stages=1, dx=(64, 64, 2), dx_splits=1)),
    ((2, 64, 4128), dict(act=(64, 32, 4), dx_splits=32)),
    ((1, 64, 8256), dict(act=(64, 32, 1))),
    ((39, 72, 64), dict(act=(32, 64, 4))),
    ((40, 64, 4408), dict(act=(64, 64, 2))),
    ((40, 64, 8368), dict(act=(128, 64, 1))),
    ((77, 64, 72), dict(act=(64, 128, 1), dx=T128, dx_splits=1)),
    ((134, 144, 2584), dict(act=(64, 64, 2))),
    ((419, 64, 4104), dict(act=T128)),
    ((279, 64, 11024), dict(act=T192)),
    ((341, 64, 13240), dict(act=T256)),
    ((2, 560, 13248), dict(dweight=T128, dweight_stages=1)),
    ((1093, 72, 72), dict(dweight=T128, dweight_stages=4)),
    ((69, 280, 11016), dict(dweight=T192, dweight_stages=2)),
    ((70, 400, 12128), dict(dweight=T256, dweight_stages=4)),
    ((3, 3264, 7808), dict(dx=(256, 64, 1), dx_splits=19)),
    ((7223, 1128, 64), dict(dx=T256, dx_splits=1)),
    ((3739, 136, 6416), dict(dx=T256)),
]


@pytest.mark.parametrize("sizes, want", TILES, ids=[str(s) for s, _ in TILES])
def test_plans(sizes, want):
    A = call(*sizes)._obj
    info = {**_lib.gated_info(A, BACKWARD), "act": _lib.gated_info(A, FORWARD)["act"]}
    assert {k: info[k] for k in want} == want, info
    A.kept = None
    assert _lib.gated_info(A, BACKWARD)["act"] == info["act"]
    if want.get("dx") == T256 and "dx_splits" not in want:
        assert info["dx_splits"] > 1


def _asm(tmp_path):
    import __graft_entry__ as G

    hipcc = G.HIPCC if Path(G.HIPCC).exists() else shutil.which("hipcc")
    if hipcc is None:
        pytest.skip("no hipcc")
    src = next(s for s in G.SOURCES if s.name == "gated.hip")
    flags = [f for f in G.FLAGS if f not in ("-shared", "-fPIC")]
    dst = tmp_path / "gated.s"
    subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", str(src), "-o", str(dst)], check=True, capture_output=True)
    return dst.read_text()


def test_emitted_code(tmp_path):
    """In every K loop the waits for loads from memory are those asked for before each barrier, and no more; behind the sums every
    wavefront meets the same barriers; no kernel spills."""
    asm = _asm(tmp_path)
    loops = asm.replace("gt_gemm", "hl_gemm")
    # (a workgroup of one wavefront has no barriers left, but as many waits as its loop has stages: five)
    alone = {name for name, _ in k_loops(loops) if re.search(r"ILi64ELi32ELi1ELi1ELi1ELi5E", name)}
    assert len(k_loops(loops)) >= 15 and set(extra_waits(loops)) == alone
    for name, part in k_loops(loops):
        if name in alone:
            assert sum(s.startswith("s_waitcnt") and "vmcnt" in s for s in part) <= 5
    found = dict(re.findall(r"^(_Z\S*gt_gemm\S+):(.*?)^\.Lfunc_end", asm, re.M | re.S))
    ways = {name: barriers_left(body) for name, body in found.items()}
    # (EPI_DXJ: two barriers more where a launch's sums are split, all of its workgroups alike)
    joined = [w for name, w in ways.items() if re.search(r"ELi6ELb0E", name)]
    assert joined and all(len(w) == 2 and max(w) == min(w) + 2 for w in joined), joined
    ways = {name: w for name, w in ways.items() if w not in joined}
    assert len(found) >= 15 and all(len(w) == 1 for w in ways.values()), {n: w for n, w in ways.items() if len(w) != 1}
    assert set(re.findall(r"\.private_segment_fixed_size: (\d+)", asm)) == {"0"}


@pytest.mark.parametrize("rows, dim, width", [(1, 64, 64), (32, 4096, 14336), (33, 2048, 8192), (64, 1024, 4352), (65, 1024, 4096), (128, 2880, 2880),
                                              (256, 512, 1408), (300, 4096, 14336)])
@pytest.mark.parametrize("what, kept", [(FORWARD, 4096), (FORWARD, None), (BACKWARD, None)])
def test_weights_past_the_caches(rows, dim, width, what, kept):
    """Only where one tile has all rows, so that no other reads the weights again."""
    info = _lib.gated_info(call(rows, dim, width, kept=kept)._obj, what)
    assert info["act_once"] == (rows <= 64) and (not info["act_once"] or rows <= info["act"][1])


def test_loads_past_the_caches(tmp_path):
    """The kernels of one column tile alone load anything past the caches: the weights (64 x 64 in both kinds: of many rows too)."""
    found = dict(re.findall(r"^(_Z\S*gt_gemm\S+):(.*?)^\.Lfunc_end", _asm(tmp_path), re.M | re.S))
    past = {name: bool(re.search(r"buffer_load_dwordx4 .* lds.* nt|buffer_load_dwordx4 .* nt .*lds", body)) for name, body in found.items()}
    assert past and all(p == name.split("EEEv")[0].endswith("Lb1") for name, p in past.items()), past
    assert {p for name, p in past.items() if "ILi64ELi64ELi1ELi2ELi2E" in name} == {False, True}


@pytest.mark.parametrize("rows, dim, width", [(1 << 20, 8, 16384), (1 << 20, 64, 65536), (1 << 18, 1 << 17, 64), (1 << 20, 4096, 14336)])
def test_sizes_past_small_tiles(rows, dim, width):
    """Sizes within the header's of which a launch could not hold the smaller tiles: they go by large ones."""
    L = _lib.lib()
    A = call(rows, dim, width)._obj
    assert L.dr_gated_kept_bytes(ctypes.byref(A)) == 3 * -(-width // 256) * rows * 512
    assert L.dr_gated_workspace_bytes(ctypes.byref(A), BACKWARD) >= 2 * -(-width // 256) * rows * 512
    info = {**_lib.gated_info(A, BACKWARD), "act": _lib.gated_info(A, FORWARD)["act"]}
    for (bm, bn, _), m, n in ((info["act"], 2 * width, rows), (info["dx"], dim, rows), (info["dweight"], dim, 2 * width)):
        assert -(-m // bm) * -(-n // bn) < 1 << 23
