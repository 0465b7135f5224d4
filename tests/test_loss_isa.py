"""The gfx950 code of the LM head's losses (CPU only): in every K loop of hl_gemm, the waits for loads from memory are those
that the source asks for before each barrier, and no more.

The loads go straight to LDS, some steps ahead of the sums that read them. The compiler has a read of LDS wait for every load
to LDS that it cannot tell apart from it, which it can only while it sees which array an address comes from: a longer chain of
address arithmetic, or an array reached through a capture, and each step waits for the loads of the next (dhead's product then
took 1.3 times as long, with the same results)."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest


def k_loops(asm):
    """[(function, instructions)] of the innermost loops of hl_gemm that hold matrix instructions and no other memory access
    than loads to LDS and reads of it (a branch back over code laid in between, an epilogue's, makes none)."""
    out = []
    for name, body in re.findall(r"^(_Z\S*hl_gemm\S+):(.*?)^\.Lfunc_end", asm, re.M | re.S):
        lines = [s.split(";")[0].strip() for s in body.split("\n")]
        at = {s[:-1]: i for i, s in enumerate(lines) if s.startswith(".LBB") and s.endswith(":")}
        loops = [(at[t], i) for i, s in enumerate(lines) if s.startswith(("s_branch", "s_cbranch"))
                 for t in [s.split()[1]] if at.get(t, i) < i]
        for b, e in loops:
            if any((b, e) != (b2, e2) and b <= b2 and e2 <= e for b2, e2 in loops):
                continue
            part = [s for s in lines[b:e] if s and not s.endswith(":")]
            if any(s.startswith("v_mfma") for s in part) and not any(s.startswith("global_") for s in part):
                out.append((name, part))
    return out


def extra_waits(asm):
    """[function] of the K loops with more waits for memory than barriers."""
    return [name for name, part in k_loops(asm)
            if sum(s.startswith("s_waitcnt") and "vmcnt" in s for s in part) > sum(s == "s_barrier" for s in part)]


_LOOP = """_Z7hl_gemmILi1EEvv:
.LBB0_1:
\ts_waitcnt vmcnt(0) lgkmcnt(0)
\ts_barrier
\tbuffer_load_dwordx4 v1, s[4:7], 0 offen lds
%s\tds_read_b128 v[4:7], v2
\ts_waitcnt lgkmcnt(0)
\tv_mfma_f32_32x32x16_bf16 a[0:15], v[4:7], v[4:7], a[0:15]
\ts_cbranch_scc1 .LBB0_1
.Lfunc_end0:
"""


def test_the_scan_finds_a_planted_wait():
    assert not extra_waits(_LOOP % "") and len(k_loops(_LOOP % "")) == 1
    assert extra_waits(_LOOP % "\ts_waitcnt vmcnt(0)\n")


def test_no_wait_beyond_the_barriers(tmp_path):
    import __graft_entry__ as G

    hipcc = G.HIPCC if Path(G.HIPCC).exists() else shutil.which("hipcc")
    if hipcc is None:
        pytest.skip("no hipcc")
    src = next(s for s in G.SOURCES if s.name == "head_loss.hip")
    flags = [f for f in G.FLAGS if f not in ("-shared", "-fPIC")]
    dst = tmp_path / "head_loss.s"
    subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", str(src), "-o", str(dst)], check=True, capture_output=True)
    asm = dst.read_text()
    assert len(k_loops(asm)) >= 15, "the scan is not looking at the loops it guards"
    assert not extra_waits(asm)
