"""The gfx950 code of the LM head's losses (CPU only): between hl_gemm's sums and its end, every wavefront of a workgroup meets
as many barriers as the others, whichever way it goes. (A wavefront that has ended is not waited for on gfx950, but HIP does
not promise that.)"""

import re
import shutil
import subprocess
from pathlib import Path

import pytest


def blocks_of(body):
    """{label: (barriers, has matrix instructions, successors, ends)} of a function's assembly."""
    out, name, lines = {}, "entry", []
    cuts = []
    for s in (s.split(";")[0].strip() for s in body.split("\n")):
        if s.startswith(".LBB") and s.endswith(":"):
            cuts.append((name, lines))
            name, lines = s[:-1], []
        elif s and not s.startswith("."):
            lines.append(s)
            if s.startswith(("s_cbranch", "s_branch", "s_endpgm")):  # (a block ends at its branch; what follows has no label)
                cuts.append((name, lines))
                name, lines = f"{name}+", []
    cuts.append((name, lines))
    for i, (name, lines) in enumerate(cuts):
        last = lines[-1] if lines else ""
        to = [last.split()[1]] if last.startswith(("s_cbranch", "s_branch")) else []
        if not last.startswith(("s_branch", "s_endpgm")) and i + 1 < len(cuts):
            to.append(cuts[i + 1][0])
        out[name] = (sum(s == "s_barrier" for s in lines), any(s.startswith("v_mfma") for s in lines), to,
                     last.startswith("s_endpgm"))
    return out


def components(blocks):
    """{label: its loop's number}: blocks that reach each other."""
    reach = {}
    for b in blocks:
        seen, todo = set(), list(blocks[b][2])
        while todo:
            t = todo.pop()
            if t not in seen:
                seen.add(t)
                todo += blocks[t][2]
        reach[b] = seen
    return {b: frozenset([b] + [t for t in reach[b] if b in reach[t]]) for b in blocks}, reach


def barriers_left(body):
    """The numbers of barriers that lie ahead of a wavefront that leaves a loop of matrix instructions, over all ways to the
    end; None in it: a loop of barriers."""
    blocks = blocks_of(body)
    loop, reach = components(blocks)
    memo = {}

    def ahead(b):
        if b not in memo:
            part = loop[b]
            own = sum(blocks[t][0] for t in part)
            cyclic = len(part) > 1 or b in blocks[b][2]
            to = {t for p in part for t in blocks[p][2] if t not in part}
            ways = set().union(*(ahead(t) for t in to)) if to else {0}
            memo[b] = {None} if cyclic and own else {None if w is None else w + own for w in ways}
        return memo[b]

    # (the last loops: no further loop of matrix instructions behind them)
    sums = [b for b in blocks if b in reach[b] and any(blocks[t][1] for t in loop[b])]
    sums = [b for b in sums if not any(t in reach[b] and t not in loop[b] for t in sums)]
    return set().union(*(ahead(t) for b in sums for t in blocks[b][2] if t not in loop[b]))


_END = """
.LBB0_1:
\tv_mfma_f32_32x32x16_bf16 a[0:15], v[4:7], v[4:7], a[0:15]
\ts_barrier
\ts_cbranch_scc1 .LBB0_1
\ts_barrier
\ts_cbranch_scc1 .LBB0_3
%s\ts_barrier
.LBB0_3:
%s\ts_endpgm
"""


def test_the_scan_finds_a_way_past_a_barrier():
    assert barriers_left(_END % ("", "")) == {1, 2}
    assert barriers_left(_END % ("", "\ts_barrier\n")) == {2, 3}
    assert barriers_left((_END % ("", "")).replace("\ts_cbranch_scc1 .LBB0_3\n", "")) == {2}


def test_every_wavefront_meets_the_same_barriers(tmp_path):
    import __graft_entry__ as G

    hipcc = G.HIPCC if Path(G.HIPCC).exists() else shutil.which("hipcc")
    if hipcc is None:
        pytest.skip("no hipcc")
    src = next(s for s in G.SOURCES if s.name == "head_loss.hip")
    flags = [f for f in G.FLAGS if f not in ("-shared", "-fPIC")]
    dst = tmp_path / "head_loss.s"
    subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", str(src), "-o", str(dst)], check=True, capture_output=True)
    found = dict(re.findall(r"^(_Z\S*hl_gemm\S+):(.*?)^\.Lfunc_end", dst.read_text(), re.M | re.S))
    assert len(found) >= 15
    ways = {name: barriers_left(body) for name, body in found.items()}
    assert any(w == {2} for w in ways.values()), ways  # (the statistics' own barrier is among what is looked at)
    assert all(len(w) == 1 for w in ways.values()), {n: w for n, w in ways.items() if len(w) != 1}
