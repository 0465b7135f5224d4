"""The gated block in training (dense_reader/gated.py) on the GPU against its definition in 64 bits.

Bounds, value by value, u = 2^-24 (float32) and b = 2^-8 (bf16) being a rounding's largest relative size:
- g and u sum dim products of bf16 (exact in float32): off by at most (dim + 2) u sum |x w|;
- the sigmoid p of v (v = g, or gelu's c (g + 0.044715 g^3), itself 4 u of its size off) is off by at most (8 |v| + 16) u of itself:
  the exponent's rounding, the functions' own few units;
- a = g p: 1.13 |dg| (the largest |a'| of either) and its own roundings; a': 0.8 |dg| (the largest |a''|), its terms' roundings,
  and 1 - p, which is off by u and by p's own error, times what it is multiplied by;
- what is kept, g and u, is cut to 24 bits: 2^-15 of itself; dg and du are rounded to bf16; h, dx and the weights' gradients once at the end.
"""

import math
import threading

import pytest
import torch
from torch.autograd import forward_ad

from common.testing import raises, same, within
from dense_reader import _lib, gated
from test_gated_host import TILES

pytestmark = pytest.mark.gpu

U, B, CUT = 2.0**-24, 2.0**-8, 2.0**-15
TINY = 2.0**-120


def inputs(device, n, d, f, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g)
    x[:, :4] *= 8
    bf16 = lambda t: t.to(torch.bfloat16).to(device.torch)
    return (bf16(x), bf16(torch.randn(f, d, generator=g) * scale / d**0.5), bf16(torch.randn(f, d, generator=g) / d**0.5),
            bf16(torch.randn(n, f, generator=g)))


def act_of(g, kind):
    """(a, a', the sigmoid, v, what 1 - p is multiplied by in a') in 64 bits."""
    if kind == "swiglu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * torch.sigmoid(-g)), p, g, g.abs()
    c = 2 * math.sqrt(2 / math.pi)
    v = c * (g + 0.044715 * g**3)
    p, q = torch.sigmoid(v), c * (1 + 3 * 0.044715 * g * g)
    return g * p, p + g * p * torch.sigmoid(-v) * q, p, v, (g * q).abs().clamp(max=16 * 60)


def expected(x, wg, wu, dh, kind, cut):
    """{what: (value, bound)} of h, dx and both weights' gradients; cut: how far what is kept is off."""
    x, wg, wu, dh = (t.double() for t in (x, wg, wu, dh))
    n, d = x.shape
    g, u = x @ wg.T, x @ wu.T
    eg, eu = ((d + 2) * U * (x.abs() @ w.abs().T) for w in (wg, wu))
    a, s, p, v, t = act_of(g, kind)
    r = (8 * v.abs().clamp(max=200) + 16) * U
    ea = 1.13 * eg + a.abs() * (r + 2 * U) + TINY
    h, eh = a * u, u.abs() * ea + a.abs() * eu + ea * eu
    out = {"h": (h, eh + (B + U) * (h.abs() + eh) + TINY)}
    eg, eu = (e + cut * (m.abs() + e) for e, m in ((eg, g), (eu, u)))
    ea = 1.13 * eg + a.abs() * (r + 2 * U) + TINY
    es = 0.8 * eg + (p + t * p * (1 - p)) * (r + 8 * U) + t * p * (p * r + U) + TINY
    su, esu = s * u, es * u.abs() + s.abs() * eu + es * eu
    esu += 2 * U * (su.abs() + esu)
    dg, du = dh * su, dh * a
    edg, edu = ((e * dh.abs() + (B + U) * (m.abs() + e * dh.abs())) for e, m in ((esu, dg), (ea, du)))
    for name, val, err, mag, depth in (
        ("dx", dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs(), dg.abs() @ wg.abs() + du.abs() @ wu.abs(), 2 * wg.shape[0]),
        ("dgate", dg.T @ x, edg.T @ x.abs(), dg.abs().T @ x.abs(), n),
        ("dup", du.T @ x, edu.T @ x.abs(), du.abs().T @ x.abs(), n),
    ):
        e = err + (depth + 64) * U * 1.02 * mag
        out[name] = val, e + (B + U) * (val.abs() + e) + TINY
    return out


NAMES = ("dx", "dgate", "dup")
SIZES = [(1, 8, 8), (1, 64, 4096), (2, 1024, 264), (5, 72, 1000), (31, 520, 96), (32, 256, 256), (33, 2048, 512), (64, 128, 14336),
         (65, 72, 520), (127, 1000, 248), (128, 64, 64), (129, 264, 2312), (257, 4096, 136), (300, 384, 1504), (513, 1000, 768),
         (1000, 128, 5000), (1003, 2056, 1288), (2100, 512, 2048), (5000, 64, 40), (4100, 1032, 2056)]


@pytest.mark.parametrize("n, d, f", SIZES + [sizes for sizes, _ in TILES])
@pytest.mark.parametrize("kind", ["swiglu", "geglu"])
def test_step(device, n, d, f, kind):
    x, wg, wu, dh = inputs(device, n, d, f, n + d + f)
    want, again = (expected(x, wg, wu, dh, kind, cut) for cut in (CUT, 0.0))
    h, kept = gated.gated_keep(x, wg, wu, kind)
    within(f"{kind} {n} x {d} x {f}: h", h, *want["h"])
    same("h alone", gated.gated(x, wg, wu, kind), h)
    grads = gated.gated_grads(x, wg, wu, dh, kind, kept=kept)
    for name, t in zip(NAMES, grads):
        within(f"  {name}", t, *want[name])
    for name, t in zip(NAMES, gated.gated_grads(x, wg, wu, dh, kind)):
        within(f"  {name} again", t, *again[name])
    dx, dg, du = gated.gated_grads(x, wg, wu, dh, kind, kept=kept, w_grad=False)
    assert dg is None and du is None
    same("dx alone", dx, grads[0])
    dx, dg, du = gated.gated_grads(x, wg, wu, dh, kind, kept=kept, x_grad=False)
    assert dx is None
    same("dgate alone", dg, grads[1]), same("dup alone", du, grads[2])
    assert gated.gated_grads(x, wg, wu, dh, kind, x_grad=False, w_grad=False) == (None, None, None)


@pytest.mark.parametrize("n", [3, 200, 1500])
def test_strides(device, n):
    """x, the weights and dh as views: of wider rows, of one fused parameter, off their alignment, transposed, NaN around them."""
    d, f = 264, 520
    x, wg, wu, dh = inputs(device, n, d, f, 7)
    h, kept = gated.gated_keep(x, wg, wu)
    want = gated.gated_grads(x, wg, wu, dh, kept=kept)

    def wide(t, left, right):
        w = torch.full((t.shape[0] + 2, t.shape[1] + left + right), float("nan"), dtype=t.dtype, device=t.device)
        view = w[1:-1, left : left + t.shape[1]]
        view.copy_(t)
        return view

    fused = torch.cat([wg, wu])
    views = [
        ("wide rows", [wide(t, 8, 16) for t in (x, wg, wu, dh)]),
        ("gate alone", [x, wide(wg, 16, 0), wu, dh]),
        ("up alone", [x, wg, wide(wu, 0, 8), dh]),
        ("fused", [x, fused[:f], fused[f:], dh]),
        ("every other row", [torch.stack([t, t], 1).flatten(0, 1)[::2] for t in (x, wg, wu, dh)]),
        ("off alignment", [wide(t, 3, 2) for t in (x, wg, wu, dh)]),
        ("transposed", [t.T.contiguous().T for t in (x, wg, wu, dh)]),
        ("far rows", [wide(x, 0, 1 << 21), wg, wu, dh] if n == 3 else [x, wg, wu, dh]),
    ]
    for what, (vx, vg, vu, vdh) in views:
        got, k = gated.gated_keep(vx, vg, vu)
        same(f"{what}: h", got, h)
        for name, a, b in zip(NAMES, gated.gated_grads(vx, vg, vu, vdh, kept=k), want):
            same(f"  {name}", a, b)
        for name, a, b in zip(NAMES, gated.gated_grads(vx, vg, vu, vdh), gated.gated_grads(x, wg, wu, dh)):
            same(f"  {name} again", a, b)


def test_shapes(device):
    x, wg, wu, dh = inputs(device, 12, 64, 96, 3)
    h = gated.gated(x, wg, wu)
    for lead in ((3, 4), (2, 1, 6), (12,)):
        got, kept = gated.gated_keep(x.reshape(*lead, 64), wg, wu)
        assert got.shape == (*lead, 96)
        same("h", got.reshape(12, 96), h)
        dx = gated.gated_grads(x.reshape(*lead, 64), wg, wu, dh.reshape(*lead, 96), kept=kept)[0]
        assert dx.shape == (*lead, 64)
    one = gated.gated(x[5], wg, wu)
    assert one.shape == (96,)
    same("a vector", one, gated.gated(x[5:6], wg, wu)[0])
    empty = x[:0].requires_grad_()
    wg = wg.clone().requires_grad_()
    h = gated.gated(empty, wg, wu)
    assert h.shape == (0, 96)
    h.sum().backward()
    assert empty.grad.shape == (0, 64) and not wg.grad.any()


@pytest.mark.parametrize("kind", ["swiglu", "geglu"])
def test_far_values(device, kind):
    """Gates far from 0, where the sigmoid is 0 or 1 and a' times u neither overflows nor is lost."""
    x, wg, wu, dh = inputs(device, 40, 64, 96, 5, scale=300.0)
    want = expected(x, wg, wu, dh, kind, CUT)
    h, kept = gated.gated_keep(x, wg, wu, kind)
    within("h", h, *want["h"])
    for name, t in zip(NAMES, gated.gated_grads(x, wg, wu, dh, kind, kept=kept)):
        within(name, t, *want[name])
    huge = wg * 2.0**60  # g to 2^70: g^3 is no float32
    h = gated.gated(x, huge, wu, kind)
    g, u = x.double() @ huge.double().T, x.double() @ wu.double().T
    eg, eu = (66 * U * (x.double().abs() @ w.double().abs().T) for w in (huge, wu))
    on = g.abs() > 4 * eg
    bound = (B + 4 * U) * (g * u).abs() + 1.01 * (eg * u.abs() + g.abs() * eu + eg * eu)
    within("positive", h[on & (g > 0)], (g * u)[on & (g > 0)], bound[on & (g > 0)])
    assert not h[on & (g < 0)].any()
    dx, dgate, dup = gated.gated_grads(x, huge, wu, dh, kind)
    assert bool(dup.isfinite().all()) and bool(dgate.isfinite().all())


@pytest.mark.parametrize("n", [6, 300])
def test_not_finite(device, n):
    """A NaN or an infinity in a row of x or dh, or in a weight's row, reaches what depends on it and nothing else."""
    x, wg, wu, dh = inputs(device, n, 64, 520, 9)
    h, kept = gated.gated_keep(x, wg, wu)
    dx = gated.gated_grads(x, wg, wu, dh, kept=kept)[0]
    rest = torch.arange(n, device=x.device) != 4
    for bad in (float("nan"), float("inf")):
        xb = x.clone()
        xb[4, 7] = bad
        hb, kb = gated.gated_keep(xb, wg, wu)
        same("the other rows", hb[rest], h[rest])
        assert not hb[4].isfinite().all()
        same("their dx", gated.gated_grads(xb, wg, wu, dh, kept=kb)[0][rest], dx[rest])
        wb = wu.clone()
        wb[3, 5] = bad
        hb = gated.gated(x, wg, wb)
        others = torch.arange(520, device=x.device) != 3
        same("the other outputs", hb[:, others], h[:, others])
        db = dh.clone()
        db[4, 3] = bad
        got = gated.gated_grads(x, wg, wu, db, kept=kept)
        same("dx of the other rows", got[0][rest], dx[rest])
        assert not got[0][4].isfinite().any() and not got[2][3].isfinite().all()
        assert bool(got[2][others].isfinite().all())


def test_differences(device):
    """The gradients against differences of the definition in 64 bits along random directions."""
    x, wg, wu, dh = inputs(device, 24, 64, 80, 13)
    for kind in ("swiglu", "geglu"):
        def loss(x, wg, wu):
            return (act_of(x @ wg.T, kind)[0] * (x @ wu.T) * dh.double()).sum()

        want = expected(x, wg, wu, dh, kind, 0.0)
        at = [t.double() for t in (x, wg, wu)]
        for i, (name, got) in enumerate(zip(NAMES, gated.gated_grads(x, wg, wu, dh, kind))):
            v = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(x.device)
            ends = [loss(*[t + e * v if j == i else t for j, t in enumerate(at)]) for e in (1e-5, -1e-5)]
            slope, bound = (ends[0] - ends[1]) / 2e-5, (want[name][1] * v.abs()).sum() + 1e-6 * loss(*[t.abs() for t in at]).abs()
            within(f"{kind} {name}", (got.double() * v).sum()[None], slope[None], bound[None])


def leaves(*ts):
    return [t.clone().requires_grad_() for t in ts]


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("n", [3, 140])
def test_autograd(device, n, keep):
    x, wg, wu, dh = inputs(device, n, 128, 264, 21)
    kept = gated.gated_keep(x, wg, wu, "geglu")[1] if keep else None
    want = gated.gated_grads(x, wg, wu, dh, "geglu", kept=kept)
    for mask in range(1, 8):
        ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, wg, wu))]
        h = gated.gated(*ts, "geglu", keep=keep)
        h.backward(dh, retain_graph=True)
        for i, (t, w) in enumerate(zip(ts, want)):
            if mask >> i & 1:
                same(f"{mask} {i}", t.grad, w)
            else:
                assert t.grad is None
        h.backward(dh)  # (a second time: what is kept is not used up)
        for i, (t, w) in enumerate(zip(ts, want)):
            if mask >> i & 1:
                same(f"{mask} {i} twice", t.grad, w * 2)
    a, w = leaves(x, wg)
    gated.gated(a, w, w, "geglu", keep=keep).backward(dh)  # one weight in both places
    _, g2, u2 = gated.gated_grads(x, wg, wg, dh, "geglu", kept=gated.gated_keep(x, wg, wg, "geglu")[1] if keep else None)
    same("one weight twice", w.grad, g2 + u2)
    a, w, v = leaves(x, wg, wu)
    gated.gated(a, w, v, "geglu", keep=keep).sum().backward()  # (dh a broadcast of one value)
    ones = gated.gated_grads(x, wg, wu, torch.ones_like(dh), "geglu", kept=kept)
    same("a broadcast dh", w.grad, ones[1])
    with torch.no_grad():
        assert not gated.gated(a, w, v, "geglu").requires_grad
    (fused,) = leaves(torch.cat([wg, wu]))  # both halves of one parameter
    gated.gated(x, fused[:264], fused[264:], "geglu", keep=keep).backward(dh)
    same("a fused parameter", fused.grad, torch.cat(want[1:]))


@pytest.mark.parametrize("n, d, f", [(60, 128, 264), (70, 400, 12128), (69, 280, 11016), (1100, 72, 520)])
def test_one_weight(device, n, d, f):
    """Either weight's gradient alone, in each kind of tile."""
    x, wg, wu, dh = inputs(device, n, d, f, 25)
    want = gated.gated_grads(x, wg, wu, dh, kept=gated.gated_keep(x, wg, wu)[1])
    for i in (0, 1):
        ts = [wg.clone().requires_grad_(i == 0), wu.clone().requires_grad_(i == 1)]
        gated.gated(x, *ts).backward(dh)
        same(f"weight {i}", ts[i].grad, want[1 + i])
        assert ts[1 - i].grad is None


def test_inputs_written_in_between(device):
    x, wg, wu, dh = inputs(device, 20, 64, 96, 23)
    for i in range(3):
        ts = [t.clone().requires_grad_() for t in (x, wg, wu)]
        h = gated.gated(*ts)
        with torch.no_grad():
            ts[i].mul_(2)
        raises("written", RuntimeError, lambda: h.backward(dh))
    a = x.clone().requires_grad_()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        raises("dual", NotImplementedError, lambda: gated.gated(dual, wg, wu))
        raises("dual dh", NotImplementedError,
               lambda: gated.gated_grads(x, wg, wu, forward_ad.make_dual(dh, torch.ones_like(dh))))
    h = gated.gated(a, wg, wu)
    (dx,) = torch.autograd.grad(h, a, dh, create_graph=True)
    raises("a second derivative", RuntimeError, lambda: dx.sum().backward())


def test_graph(device):
    """A captured step, replayed on new inputs with eager work between, and two graphs at once; backward() refuses capture."""
    sets = [inputs(device, n, 256, 1000, 30 + n) for n in (40, 700)]
    graphs, outs, bufs = [], [], []
    for s in sets:
        bufs.append([t.clone() for t in s])
        x, wg, wu, dh = bufs[-1]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            gated.gated_keep(x, wg, wu)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h, kept = gated.gated_keep(x, wg, wu)
            outs.append([h, *gated.gated_grads(x, wg, wu, dh, kept=kept), *gated.gated_grads(x, wg, wu, dh)])
        graphs.append(graph)
    for turn in range(4):
        for b, s in zip(bufs, sets):
            for i, (t, v) in enumerate(zip(b, s)):
                t.copy_(v.roll(turn * (i + 1), 0))
        for g in graphs:
            g.replay()
        eager = []
        for b in bufs:
            x, wg, wu, dh = b
            h, kept = gated.gated_keep(x, wg, wu)
            eager.append([h, *gated.gated_grads(x, wg, wu, dh, kept=kept), *gated.gated_grads(x, wg, wu, dh)])
        torch.cuda.synchronize()
        for i, (got, want) in enumerate(zip(outs, eager)):
            for j, (a, b) in enumerate(zip(got, want)):
                same(f"turn {turn}, graph {i}, output {j}", a, b)
    x, wg, wu, dh = bufs[0]
    leaf = x.clone().requires_grad_()
    h = gated.gated(leaf, wg, wu)
    real = torch.cuda.is_current_stream_capturing
    torch.cuda.is_current_stream_capturing = lambda: True  # (as a capture would have it; none is begun)
    try:
        raises("backward in a capture", RuntimeError, lambda: h.backward(dh))
    finally:
        torch.cuda.is_current_stream_capturing = real

def test_streams_and_threads(device):
    sets = [inputs(device, n, 256, 1000, 50 + n) for n in (40, 300, 700)]
    want = []
    for x, wg, wu, dh in sets:
        h, kept = gated.gated_keep(x, wg, wu)
        want.append([h, *gated.gated_grads(x, wg, wu, dh, kept=kept)])
    torch.cuda.synchronize()
    got = [None] * len(sets)

    def work(i):
        x, wg, wu, dh = sets[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                ts = [t.detach().requires_grad_() for t in (x, wg, wu)]
                h = gated.gated(*ts)
                got[i] = [h.detach(), *torch.autograd.grad(h, ts, dh)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        for s, t in zip(a, b):
            same("on its own stream and thread", s, t)


def test_large(device):
    """Offsets past 32 bits in h, in what is kept, in dg and du: the last rows and outputs against the definition."""
    n, d, f = 70001, 64, 32776
    g = torch.Generator(device.torch).manual_seed(4)
    bf16 = lambda *s: torch.randn(*s, generator=g, device=device.torch).to(torch.bfloat16)
    x, wg, wu = bf16(n, d), bf16(f, d) / 8, bf16(f, d) / 8
    dh = torch.empty(n, f, dtype=torch.bfloat16, device=device.torch)
    for i in range(0, n, 7001):
        dh[i : i + 7001] = bf16(min(7001, n - i), f)
    h, kept = gated.gated_keep(x, wg, wu)
    rows = torch.tensor([0, 35000, n - 2, n - 1], device=device.torch)
    for cut, k in ((CUT, kept), (0.0, None)):
        dx, dg, du = gated.gated_grads(x, wg, wu, dh, kept=k)
        part = expected(x[rows], wg, wu, dh[rows], "swiglu", cut)
        within("h of rows", h[rows], *part["h"])
        within("dx of rows", dx[rows], *part["dx"])
        outs = torch.tensor([0, 1, 255, 256, 16384, f - 9, f - 1], device=device.torch)
        part = expected(x, wg[outs], wu[outs], dh[:, outs], "swiglu", cut)
        within("h of outputs", h[:, outs], *part["h"])
        within("dgate of outputs", dg[outs], *part["dgate"])
        within("dup of outputs", du[outs], *part["dup"])


def test_refusals(device):
    x, wg, wu, dh = inputs(device, 4, 64, 96, 1)
    h, kept = gated.gated_keep(x, wg, wu)
    bad = AssertionError
    for what, fn in {
        "activation": lambda: gated.gated(x, wg, wu, "relu"),
        "float32 x": lambda: gated.gated(x.float(), wg, wu),
        "float32 weight": lambda: gated.gated(x, wg.float(), wu),
        "x on the host": lambda: gated.gated(x.cpu(), wg, wu),
        "a weight on the host": lambda: gated.gated(x, wg, wu.cpu()),
        "other widths": lambda: gated.gated(x, wg[:88], wu),
        "other dims": lambda: gated.gated(x[:, :56], wg, wu),
        "dim 60": lambda: gated.gated(x[:, :60], wg[:, :60], wu[:, :60]),
        "width 90": lambda: gated.gated(x, wg[:90], wu[:90]),
        "a weight of three dims": lambda: gated.gated(x, wg[None], wu[None]),
        "dh's rows": lambda: gated.gated_grads(x, wg, wu, dh[:3]),
        "dh's type": lambda: gated.gated_grads(x, wg, wu, dh.float()),
        "dh on the host": lambda: gated.gated_grads(x, wg, wu, dh.cpu()),
        "kept of other rows": lambda: gated.gated_grads(x, wg, wu, dh, kept=gated.gated_keep(x[:3], wg, wu)[1]),
        "kept of another type": lambda: gated.gated_grads(x, wg, wu, dh, kept=kept.view(torch.bfloat16)),
        "kept strided": lambda: gated.gated_grads(x, wg, wu, dh, kept=torch.cat([kept, kept], 3)[..., :256]),
    }.items():
        raises(what, bad, fn)
    assert _lib.DR_GATED_BACKWARD == 2


def test_most_rows(device):
    """2^20 rows by 16384 outputs, more tiles of 64 x 64 than a launch holds: the large tiles'."""
    n, d, f = 1 << 20, 8, 16384
    g = torch.Generator(device.torch).manual_seed(5)
    bf16 = lambda *s: torch.randn(*s, generator=g, device=device.torch).to(torch.bfloat16)
    x, wg, wu = bf16(n, d), bf16(f, d), bf16(f, d)
    h = gated.gated(x, wg, wu)
    rows = torch.tensor([0, 1, 255, 256, 524287, 1 << 19, n - 257, n - 1], device=device.torch)
    part = expected(x[rows], wg, wu, torch.zeros(len(rows), f, device=device.torch), "swiglu", 0.0)
    within("h of rows", h[rows], *part["h"])


@pytest.mark.parametrize("kind", ["swiglu", "geglu"])
@pytest.mark.parametrize("n", [5, 64, 65, 700])
def test_saturated_gradients(device, n, kind):
    """Gates to 2^70, where a is g or 0 and a' 1 or 0: every gradient against those, by what was kept (few rows and many) and again."""
    x, wg, wu, dh = inputs(device, n, 64, 96, 6)
    wg = wg * 2.0**70
    gx, gw, gu, gd = (t.double() for t in (x, wg, wu, dh))
    g, u = gx @ gw.T, gx @ gu.T
    eg, eu = (66 * U * (gx.abs() @ w.abs().T) for w in (gw, gu))
    sure = (g.abs() > 4 * eg) & (g.abs() > 1e4)  # (the sign is the kernel's too, and the sigmoid 0 or 1 in 64 bits)
    dh = torch.where(sure, dh, torch.zeros_like(dh))  # (the others count for nothing)
    gd = dh.double()
    on = ((g > 0) & sure).double()
    dg, du = gd * u * on, gd * g * on
    h, kept = gated.gated_keep(x, wg, wu, kind)
    for what, k, cut in (("kept", kept, CUT), ("again", None, 0.0)):
        edg = gd.abs() * (eu + cut * (u.abs() + eu) + 4 * U * u.abs()) * on
        edu = gd.abs() * (eg + cut * (g.abs() + eg) + 4 * U * g.abs()) * on
        edg, edu = edg + (B + U) * (dg.abs() + edg), edu + (B + U) * (du.abs() + edu)
        got = gated.gated_grads(x, wg, wu, dh, kind, kept=k)
        for name, t, val, err, mag, depth in (
            ("dx", got[0], dg @ gw + du @ gu, edg @ gw.abs() + edu @ gu.abs(), dg.abs() @ gw.abs() + du.abs() @ gu.abs(), 2 * 96),
            ("dgate", got[1], dg.T @ gx, edg.T @ gx.abs(), dg.abs().T @ gx.abs(), n),
            ("dup", got[2], du.T @ gx, edu.T @ gx.abs(), du.abs().T @ gx.abs(), n),
        ):
            e = err + (depth + 64) * U * 1.02 * mag
            within(f"{kind} {n} {what}: {name}", t, val, e + (B + U) * (val.abs() + e) + TINY)
