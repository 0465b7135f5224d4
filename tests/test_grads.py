"""The gradients' global norm and clipping (common/grads.py) on the GPU against their definition in 64 bits.

Bounds, u = 2^-24: the norm's squares and sums are float64, so it is off by its own rounding (u) and next to nothing else (1e-9 of
itself for up to 2^22 values); the factor is rounded once (u), its product with a value once (u), and to bf16 or float16 once (2^-8,
2^-11; float16 below 2^-14 by half of 2^-24)."""

import math
import threading

import pytest
import torch
from torch.autograd import forward_ad

from common import grads
from common.testing import raises, same, within
from dense_reader import gated
from lm_head_topk import head_loss

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.float32: (0.0, 2.0**-149), torch.bfloat16: (2.0**-8, 2.0**-133), torch.float16: (2.0**-11, 2.0**-25)}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(device, sizes, types, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, s in enumerate(sizes):
        t = torch.randn(s, generator=g) * scale * 10 ** -(i % 4)
        out.append(t.to(types[i % len(types)]).to(device.torch))
    return out


def norm64(ts):
    return torch.stack([t.double().square().sum() for t in ts]).sum().sqrt()


def check(what, ts, norm, outs, max_norm):
    want = norm64(ts)
    within(f"{what}: norm", norm[None], want[None], (want * U * 1.01)[None] + 2.0**-149)
    factor = torch.minimum(max_norm / (want + 1e-6), want.new_ones(()))
    for i, (t, o) in enumerate(zip(ts, outs)):
        r = t.double() * factor
        half, least = HALF[o.dtype]
        if o.numel():
            within(f"{what}: {i} {tuple(o.shape)} {t.dtype} to {o.dtype}", o, r, (half + 2.1 * U) * r.abs() + least + 2.0**-149)


LISTS = [[1], [7], [8], [255, 256, 257], [8191, 8192, 8193], [100003], [0, 5, 0, 8192 * 3, 1], [(33, 65), (1, 1), (128, 256), (3, 5, 7)],
         [1 << 22], [(i * 37) % 300 for i in range(300)], [8192 * 2 + i for i in range(130)], [3_000_017, 1, 2_000_000]]
MIXES = [[F32], [BF16], [F16], [F32, BF16, F16]]


@pytest.mark.parametrize("types", MIXES)
@pytest.mark.parametrize("sizes", LISTS, ids=range(len(LISTS)))
def test_norm_and_clip(device, sizes, types):
    ts = make(device, sizes, types, len(sizes))
    norm = grads.global_norm(ts)
    assert norm.shape == () and norm.dtype == F32
    for max_norm in (norm.item() * 0.3, norm.item() * 3, 0.0):
        n, outs = grads.clipped(ts, max_norm)
        same("the norm alone", norm, n)
        check("own types", ts, n, outs, max_norm)
        for dtype in (F32, BF16, F16):
            n, wide = grads.clipped(ts, max_norm, dtype=dtype)
            check(f"to {dtype}", ts, n, wide, max_norm)
        mine = [t.clone() for t in ts]
        same("in place: norm", grads.clip_(mine, max_norm), norm)
        for a, b in zip(mine, outs):
            same("in place", a, b)
        outs2 = [torch.full_like(t, 7) for t in ts]
        got = grads.clipped(ts, max_norm, out=outs2)[1]
        for a, b, c in zip(got, outs2, outs):
            assert a is b
            same("into out", a, c)


@pytest.mark.parametrize("types", MIXES)
def test_off_alignment(device, types):
    """Tensors and outs that begin anywhere in memory, with other values right around them."""
    pool, ts, outs, at = [], [], [], []
    for i, n in enumerate([1, 9, 8192, 8200, 20001, 5]):
        for shift in (0, 1, 3, 8):
            t = types[(i + shift) % len(types)]
            a, b = (torch.full((n + 40,), 1e4, dtype=t, device=device.torch) for _ in range(2))
            a[shift : shift + n] = torch.randn(n, generator=torch.Generator().manual_seed(i)).to(t).to(device.torch)
            ts.append(a[shift : shift + n]), pool.append(b), outs.append(b[i : i + n]), at.append((i, n))
    norm, got = grads.clipped(ts, 1.5, out=outs)
    check("views", ts, norm, got, 1.5)
    for p, (i, n) in zip(pool, at):
        assert bool((p[:i] == 1e4).all()) and bool((p[i + n :] == 1e4).all())


def test_orders_and_strides(device):
    """Dense memory in another order of its dims, and views that are not dense."""
    base = make(device, [(48, 40, 24)], [F32], 3)[0]
    t = base.permute(2, 0, 1)
    rows = make(device, [(64, 50)], [BF16], 4)[0][:, :33]
    wide = make(device, [(1, 40)], [F32], 5)[0].expand(30, 40)
    ts = [t, rows, wide, base[:, 0]]
    check("strided", ts, grads.global_norm(ts), [], 1.0)
    norm, outs = grads.clipped(ts, 2.0)
    check("strided, clipped", ts, norm, outs, 2.0)
    mine = base.clone().permute(2, 0, 1)
    norm = grads.clip_([mine], 2.0)
    check("another order, in place", [t], norm, [mine], 2.0)
    for bad in (rows, wide):
        raises("in place, not dense", AssertionError, lambda: grads.clip_([bad], 1.0))


def test_extremes(device):
    """Values whose squares no float32 holds, subnormal ones, zeros, NaN and infinities."""
    big = [torch.full((5000,), 1e30, device=device.torch), torch.full((10,), -1e30, dtype=BF16, device=device.torch)]
    norm, outs = grads.clipped(big, 1.0)
    check("large", big, norm, outs, 1.0)
    small = [torch.full((5000,), 1e-30, device=device.torch), torch.full((9,), 6e-8, dtype=F16, device=device.torch)]
    norm, outs = grads.clipped(small, 1e-9)
    check("small", small, norm, outs, 1e-9)
    none = [torch.zeros(9000, device=device.torch)]
    assert grads.clip_(none, 1.0).item() == 0 and not none[0].any()
    past = [torch.full((1 << 20,), 3e38, device=device.torch)]
    norm, outs = grads.clipped(past, 1.0)  # (the norm, 3e41, is no float32; the factor is)
    assert norm.item() == math.inf
    want = 1 / 2.0**10
    within("past float32", outs[0], torch.full_like(outs[0], want, dtype=torch.float64),
           torch.full_like(outs[0], 0.01 * want, dtype=torch.float64))
    ts = make(device, [9000, 50], [F32, BF16], 2)
    ts[0][8500] = math.inf
    norm, outs = grads.clipped(ts, 1.0)
    assert norm.item() == math.inf and outs[0].isnan().sum().item() == 1 and bool(outs[0][8500].isnan()) and not outs[1].any()
    ts[1][3] = math.nan
    norm, outs = grads.clipped(ts, 1.0)
    assert bool(norm.isnan()) and all(bool(o.isnan().all()) for o in outs)
    assert bool(grads.global_norm(ts).isnan())


def test_no_values(device):
    e = torch.empty(0, 3, device=device.torch)
    assert grads.global_norm([e, None]).item() == 0.0
    norm, outs = grads.clipped([None, e], 1.0)
    assert norm.item() == 0.0 and outs[0] is None and outs[1].shape == (0, 3)
    assert grads.clip_([e, e], 1.0).item() == 0.0
    raises("no gradients", ValueError, lambda: grads.global_norm([None]))


def test_given_norm(device):
    ts = make(device, [9000, 77, 200_000], [F32, BF16], 6)
    whole = grads.global_norm(ts)
    total = sum(grads.global_norm([t]).square() for t in ts).sqrt()
    for given in (whole, total, torch.tensor([3.0], device=device.torch)):
        kept = given.clone()
        norm, outs = grads.clipped(ts, 1.0, norm=given)
        assert norm is given
        same("left as it was", given, kept)
        factor = torch.minimum(1.0 / (given.double() + 1e-6), torch.ones_like(given, dtype=torch.float64))
        for t, o in zip(ts, outs):
            r = t.double() * factor
            half, least = HALF[o.dtype]
            within("by the given norm", o, r, (half + 2.1 * U) * r.abs() + least)
    parts = [t.clone() for t in ts]
    for p in parts:
        grads.clip_([p], 1.0, norm=whole)
    for a, b in zip(parts, grads.clipped(ts, 1.0, norm=whole)[1]):
        same("one at a time", a, b)


def test_model(device):
    """A step's gradients, of the gated block and the head's loss with torch's own between them, clipped in place: as torch's clip."""
    g = torch.Generator().manual_seed(8)
    n, d, f, v = 200, 128, 264, 999
    rand = lambda *s: (torch.randn(*s, generator=g) / s[-1] ** 0.5).to(BF16).to(device.torch)
    x = rand(n, d).requires_grad_()
    params = [rand(f, d), rand(f, d), rand(d, f), rand(v, d), torch.ones(d, device=device.torch)]
    for p in params:
        p.requires_grad_()
    ids = torch.randint(0, v, (n,), generator=g).to(device.torch)

    def step():
        y = x + torch.nn.functional.linear(gated.gated(x, params[0], params[1]), params[2])
        y = (y.float() * params[4]).to(BF16)
        return head_loss.token_loss(y, params[3], ids).mean()

    step().backward()
    kept = [p.grad.clone() for p in params]
    norm = grads.clip_((p.grad for p in params), 0.01)
    check("a step", kept, norm, [p.grad for p in params], 0.01)
    assert grads.global_norm(p.grad for p in params).item() <= 0.01 * (1 + 2**-7)
    want = torch.nn.utils.get_total_norm(kept)
    assert abs(norm.item() - want.item()) <= 2**-7 * want.item()  # (torch's partial norms are in the gradients' types)


def test_graph_streams_threads(device):
    """Captured calls replayed on new values with eager work between, two graphs at once, and calls of several streams and threads."""
    lists = [make(device, [70_000, 33, 8192, 500_000], [F32, BF16], 11), make(device, [100] * 200, [BF16, F16], 12)]
    graphs, outs = [], []
    for ts in lists:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((grads.global_norm(ts), *grads.clipped(ts, 0.5)))
        graphs.append(graph)
    for turn in range(4):
        for ts in lists:
            for t in ts:
                t.mul_(1.5)
        for graph in graphs:
            graph.replay()
        for ts, (norm, again, got) in zip(lists, outs):
            want = grads.clipped(ts, 0.5)
            same("norm", norm, want[0]), same("norm of the clip", again, want[0])
            for a, b in zip(got, want[1]):
                same(f"turn {turn}", a, b)
    want = [grads.clipped(ts, 0.5) for ts in lists]
    got = [None, None]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = grads.clipped(lists[i], 0.5)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        same("norm", a[0], b[0])
        for s, t in zip(a[1], b[1]):
            same("on its own thread", s, t)


def test_large(device):
    """More than 2^31 values in one tensor, and chunks of it past 2^32 bytes."""
    n = (1 << 31) + 4099
    t = torch.zeros(n, dtype=BF16, device=device.torch)
    t[-5], t[0], t[1 << 31] = 3.0, 4.0, 12.0
    norm = grads.clip_([t], 1.0)
    assert norm.item() == 13.0
    at = torch.tensor([0, 1, (1 << 31) - 1, 1 << 31, n - 5, n - 1], device=device.torch)
    want = torch.tensor([4, 0, 0, 12, 3, 0], dtype=torch.float64, device=device.torch) / (13 + 1e-6)
    within("its values", t[at], want, want * (2.0**-8 + 3 * U) + 1e-30)
    assert t.count_nonzero().item() == 3


def test_refusals(device):
    a, b = make(device, [64, 64], [F32], 1)
    pool = torch.randn(200, device=device.torch)
    bad = AssertionError
    leaf = a.clone().requires_grad_()
    for what, exc, fn in [
        ("the host", bad, lambda: grads.global_norm([a.cpu()])),
        ("two devices", bad, lambda: grads.global_norm([a, b.cpu()])),
        ("float64", bad, lambda: grads.global_norm([a.double()])),
        ("integers", bad, lambda: grads.global_norm([a.int()])),
        ("requires grad", bad, lambda: grads.global_norm([leaf])),
        ("max_norm < 0", bad, lambda: grads.clip_([a], -1.0)),
        ("max_norm on the device", bad, lambda: grads.clip_([a], torch.ones((), device=device.torch))),
        ("max_norm NaN", bad, lambda: grads.clip_([a], math.nan)),
        ("one tensor twice", ValueError, lambda: grads.clip_([a, a], 1.0)),
        ("shared memory", ValueError, lambda: grads.clip_([pool[:100], pool[99:]], 1.0)),
        ("out twice", ValueError, lambda: grads.clipped([a, b], 1.0, out=[pool[:64], pool[:64]])),
        ("out over another gradient", ValueError, lambda: grads.clipped([a, pool[:64]], 1.0, out=[pool[32:96], b.clone()])),
        ("out over a part of its own", ValueError, lambda: grads.clipped([pool[:64]], 1.0, out=[pool[1:65]])),
        ("out's shape", bad, lambda: grads.clipped([a], 1.0, out=[b[:63]])),
        ("out's type", bad, lambda: grads.clipped([a], 1.0, out=[b.double()])),
        ("out strided", bad, lambda: grads.clipped([a], 1.0, out=[pool[:128:2]])),
        ("outs' number", bad, lambda: grads.clipped([a, b], 1.0, out=[b])),
        ("out for None", bad, lambda: grads.clipped([a, None], 1.0, out=[pool[:64], b])),
        ("None for a gradient", bad, lambda: grads.clipped([a, b], 1.0, out=[pool[:64], None, pool[64:128]])),
        ("a None too many", bad, lambda: grads.clipped([a], 1.0, out=[b, None])),
        ("out and dtype", bad, lambda: grads.clipped([a], 1.0, out=[b], dtype=F32)),
        ("dtype", bad, lambda: grads.clipped([a], 1.0, dtype=torch.float64)),
        ("a norm of the host", bad, lambda: grads.clip_([a], 1.0, norm=torch.ones(()))),
        ("a norm of two", bad, lambda: grads.clip_([a], 1.0, norm=torch.ones(2, device=device.torch))),
    ]:
        raises(what, exc, fn)
    with torch.no_grad():
        grads.clip_([leaf], 1e9)
    with forward_ad.dual_level():
        raises("dual", NotImplementedError, lambda: grads.global_norm([forward_ad.make_dual(a, torch.ones_like(a))]))
    y = (leaf * leaf).sum()
    with torch.no_grad():
        grads.clip_([leaf], 1.0)
    raises("written before its backward", RuntimeError, y.backward)
    same("gradients beside each other", grads.clipped([a], 1.0, out=[a])[1][0], a)


@pytest.mark.parametrize("lists", [1, 3])
def test_no_limit(device, lists):
    """max_norm infinite: the norm alone is asked for. Nothing is clipped whatever the norm is, but for a NaN, which makes all NaN."""
    ts = make(device, [9000, 50, 8192] + [3] * (128 * (lists - 1)), [F32, BF16, F16], 4)
    for what, value, want in [("finite", 1.0, None), ("infinite", -math.inf, math.inf), ("past float32", None, math.inf), ("NaN", math.nan, math.nan)]:
        mine = [t.clone() for t in ts]
        if value is None:
            mine[0][:] = 3e38
        else:
            mine[0][8500] = value
        norm = grads.global_norm(mine)
        for given in (None, norm):
            n, outs = grads.clipped(mine, math.inf, norm=given)
            wide = grads.clipped(mine, math.inf, dtype=F32, norm=given)[1]
            there = [t.clone() for t in mine]
            same_norm = grads.clip_(there, math.inf, norm=given)
            for v in (n, same_norm):
                assert v.isnan() if want is math.nan else v.item() == (norm.item() if want is None else want), (what, v)
            for t, o, w, p in zip(mine, outs, wide, there):
                if want is math.nan:
                    assert bool(o.isnan().all()) and bool(w.isnan().all()) and bool(p.isnan().all()), what
                else:
                    same(f"{what}: as it was", o, t), same("float32", w, t.float()), same("in place", p, t)


def test_many_lists(device):
    """8192 tensors, 64 launches' worth: right, and a clip takes about the time of its norm and of a clip by a given norm (each
    launch of it would add up all 131072 sums again otherwise, several times as long)."""
    count, each = 8192, 16 * 8192
    g = torch.Generator(device.torch).manual_seed(3)
    pool = torch.randn(count, each, generator=g, device=device.torch, dtype=BF16)
    out = torch.empty_like(pool)
    ts, outs = list(pool.unbind()), list(out.unbind())
    want = torch.stack([t.double().square().sum() for t in pool.split(512)]).sum().sqrt()
    norm = grads.global_norm(ts)
    within("norm", norm[None], want[None], (want * U * 1.01)[None])
    given = norm.clone()
    calls = {"clip": lambda: grads.clipped(ts, 1.0, out=outs)[0], "norm": lambda: grads.global_norm(ts),
             "given": lambda: grads.clipped(ts, 1.0, out=outs, norm=given)[0]}
    us = {}
    for name, call in calls.items():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        out.fill_(7)
        for _ in range(3):
            graph.replay()
        ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        ends[0].record()
        for _ in range(5):
            graph.replay()
        ends[1].record()
        torch.cuda.synchronize()
        us[name] = ends[0].elapsed_time(ends[1]) * 200
        same(name, got, norm)
        if name == "norm":
            continue
        for i in (0, 127, 128, 5000, 8191):
            r = ts[i].double() * (1.0 / (want + 1e-6))
            within(f"{name}: {i}", outs[i], r, (2.0**-8 + 2.1 * U) * r.abs() + 2.0**-133)
    print(us, flush=True)
    assert us["clip"] < 1.5 * (us["norm"] + us["given"]), us


def test_norm_that_requires_grad(device):
    """A given norm in a graph: its derivative would be dropped, so it is refused as gradients in a graph are."""
    (a,) = make(device, [64], [F32], 1)
    leaf = torch.full((), 0.5, device=device.torch, requires_grad=True)
    for norm in (leaf, leaf * 2):
        raises("in place", AssertionError, lambda: grads.clip_([a.clone()], 1.0, norm=norm))
        raises("copies", AssertionError, lambda: grads.clipped([a], 1.0, norm=norm))
        want = grads.clipped([a], 1.0, norm=torch.full((), norm.item(), device=device.torch))[1][0]
        with torch.no_grad():
            same("without a graph", grads.clipped([a], 1.0, norm=norm)[1][0], want)
        same("detached", grads.clipped([a], 1.0, norm=norm.detach())[1][0], want)


def test_negative_views(device):
    """The imaginary part of a conjugate is a view of memory with the other sign: one value of it is contiguous."""
    for n in (1, 5):
        z = torch.randn(n, dtype=torch.complex64, generator=torch.Generator().manual_seed(n)).to(device.torch)
        view, plain = z.conj().imag, -z.imag.clone()
        assert view.is_neg() and view.is_contiguous() == (n == 1)
        for max_norm in (0.1, 1e3):
            norm, (got,) = grads.clipped([view], max_norm)
            same("clipped", got, grads.clipped([plain], max_norm)[1][0]), same("norm", norm, grads.global_norm([view]))
            into = torch.empty_like(plain)
            same("into out", grads.clipped([view], max_norm, out=[into])[1][0], got)
            if n == 1:
                there = z.clone()
                grads.clip_([there.conj().imag], max_norm)
                same("in place", -there.imag, got)
    one = torch.ones(1, dtype=torch.complex64, device=device.torch).conj().imag
    raises("a negative out", AssertionError, lambda: grads.clipped([torch.ones(1, device=device.torch)], 1.0, out=[one]))
    raises("a negative norm", AssertionError, lambda: grads.clipped([torch.ones(1, device=device.torch)], 1.0, norm=one))
