"""The LM head's losses (lm_head_topk/head_loss.py) on the GPU against their definition in 64 bits.

Bounds, value by value, u = 2^-24 (float32) and b = 2^-8 (bf16) being a rounding's largest relative size:
- a logit sums dim products of bf16 (exact in float32): off by at most dim u sum |x w| (any order of the sum); ez is that of
  the row's largest, with one rounding more for the scaling by 1 / T;
- lse and loss add the exponents' roundings (|z| u each, both ways of the base change, and the functions' own few units) and
  the sums' of at most 1024 parts;
- dz = g / T (p - q): p off by the factor exp of those, dz rounded to bf16 (b) and scaled there and back (2 u);
- dx and dhead sum products of it in float32 and are rounded to bf16 once.
"""

import math

import pytest
import torch

from common.testing import raises, same, within
from dense_reader import linear
from lm_head_topk import head_loss, head_pick, lmhead
from moe import balance, moe8

pytestmark = pytest.mark.gpu

U, B = 2.0**-24, 2.0**-8


def inputs(device, n, v, d, seed, spread=0.1, ld=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g)
    x[:, :4] *= 8
    x = x.to(torch.bfloat16).to(device.torch)
    if ld:
        wide = torch.full((n, ld), float("nan"), dtype=torch.bfloat16, device=device.torch)
        wide[:, :d] = x
        x = wide[:, :d]
    head = (torch.randn(v, d, generator=g) * spread).to(torch.bfloat16).to(device.torch)
    return x, head, torch.rand(n, generator=g).to(device.torch), g


def entries(ids, vals, valid, t):
    """(ids, q, rows that count, sum of q log q) in 64 bits."""
    if vals is None:
        on = (ids >= 0) & (ids < valid)
        return torch.where(on, ids, 0).long()[:, None], on.double()[:, None], on, 0.0
    held = (ids >= 0) & (ids < valid) & (vals != -math.inf)
    on = held.any(1)
    lq = torch.where(held, vals.double() / t, -math.inf)
    q = torch.where(on[:, None], torch.softmax(lq, 1), 0.0)
    return torch.where(held, ids, 0).long(), q, on, -torch.special.entr(q).sum(1)


def expected(x, head, ids, vals, t, valid, g, b=B):
    """[(value, bound)] of loss, dx and dhead, in 64 bits; b: how far dz's rounding is off."""
    n, d = x.shape
    ids, q, on, ent = entries(ids, vals, valid, t)
    x = torch.where(on[:, None], x.double(), 0.0)
    w = head[:valid].double()
    z = x @ w.T / t
    lse = torch.logsumexp(z, 1)
    p = (z - lse[:, None]).exp()
    ez = (d + 2) * U * (x.abs() @ w.abs().T).amax(1) / t
    zt = z.gather(1, ids)
    big = z.abs().amax(1) + lse.abs() + 1
    loss = torch.where(on, (q * (lse[:, None] - zt)).sum(1) + ent, 0.0)
    eloss = torch.where(on, 2 * ez + (1024 + 8 * 64) * U + 16 * U * big + 8 * U * (abs(ent) if vals is not None else 0) +
                        (0 if vals is None else 8 * U * (torch.where(q > 0, vals.double(), 0.0).abs().amax(1) / t + 1)), U)
    gt = torch.where(on, g.double(), 0.0)[:, None] / t
    dz = p * on[:, None]
    eq = torch.zeros_like(dz).scatter_add_(1, ids, q)
    ep = dz * (3 * ez + (1024 + 16) * U + 16 * U * big)[:, None]
    # the teacher's q: the difference's rounding, exp and the division's
    evals = 0 if vals is None else torch.where(q > 0, vals.double(), 0.0).abs().amax(1)[:, None] / t
    ep += eq * (64 + 8 + 4 * evals) * U * (vals is not None)
    dz, ep = (dz - eq) * gt, ep * gt.abs()
    ez2 = ep + (b + 4 * U) * (dz.abs() + ep)
    out = [(loss, eloss)]
    for val, err, mag, depth in (
        (dz @ w, ez2 @ w.abs(), dz.abs() @ w.abs(), valid),
        (dz.T @ x, ez2.T @ x.abs(), dz.abs().T @ x.abs(), n),
    ):
        e = err + (depth + 64) * U * 1.01 * mag
        out.append((val, e + (B + 4 * U) * (val.abs() + e) + 2.0**-133))
    full = torch.zeros(2, *head.shape, dtype=torch.float64, device=head.device)
    full[0, :valid], full[1], full[1, :valid] = out[2][0], 2.0**-133, out[2][1]
    out[2] = (full[0], full[1])
    return out


def check(name, got, want):
    for part, y, (r, bound) in zip(("loss", "dx", "dhead"), got, want):
        if y is not None:
            within(f"{name}: {part}", y, r, bound)


def teacher(n, k, valid, g, device, empty=True):
    ids = torch.randint(-2 if empty else 0, valid + (2 if empty else 0), (n, k), generator=g).int()
    vals = torch.randn(n, k, generator=g) * 3
    if empty:
        vals[torch.rand(n, k, generator=g) < 0.1] = -math.inf
    return ids.to(device.torch), vals.to(device.torch)


TOKEN = [(1, 1, 1, 8), (1, 1000, 1000, 64), (2, 257, 257, 72), (33, 999, 998, 520), (64, 8192, 8192, 1024),
         (65, 513, 500, 96), (127, 3000, 3000, 200), (128, 255, 255, 264), (129, 1025, 1024, 64), (300, 2048, 2047, 384),
         (513, 769, 769, 1000), (1000, 5003, 5000, 128),
         (40, 70001, 70000, 64), (700, 2900, 2899, 520), (2100, 20000, 19999, 72), (70000, 300, 300, 8)]


@pytest.mark.parametrize("n, v, valid, d", TOKEN)
def test_token(device, n, v, valid, d):
    x, head, w, g = inputs(device, n, v, d, n + v + d)
    ids = torch.randint(0, valid, (n,), generator=g)
    ids[torch.rand(n, generator=g) < 0.2] = -100
    if n > 2:
        ids[0], ids[1], ids[2] = valid, valid - 1, 0
    ids = ids.to(device.torch)
    out = head_loss.token_loss_grads(x, head, ids, w, valid=valid)
    check(f"token {n} x {v} ({valid}) x {d}", out, expected(x, head, ids, None, 1.0, valid, w))
    assert bool((out[1][(ids < 0) | (ids >= valid)] == 0).all()) and bool((out[2][valid:] == 0).all())
    same("the loss alone", head_loss.token_loss(x, head, ids.int(), valid=valid), out[0])
    one = head_loss.token_loss_grads(x, head, ids, w, valid=valid, head_grad=False)
    assert one[2] is None
    same("dx alone", one[1], out[1])
    one = head_loss.token_loss_grads(x, head, ids, w, valid=valid, x_grad=False)
    assert one[1] is None
    same("dhead alone", one[2], out[2])


@pytest.mark.parametrize("n, v, valid, d, k, t", [
    (1, 64, 64, 8, 1, 1.0), (3, 1000, 990, 64, 64, 0.5), (40, 8192, 8192, 256, 8, 1.0), (100, 700, 700, 136, 5, 2.0),
    (200, 2049, 2048, 64, 33, 0.7), (600, 1300, 1300, 320, 16, 4.0),
])
def test_distill(device, n, v, valid, d, k, t):
    x, head, w, g = inputs(device, n, v, d, n + v + k)
    ids, vals = teacher(n, k, valid, g, device)
    if n > 2:
        ids[0] = -1  # a row of empty slots
        ids[1] = 7  # one id in every slot
        vals[2] = -math.inf
    out = head_loss.distill_loss_grads(x, head, vals, ids, w, temperature=t, valid=valid)
    check(f"distill {n} x {v} ({valid}) x {d}, {k} at {t}", out, expected(x, head, ids, vals, t, valid, w))
    if n > 2:
        assert out[0][0] == 0 and out[0][2] == 0 and not out[1][[0, 2]].any()
    same("the loss alone", head_loss.distill_loss(x, head, vals, ids, temperature=t, valid=valid), out[0])


@pytest.mark.parametrize("n, v, valid, d, k", [
    (100, 700, 690, 768, 0), (70, 257, 257, 2048, 0), (300, 5003, 5000, 1024, 0), (2100, 2900, 2899, 776, 0),
    (600, 20000, 19990, 800, 0), (100, 700, 690, 768, 64), (70, 257, 257, 2048, 1), (300, 5003, 5000, 1024, 5),
    (2100, 2900, 2899, 776, 16), (600, 20000, 19990, 800, 2), (64, 32768, 32768, 64, 0), (64, 32769, 32769, 64, 0),
    (64, 32768, 32760, 64, 64), (63, 40000, 40000, 72, 7), (5, 300, 299, 8, 64), (64, 513, 512, 1024, 3),
    (256, 1000, 999, 64, 0), (129, 2900, 2899, 264, 0), (193, 600, 600, 72, 16), (256, 1000, 1000, 64, 17),
    (257, 600, 600, 64, 0),
])
def test_logits_kept_for_the_gradient(device, n, v, valid, d, k):
    """Many values a row, and few rows: the gradient is made of the loss's own logits. Some rows are left out, one id comes in
    every slot, weights and vocabularies of any size."""
    x, head, w, g = inputs(device, n, v, d, n + v + d + k)
    w[0] = -2.0
    if k:
        ids, vals = teacher(n, k, valid, g, device)
        ids[1], vals[2], ids[3] = 7, -math.inf, -1
        x[2:4] = math.nan
        run = lambda fn, *a, **kw: fn(x, head, vals, ids, *a, temperature=1.5, valid=valid, **kw)
        loss, grads = head_loss.distill_loss, head_loss.distill_loss_grads
        want = expected(x, head, ids, vals, 1.5, valid, w)
    else:
        ids = torch.randint(0, valid, (n,), generator=g)
        ids[torch.rand(n, generator=g) < 0.2] = -100
        ids[0], ids[1], ids[2] = valid, valid - 1, 0
        ids = ids.to(device.torch)
        x[0] = math.nan
        run = lambda fn, *a, **kw: fn(x, head, ids, *a, valid=valid, **kw)
        loss, grads = head_loss.token_loss, head_loss.token_loss_grads
        want = expected(x, head, ids, None, 1.0, valid, w)
    out = run(grads, w)
    check(f"{n} x {v} ({valid}) x {d}, {k} entries", out, want)
    same("the loss alone", run(loss), out[0])
    same("dx alone", run(grads, w, head_grad=False)[1], out[1])
    same("dhead alone", run(grads, w, x_grad=False)[2], out[2])
    same("again", run(grads, w)[1], out[1])


@pytest.mark.parametrize("n, v, valid, d, k", [
    (1, 2900, 2899, 552, 5), (1, 1, 1, 8, 0), (2, 257, 256, 64, 0), (32, 8192, 8192, 1024, 8), (31, 40000, 40000, 72, 64),
    (17, 5000, 4999, 264, 0), (8, 100, 100, 4096, 3),
])
def test_few_rows_keep_what_rounding_leaves(device, n, v, valid, d, k):
    """Of up to 32 rows the products take dz with what its rounding to bf16 leaves, rounded too: off by b^2 instead of b."""
    x, head, w, g = inputs(device, n, v, d, n + v + d + k)
    if k:
        ids, vals = teacher(n, k, valid, g, device)
        if n > 2:
            ids[1] = -1
        out = head_loss.distill_loss_grads(x, head, vals, ids, w, valid=valid)
    else:
        ids, vals = torch.randint(0, valid, (n,), generator=g).to(device.torch), None
        if n > 2:
            ids[1] = -100
        out = head_loss.token_loss_grads(x, head, ids, w, valid=valid)
    check(f"{n} x {v} x {d}, {k}", out, expected(x, head, ids, vals, 1.0, valid, w, B * B))


@pytest.mark.parametrize("k", [0, 4])
def test_pieces_of_the_vocabulary(device, k):
    """So many rows and tokens that the logits' gradient comes in two pieces: dx sums over both, dhead's rows come from each,
    entries lie in both."""
    n, v, valid, d = 8200, 66000, 65990, 64
    x, head, w, g = inputs(device, n, v, d, 20 + k)
    if k:
        ids, vals = teacher(n, k, valid, g, device)
        out = head_loss.distill_loss_grads(x, head, vals, ids, w, valid=valid)
    else:
        ids, vals = torch.randint(-valid // 4, valid, (n,), generator=g).to(device.torch), None
        out = head_loss.token_loss_grads(x, head, ids, w, valid=valid)
    check(f"pieces, k {k}", out, expected(x, head, ids, vals, 1.0, valid, w))


def test_offsets_past_32_bits(device):
    """A head of more than 2^32 bytes and 2^31 values: the loss against a chunked sum in 64 bits, dhead's last rows against
    the formula's."""
    n, v, d = 5, 530_003, 4096
    x, _, w, g = inputs(device, n, 8, d, 22)
    gen = torch.Generator(device=device.torch).manual_seed(23)
    head = torch.empty(v, d, dtype=torch.bfloat16, device=device.torch)
    step = 32768
    for i in range(0, v, step):
        head[i : i + step] = torch.randn(min(step, v - i), d, generator=gen, device=device.torch) * 0.05
    ids = torch.tensor([v - 1, 0, v - 3, -100, v // 2], device=device.torch)
    loss, dx, dhead = head_loss.token_loss_grads(x, head, ids, w)
    z = torch.cat([x.double() @ head[i : i + step].double().T for i in range(0, v, step)], 1)
    lse = torch.logsumexp(z, 1)
    on = ids >= 0
    want = torch.where(on, lse - z.gather(1, ids.clamp(min=0)[:, None])[:, 0], 0.0)
    ez = (d + 2) * U * (x.double().abs().sum(1) * 0.4)  # (|head| < 0.4)
    assert float(head.abs().max()) < 0.4
    within("loss", loss, want, 2 * ez + (4096 + 64) * U + 16 * U * (lse.abs() + z.abs().amax(1)) + 1e-30)
    dz = (z - lse[:, None]).exp()
    dz[torch.arange(n, device=device.torch)[on], ids[on]] -= 1
    dz = dz * torch.where(on, w.double(), 0.0)[:, None]
    ep = (3 * ez + (4096 + 64) * U + 16 * U * (lse.abs() + z.abs().amax(1)))[:, None] * (dz.abs() + 1e-12)
    for rows in (slice(0, 300), slice(v - 300, v)):
        e = ((ep + (B + 4 * U) * (dz.abs() + ep))[:, rows]).T @ x.double().abs() * 1.01
        val = dz[:, rows].T @ x.double()
        within(f"dhead rows {rows.start} ..", dhead[rows], val, e + (B + 4 * U) * (val.abs() + e) + 2.0**-133)
    val = sum(dz[:, i : i + step] @ head[i : i + step].double() for i in range(0, v, step))
    mag = sum(dz.abs()[:, i : i + step] @ head[i : i + step].double().abs() for i in range(0, v, step))
    err = sum((ep + (B + 4 * U) * (dz.abs() + ep))[:, i : i + step] @ head[i : i + step].double().abs() for i in range(0, v, step))
    e = err + (v + 64) * U * 1.01 * mag
    within("dx", dx, val, e + (B + 4 * U) * (val.abs() + e) + 2.0**-133)


def test_every_row_left_out(device):
    for n in (1, 70, 300):
        x, head, w, g = inputs(device, n, 500, 64, 5)
        x[:] = float("nan")
        w[:] = float("inf")
        loss, dx, dhead = head_loss.token_loss_grads(x, head, torch.full((n,), -1, device=device.torch), w)
        assert not loss.any() and not dx.any() and not dhead.any()
        ids = torch.full((n, 3), 500, dtype=torch.int32, device=device.torch)
        vals = torch.full((n, 3), float("nan"), device=device.torch)
        loss, dx, dhead = head_loss.distill_loss_grads(x, head, vals, ids, w)
        assert not loss.any() and not dx.any() and not dhead.any()


@pytest.mark.parametrize("n", [20, 200])
def test_rows_left_out_hold_anything(device, n):
    """NaN and infinities in rows left out, in their weights, in empty slots and in the head's rows past valid change
    nothing, bit for bit."""
    v, valid, d = 700, 650, 136
    x, head, w, g = inputs(device, n, v, d, 6)
    ids = torch.randint(0, valid, (n,), generator=g)
    out_rows = torch.rand(n, generator=g) < 0.5
    ids[out_rows] = -100
    ids, out_rows = ids.to(device.torch), out_rows.to(device.torch)
    want = head_loss.token_loss_grads(x, head, ids, w, valid=valid)
    x2, head2, w2 = x.clone(), head.clone(), w.clone()
    x2[out_rows] = float("nan")
    w2[out_rows] = float("inf")
    head2[valid:] = float("nan")
    got = head_loss.token_loss_grads(x2, head2, ids, w2, valid=valid)
    for part, a, b in zip(("loss", "dx", "dhead"), got, want):
        same(f"{n} rows: {part}", a, b)
    ti, tv = teacher(n, 6, valid, g, device)
    ti[out_rows] = -1
    tv2 = torch.where((ti < 0) | (ti >= valid), float("nan"), tv)
    want = head_loss.distill_loss_grads(x, head, tv, ti, w, valid=valid)
    got = head_loss.distill_loss_grads(x2, head2, tv2, ti, w2, valid=valid)
    for part, a, b in zip(("loss", "dx", "dhead"), got, want):
        same(f"{n} rows, a teacher: {part}", a, b)


def test_masked_vocabulary_and_extremes(device):
    """Logits of the type's lowest values and of minus infinity (a vocabulary row that x makes -inf) are probability 0; a
    logit of plus infinity or a NaN gives a NaN in its row alone."""
    n, v, d = 70, 600, 64
    x, head, w, g = inputs(device, n, v, d, 8)
    x[:, 0] = 1.0
    head[:, 0] = 0.0
    ids = torch.randint(2, v, (n,), generator=g).to(device.torch)
    clean = head_loss.token_loss(x, head, ids)
    head[0, 0] = -3e38  # (a masked entry of the vocabulary)
    head[1, 0] = -math.inf
    masked = head_loss.token_loss_grads(x, head, ids)
    z = x.double() @ head[2:].double().T
    within("masked entries", masked[0], torch.logsumexp(z, 1) - z.gather(1, ids[:, None] - 2)[:, 0],
           torch.full((n,), 1e-4, dtype=torch.float64, device=device.torch))
    assert not masked[2][:2].any() and bool(torch.isfinite(masked[2][2:]).all())
    assert not torch.equal(clean, masked[0])
    head[1, 0] = 0.0
    x[5, 0] = float("nan")
    loss = head_loss.token_loss(x, head, ids)
    assert loss.isnan().nonzero().tolist() == [[5]]


@pytest.mark.parametrize("n", [1, 40, 100, 1000])
def test_a_row_of_nan_in_the_head(device, n):
    """A NaN in one row of the head is in every row's loss, also where that row is alone in its tile."""
    x, head, w, g = inputs(device, n, 2049, 64, n)
    ids = torch.randint(0, 64, (n,), generator=g).to(device.torch)
    head[64], head[256], head[2048] = 0.0, 0.0, 0.0
    for valid in (65, 257, 2049):
        assert not head_loss.token_loss(x, head, ids, valid=valid).isnan().any()
        head[valid - 1] = float("nan")
        assert bool(head_loss.token_loss(x, head, ids, valid=valid).isnan().all()), valid
        loss, dx, _ = head_loss.token_loss_grads(x, head, ids, valid=valid)
        assert bool(loss.isnan().all()) and bool(dx.isnan().all()), valid
        head[valid - 1] = 0.0


@pytest.mark.parametrize("n", [20, 700])
def test_teacher_of_lowest_values(device, n):
    """The type's lowest value, at a temperature that takes it past float32, is an entry of probability 0, and a row of
    nothing else one of equal probabilities: bit by bit what the same entries give with a value of little and of 0."""
    x, head, w, g = inputs(device, n, 500, 64, n)
    ids, vals = teacher(n, 8, 500, g, device, empty=False)
    plain = vals.clone()
    low = torch.rand(n, 8, generator=g).to(device.torch) < 0.5
    low[:, 0], low[3], low[n - 1] = False, True, True
    vals[low], plain[low] = torch.finfo(torch.float32).min, -200.0  # (exp(-200 / 0.5) is 0 in float32 and below any bound)
    plain[3] = plain[n - 1] = 0.0
    want = head_loss.distill_loss_grads(x, head, plain, ids, w, temperature=0.5)
    check(f"lowest values, {n} rows", want, expected(x, head, ids, plain, 0.5, 500, w))
    for part, a, b in zip(("loss", "dx", "dhead"), head_loss.distill_loss_grads(x, head, vals, ids, w, temperature=0.5), want):
        same(part, a, b)


def test_weights(device):
    """Weights of zero, and of both signs and far apart; an infinite one or a NaN stays in its row's dx."""
    n, v, d = 40, 300, 64
    x, head, w, g = inputs(device, n, v, d, 30)
    ids = torch.randint(0, v, (n,), generator=g).to(device.torch)
    zero = head_loss.token_loss_grads(x, head, ids, torch.zeros_like(w))
    assert not zero[1].any() and not zero[2].any() and bool((zero[0] > 0).all())
    signs = (w - 0.5) * 10.0 ** torch.arange(-20, 20, device=device.torch)
    out = head_loss.token_loss_grads(x, head, ids, signs)
    check("weights far apart", (None, out[1], out[2]), expected(x, head, ids, None, 1.0, v, signs))
    w = w / w.max()
    want = head_loss.token_loss_grads(x, head, ids, w)[1]
    top = int(w.argmax())
    for bad in (float("inf"), float("nan")):
        odd = w.clone()
        odd[(top + 1) % n] = bad
        got = head_loss.token_loss_grads(x, head, ids, odd)[1]
        rest = torch.arange(n, device=device.torch) != (top + 1) % n
        same(f"rows beside a weight of {bad}", got[rest], want[rest])
        assert not torch.isfinite(got[(top + 1) % n]).all()


@pytest.mark.parametrize("n", [7, 90])
def test_layouts(device, n):
    """x as a view with a longer row, off its alignment, transposed, of rank 4; targets of any shape; the head of rank 4."""
    v, d = 900, 80
    x, head, w, g = inputs(device, n, v, d, 9)
    ids = torch.randint(0, v, (n,), generator=g).to(device.torch)
    want = head_loss.token_loss_grads(x, head, ids, w)
    wide = inputs(device, n, v, d, 9, ld=96)[0]
    odd = torch.empty(n * d + 1, dtype=torch.bfloat16, device=device.torch)[1:].view(n, d).copy_(x)
    for what, view in (("a longer row", wide), ("off its alignment", odd), ("transposed", x.t().contiguous().t()),
                       ("expanded", x[:1].expand(n, d))):
        got = head_loss.token_loss_grads(view, head, ids, w)
        ref = want if what != "expanded" else head_loss.token_loss_grads(x[:1].repeat(n, 1), head, ids, w)
        for part, a, b in zip(("loss", "dx", "dhead"), got, ref):
            same(f"{what}: {part}", a, b)
    got = head_loss.token_loss_grads(x.reshape(1, 1, n, d), head.reshape(1, 1, v, d), ids.reshape(1, n), w.reshape(1, n))
    assert got[0].shape == (1, n) and got[1].shape == (1, 1, n, d) and got[2].shape == (1, 1, v, d)
    for a, b in zip(got, want):
        same("rank 4", a.reshape(b.shape), b)
    for g1 in (2.0, torch.tensor(2.0, device=device.torch), torch.full((n,), 2.0, dtype=torch.float64, device=device.torch), None):
        a = head_loss.token_loss_grads(x, head, ids, g1)
        b = head_loss.token_loss_grads(x, head, ids, torch.full((n,), 1.0 if g1 is None else 2.0, device=device.torch))
        same("one weight for all", a[2], b[2])


def test_no_rows(device):
    x, head, _, _ = inputs(device, 4, 300, 64, 10)
    loss, dx, dhead = head_loss.token_loss_grads(x[:0], head, torch.empty(0, dtype=torch.int64, device=device.torch))
    assert loss.shape == (0,) and dx.shape == (0, 64) and not dhead.any()
    vals = torch.empty(0, 3, device=device.torch)
    assert head_loss.distill_loss(x[:0], head, vals, vals.int()).shape == (0,)


def test_autograd(device):
    """backward() through a mean with a few rows left out: the gradients of the calls that give them at once; leaves that
    ask for none get none; the second backward adds up."""
    n, v, d = 50, 600, 64
    x, head, _, g = inputs(device, n, v, d, 11)
    ids = torch.randint(-20, v, (n,), generator=g).to(device.torch)
    ti, tv = teacher(n, 4, v, g, device)
    xl, hl = x.clone().requires_grad_(), head.clone().requires_grad_()
    loss = head_loss.token_loss(xl, hl, ids)
    loss.mean().backward()
    want = head_loss.token_loss_grads(x, head, ids, 1.0 / n)
    same("dx", xl.grad, want[1])
    same("dhead", hl.grad, want[2])
    head_loss.distill_loss(xl, hl, tv, ti, temperature=2.0).sum().backward()
    more = head_loss.distill_loss_grads(x, head, tv, ti, temperature=2.0)
    same("dx, added up", xl.grad, want[1] + more[1])
    same("dhead, added up", hl.grad, want[2] + more[2])
    frozen = x.clone().requires_grad_()
    head_loss.token_loss(frozen, head, ids).sum().backward()
    same("a frozen head", frozen.grad, head_loss.token_loss_grads(x, head, ids)[1])
    assert not head_loss.token_loss(x, head, ids).requires_grad


def test_gradients_against_differences(device):
    """Along random directions, the gradients' slope against central differences of the loss's definition in 64 bits: off by
    the gradients' own bounds and the differences' (h^2 / 6 times the third derivative, of the order of |change of z|^3)."""
    n, v, d, k, t = 12, 200, 64, 3, 1.5
    x, head, w, g = inputs(device, n, v, d, 12)
    ti, tv = teacher(n, k, v, g, device)
    got = head_loss.distill_loss_grads(x, head, tv, ti, w, temperature=t)
    want = expected(x, head, ti, tv, t, v, w)
    ids, q, on, ent = entries(ti, tv, v, t)

    def f(xx, hh):
        z = xx @ hh.T / t
        lp = torch.log_softmax(z, 1)
        return (w.double() * torch.where(on, -(q * lp.gather(1, ids)).sum(1) + ent, 0.0)).sum()

    h = 1e-4
    for which in (1, 2):
        dirn = torch.randn(got[which].shape, generator=g).double().to(device.torch)
        dx, dh = (dirn, torch.zeros_like(head).double()) if which == 1 else (torch.zeros_like(x).double(), dirn)
        slope = (f(x.double() + h * dx, head.double() + h * dh) - f(x.double() - h * dx, head.double() - h * dh)) / (2 * h)
        mine = (got[which].double() * dirn).sum()
        change = ((dx @ head.double().T + x.double() @ dh.T) / t).abs().amax(1)
        slack = (want[which][1] * dirn.abs()).sum() + h * h * (w.double() * 8 * change**3).sum() + 1e-9
        assert abs(mine - slope) <= slack, (which, mine, slope, slack)


@pytest.mark.parametrize("n, v, d", [(200, 1500, 136), (600, 3000, 136), (600, 3000, 776)])
def test_repeats_streams_and_graphs(device, n, v, d):
    """The same call twice, on another stream, and replayed in two graphs with eager work between: bit for bit."""
    x, head, w, g = inputs(device, n, v, d, 13)
    ids = torch.randint(-100, v, (n,), generator=g).to(device.torch)
    ti, tv = teacher(n, 8, v, g, device)
    calls = [lambda: head_loss.token_loss_grads(x, head, ids, w),
             lambda: head_loss.distill_loss_grads(x, head, tv, ti, w, temperature=2.0)]
    want = [[t.clone() for t in c()] for c in calls]
    for c, r in zip(calls, want):
        for a, b in zip(c(), r):
            same("again", a, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = [c() for c in calls]
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(c())
        graphs.append(graph)
    for rep in range(3):
        for o in outs:
            for t in o:
                t.fill_(7)
        for graph in graphs:
            graph.replay()
        eager = calls[0]()
        torch.cuda.synchronize()
        for got in (outs, [eager, want[1]], other):
            for r, o in zip(want, got):
                for a, b in zip(o, r):
                    same(f"replay {rep}", a, b)
    # new inputs in the captured tensors: the rows that count are found anew
    ids.copy_(torch.randint(-100, v, (n,), generator=g))
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(outs[0], calls[0]()):
        same("a replay on other targets", a, b)


def test_backward_refuses_capture(device):
    x, head, _, g = inputs(device, 30, 300, 64, 14)
    ids = torch.randint(0, 300, (30,), generator=g).to(device.torch)
    xl = x.clone().requires_grad_()
    head_loss.token_loss(xl, head, ids).sum().backward()  # (an eager graph of the leaf first)
    torch.cuda.synchronize()

    def captured():
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            head_loss.token_loss(xl, head, ids).sum().backward()

    raises("backward under capture", RuntimeError, captured)
    torch.cuda.synchronize()
    same("and the next call runs", head_loss.token_loss(x, head, ids), head_loss.token_loss(xl, head, ids).detach())


def test_refusals(device):
    x, head, w, g = inputs(device, 10, 300, 64, 15)
    ids = torch.zeros(10, dtype=torch.int64, device=device.torch)
    vals, ti = torch.zeros(10, 3, device=device.torch), torch.zeros(10, 3, dtype=torch.int32, device=device.torch)
    T, D = head_loss.token_loss_grads, head_loss.distill_loss_grads
    for name, fn in (
        ("float32 x", lambda: T(x.float(), head, ids)),
        ("float32 head", lambda: T(x, head.float(), ids)),
        ("another dim", lambda: T(x[:, :56], head, ids)),
        ("dim not a multiple of 8", lambda: T(x[:, :60], head[:, :60].contiguous(), ids)),
        ("a head that is not contiguous", lambda: T(x, head[::2], ids)),
        ("too few targets", lambda: T(x, head, ids[:9])),
        ("float targets", lambda: T(x, head, ids.float())),
        ("host targets", lambda: T(x, head, ids.cpu())),
        ("valid 0", lambda: T(x, head, ids, valid=0)),
        ("valid past the head", lambda: T(x, head, ids, valid=301)),
        ("weights of another count", lambda: T(x, head, ids, w[:3])),
        ("int64 teacher ids", lambda: D(x, head, vals, ti.long())),
        ("bf16 teacher values", lambda: D(x, head, vals.bfloat16(), ti)),
        ("entries of another shape", lambda: D(x, head, vals[:, :2], ti)),
        ("too many entries", lambda: D(x, head, vals.repeat(1, 22), ti.repeat(1, 22))),
        ("no entries", lambda: D(x, head, vals[:, :0], ti[:, :0])),
        ("temperature 0", lambda: D(x, head, vals, ti, temperature=0.0)),
        ("temperature NaN", lambda: D(x, head, vals, ti, temperature=float("nan"))),
    ):
        raises(name, AssertionError, fn)
    odd = torch.empty(300 * 64 + 1, dtype=torch.bfloat16, device=device.torch)[1:].view(300, 64)
    raises("a head off its alignment", ValueError, lambda: T(x, odd, ids))


def test_a_training_step(device):
    """The pieces as a program uses them together: a teacher head's records merged into its best logits, a student's head
    distilled from them and scored on tokens, the router's picks and their balance loss, one backward over the sum."""
    rows, dim, vocab, k = 12, 256, 2048, 8
    g = torch.Generator().manual_seed(16)
    tw = (torch.randn(vocab, dim, generator=g) * 0.05).to(torch.bfloat16)
    x = torch.randn(rows, dim, generator=g).to(torch.bfloat16).to(device.torch)
    th = lmhead.DeviceHead(device, tw, fmt="bf16", chunks=2, k=k, rescore=False)
    records = th.logits_topk(x.reshape(1, 1, rows, dim), rows)
    vals, ids = linear.topk_merge(records, rows, k, k_out=16)
    th.deallocate()
    student = head_pick.head_rows(device, tw.float() + torch.randn(vocab, dim, generator=g) * 0.02).requires_grad_()
    xl = x.clone().requires_grad_()
    targets = torch.randint(-200, vocab, (rows,), generator=g).to(device.torch)
    router = torch.randn(64, dim, generator=g).to(device.torch).requires_grad_()
    logits = (xl.float() @ router.T * 0.1).reshape(1, 1, rows, 64)
    picks = torch.empty(1, 1, rows, 4, dtype=torch.int16, device=device.torch)
    w = torch.empty(1, 1, rows, 4, dtype=torch.bfloat16, device=device.torch)
    moe8.route(logits.detach(), picks, w, 4)
    bal, counts = balance.balance_loss(logits, picks, 4)
    assert int(counts.sum()) == 4 * rows
    total = (head_loss.distill_loss(xl, student, vals, ids, temperature=2.0).mean()
             + head_loss.token_loss(xl, student, targets).mean() + 0.01 * bal.sum())
    total.backward()
    kd = head_loss.distill_loss_grads(x, student.detach(), vals, ids, 1.0 / rows, temperature=2.0)
    ce = head_loss.token_loss_grads(x, student.detach(), targets, 1.0 / rows)
    same("the head's gradient", student.grad, kd[2] + ce[2])
    dl = balance.balance_loss_grads(logits.detach(), picks, 4, 0.01)[2]
    # (the step's total is exact sums of these but for the router's products, torch's own)
    within("the router's gradient", router.grad, dl.reshape(rows, 64).double().T @ (x.double() * 0.1),
           1e-5 * (dl.reshape(rows, 64).abs().double().T @ (x.abs().double() * 0.1)) + 1e-12)
    assert bool(torch.isfinite(xl.grad).all()) and bool(xl.grad.any())
