"""The router's balance loss (moe/balance.py) on the GPU against its definition in 64 bits. Counts are equal; the float32
outputs are off by at most (u = 2^-24): a row's probabilities (E + 64) u relative (the exponents' arguments add |logit| u
each), their sums over rows R u more, the products with f a few u."""

import pytest
import torch

from common.testing import raises, same, within
from moe import balance, moe8

pytestmark = pytest.mark.gpu

U = 2.0**-24


def inputs(device, batch, rows, width, experts, k, seed, ids32=False, past=True):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(batch, rows, width, generator=g) * 2
    ids = torch.randint(0, experts + (2 if past else 0), (batch, rows, k), generator=g)
    mask = torch.rand(batch, rows, generator=g) < 0.7
    return (logits.to(device.torch), ids.to(torch.int32 if ids32 else torch.int16).to(device.torch), mask.to(device.torch),
            torch.rand(batch, generator=g).to(device.torch) + 0.5)


def expected(logits, ids, k, kind, experts, mask, g):
    """(loss, its bound, counts, dlogits, its bound) in 64 bits."""
    B, R, W = logits.shape
    z = logits[..., :experts].double()
    on = torch.ones(B, R, dtype=torch.bool, device=z.device) if mask is None else mask.bool()
    z = torch.where(on[..., None], z, 0.0)
    if kind == "softmax":
        p = torch.where((z != -torch.inf).any(-1, keepdim=True), torch.softmax(z, -1), 0.0)
        inner = p
    else:
        s = torch.sigmoid(z)
        p = s / s.sum(-1, keepdim=True)
        inner = p * (1 - s)
    p, inner = p * on[..., None], inner * on[..., None]
    wide = ids[..., :k].long() & (0xFFFF if ids.dtype == torch.int16 else 0xFFFFFFFF)
    one = (wide < experts) & on[..., None]
    counts = torch.zeros(B, experts, dtype=torch.int64, device=z.device)
    counts.scatter_add_(1, torch.where(one, wide, 0).reshape(B, -1), one.long().reshape(B, -1))
    f = experts * counts.double() / counts.sum(1, keepdim=True).clamp(min=1)
    rows = on.sum(1).clamp(min=1).double()
    loss = (f * p.sum(1)).sum(1) / rows
    big = torch.where(z.isfinite(), z, 0.0).abs().amax((-1, -2)) if R else torch.zeros(B)
    rel = (experts + 64 + 4 * big) * U
    mean = (p * f[:, None]).sum(-1, keepdim=True)
    d = (g.double() / rows)[:, None, None] * inner * (f[:, None] - mean)
    ed = (g.double().abs() / rows)[:, None, None] * inner * (f[:, None] + mean) * (3 * rel)[:, None, None]
    if kind == "sigmoid":  # (1 - s: off by the sigmoid's own rounding, 4 u and its argument's)
        ed += (g.double().abs() / rows)[:, None, None] * p * (f[:, None] + mean) * (8 * U + 4 * U * z.abs().clamp(max=100) * s)
    pad = torch.zeros(B, R, W - experts, dtype=torch.float64, device=z.device)
    return (loss, loss * (rel + (R + experts + 16) * U) + 1e-30, counts, torch.cat([d, pad], -1),
            torch.cat([ed, pad], -1) + 1e-37)


def check(name, got, want):
    within(f"{name}: loss", got[0].reshape(-1), want[0], want[1])
    same(f"{name}: counts", got[1].reshape(want[2].shape), want[2].int())
    if got[2] is not None:
        within(f"{name}: dlogits", got[2].reshape(want[3].shape), want[3], want[4])


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("batch, rows, width, experts, k, ids32", [
    (1, 1, 1, 1, 1, False), (1, 3, 32, 32, 4, False), (2, 33, 65, 64, 8, True), (3, 100, 130, 97, 2, False),
    (1, 5000, 128, 128, 4, False), (4, 257, 256, 256, 8, True), (2, 70, 600, 513, 16, False), (1, 40, 1024, 1024, 3, True),
])
def test_balance(device, kind, batch, rows, width, experts, k, ids32):
    logits, ids, mask, g = inputs(device, batch, rows, width, experts, k, batch + rows + width, ids32)
    for m in (None, mask):
        got = balance.balance_loss_grads(logits, ids, k, g, kind=kind, ids32=ids32, experts=experts, mask=m)
        check(f"{kind} {batch} x {rows} x {experts} of {width}", got, expected(logits, ids, k, kind, experts, m, g))
        loss, counts = balance.balance_loss(logits, ids, k, kind=kind, ids32=ids32, experts=experts, mask=m)
        same("the loss alone", loss, got[0])
        same("the counts alone", counts, got[1])


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("batch, rows, width, experts, k", [
    (300, 100, 41, 40, 4), (257, 33, 260, 257, 2), (1, 64, 32, 32, 4), (1, 65, 32, 32, 4), (2, 16, 512, 512, 8),
    (2, 17, 512, 512, 8), (1, 600, 1030, 1000, 8), (3, 700, 512, 500, 4), (1, 8200, 256, 250, 6),
])
def test_many_workgroups_and_one(device, kind, batch, rows, width, experts, k):
    """Many batches, as many rows as one workgroup takes and one more, and sums that a launch of its own joins."""
    logits, ids, mask, g = inputs(device, batch, rows, width, experts, k, batch + rows + width)
    mask[0] = False
    got = balance.balance_loss_grads(logits, ids, k, g, kind=kind, experts=experts, mask=mask)
    check(f"{kind} {batch} x {rows} x {experts}", got, expected(logits, ids, k, kind, experts, mask, g))
    loss, counts = balance.balance_loss(logits, ids, k, kind=kind, experts=experts, mask=mask)
    same("the loss alone", loss, got[0])
    same("the counts alone", counts, got[1])


def test_first_slots_of_wider_ids(device):
    """Of ids with more slots a row than k (a shared expert's slot behind the picks, say), the first k count."""
    logits, ids, mask, g = inputs(device, 2, 60, 64, 64, 5, 7, ids32=True)
    got = balance.balance_loss_grads(logits, ids, 4, g, ids32=True, mask=mask)
    check("the first four of five", got, expected(logits, ids, 4, "softmax", 64, mask, g))
    for a, b in zip(got, balance.balance_loss_grads(logits, ids[..., :4].contiguous(), 4, g, ids32=True, mask=mask)):
        same("the four alone", a, b)


def test_rows_that_do_not_count(device):
    """Whatever rows that do not count hold changes nothing; a batch of none gives zeros; so do ids that choose none."""
    logits, ids, mask, g = inputs(device, 3, 50, 64, 64, 4, 1)
    mask[1] = False
    want = balance.balance_loss_grads(logits, ids, 4, g, mask=mask)
    logits2, ids2 = logits.clone(), ids.clone()
    logits2[~mask], ids2[~mask] = float("nan"), -1
    for a, b in zip(balance.balance_loss_grads(logits2, ids2, 4, g, mask=mask.to(torch.uint8)), want):
        same("rows that do not count", a, b)
    assert want[0][1] == 0 and not want[1][1].any() and not want[2][1].any() and not want[2][~mask].any()
    none = balance.balance_loss_grads(logits, torch.full_like(ids, 64), 4, g)
    assert not none[0].any() and not none[1].any() and not none[2].any()


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
def test_extreme_logits(device, kind):
    """The type's lowest value and minus infinity are probability 0 (a row of nothing else: none at all, or by sigmoid
    none), large ones do not overflow; a NaN stays in its batch."""
    logits, ids, _, g = inputs(device, 2, 40, 32, 32, 4, 2, past=False)
    logits[0, :, 3] = torch.finfo(torch.float32).min
    logits[0, :, 5] = -torch.inf
    logits[0, 7] = 80.0
    logits[1, 9] = -torch.inf if kind == "softmax" else -30.0
    got = balance.balance_loss_grads(logits, ids, 4, g, kind=kind)
    check(f"extreme {kind}", got, expected(logits, ids, 4, kind, 32, None, g))
    logits[1, 0, 0] = float("nan")
    bad = balance.balance_loss(logits, ids, 4, kind=kind)[0]
    assert bad[1].isnan() and torch.equal(bad[0], got[0][0])


def test_gradients_of_large_sigmoids(device):
    """Where the sigmoid nears 1, its slope keeps float32's accuracy: off by its own roundings alone."""
    logits, ids, mask, g = inputs(device, 2, 40, 32, 32, 4, 8)
    logits = logits.abs() + 10
    logits[0, 3, 5], logits[1, 4, 6] = 100.0, -torch.inf
    loss, eloss, counts, d, _ = expected(logits, ids, 4, "sigmoid", 32, mask, g)
    got = balance.balance_loss_grads(logits, ids, 4, g, kind="sigmoid", mask=mask)
    s = torch.sigmoid(logits.double())
    down = torch.sigmoid(-logits.double())
    f = (32 * counts.double() / counts.sum(1, keepdim=True))[:, None]
    p = s / s.sum(-1, keepdim=True)
    rows = mask.sum(1).double()[:, None, None]
    scale = g.double()[:, None, None] / rows * mask[..., None]
    mean = (p * f).sum(-1, keepdim=True)
    # (the exponent's argument |z| u, and what rel and expected's bounds count)
    rel = 3 * (32 + 64 + 4 * logits[logits.isfinite()].double().abs().amax()) * U
    within("dlogits", got[2], scale * p * down * (f - mean), scale * p * down * (f + mean) * rel + 1e-37)


def test_shapes_autograd_and_differences(device):
    logits, ids, mask, g = inputs(device, 1, 30, 96, 96, 4, 3)
    flat = logits[0].clone().requires_grad_()
    loss, counts = balance.balance_loss(flat, ids[0], 4, mask=mask[0])
    assert loss.shape == () and counts.shape == (96,) and not counts.requires_grad
    (3 * loss).backward()
    want = balance.balance_loss_grads(logits, ids, 4, 3.0, mask=mask)
    same("backward", flat.grad, want[2][0])
    four = balance.balance_loss_grads(logits.reshape(1, 1, 30, 96), ids, 4, 3.0, mask=mask)
    assert four[0].shape == (1, 1) and four[1].shape == (1, 1, 96) and four[2].shape == (1, 1, 30, 96)
    strided = torch.empty(1, 30, 100, device=device.torch)[..., :96].copy_(logits)
    same("a view", balance.balance_loss_grads(strided, ids, 4, 3.0, mask=mask)[2], want[2])
    dirn = torch.randn(logits.shape, generator=torch.Generator().manual_seed(4)).to(device.torch).double()
    h = 1e-4
    one = torch.ones(1, device=device.torch)
    for kind in ("softmax", "sigmoid"):
        d, e = expected(logits, ids, 4, kind, 96, mask, one)[3:]
        up, dn = (expected(logits.double() + s * h * dirn, ids, 4, kind, 96, mask, one)[0] for s in (1, -1))
        mine = balance.balance_loss_grads(logits, ids, 4, kind=kind, mask=mask)[2].double()
        # (the third derivative of a mean of softmaxes weighted by f: at most 8 max f |direction|^3)
        slack = (e * dirn.abs()).sum() + h * h * 8 * 96 * dirn.abs().amax() ** 3 + 1e-10
        assert abs((mine * dirn).sum() - (up - dn).sum() / (2 * h)) <= slack, kind


def test_with_the_router(device):
    """route's picks, eager and captured together with the loss; each replay on the logits of the moment."""
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(1, 1, 32, 64, generator=g).to(device.torch)
    ids = torch.empty(1, 1, 32, 8, dtype=torch.int16, device=device.torch)
    w = torch.empty(1, 1, 32, 8, dtype=torch.bfloat16, device=device.torch)

    def step():
        moe8.route(logits, ids, w, 8, kind="sigmoid")
        return balance.balance_loss_grads(logits, ids, 8, kind="sigmoid")

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        logits.copy_(torch.randn(1, 1, 32, 64, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            same(f"replay {rep}", a, b)
        want = expected(logits[0], ids[0], 8, "sigmoid", 64, None, torch.ones(1, device=device.torch))
        check(f"replay {rep}", got, want)


def test_refusals(device):
    logits, ids, mask, g = inputs(device, 2, 10, 32, 32, 4, 6)
    F = balance.balance_loss_grads
    for name, fn in (
        ("bf16 logits", lambda: F(logits.bfloat16(), ids, 4)),
        ("rank 1", lambda: F(logits[0, 0], ids[0, 0], 4)),
        ("ids of another type", lambda: F(logits, ids.long(), 4)),
        ("ids32 with 16-bit ids", lambda: F(logits, ids, 4, ids32=True)),
        ("ids that are not contiguous", lambda: F(logits, ids[..., ::2], 2)),
        ("too few slots", lambda: F(logits, ids, 5)),
        ("too few ids", lambda: F(logits, ids[:1], 4)),
        ("no slots", lambda: F(logits, ids, 0)),
        ("experts past the logits", lambda: F(logits, ids, 4, experts=33)),
        ("no experts", lambda: F(logits, ids, 4, experts=0)),
        ("kind", lambda: F(logits, ids, 4, kind="relu")),
        ("mask of another size", lambda: F(logits, ids, 4, mask=mask[:1])),
        ("float mask", lambda: F(logits, ids, 4, mask=mask.float())),
        ("weights of another count", lambda: F(logits, ids, 4, torch.ones(3, device=device.torch))),
        ("host ids", lambda: F(logits, ids.cpu(), 4)),
    ):
        raises(name, AssertionError, fn)
