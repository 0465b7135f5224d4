"""Calls of the losses (lm_head_topk/head_loss.py, moe/balance.py) that a program makes and their operators' own tests do not.
Most compare two calls that mean the same, bit for bit."""

import math

import pytest
import torch
from torch.autograd import forward_ad

from common.testing import raises, same
from dense_reader import linear
from lm_head_topk import head_loss, lmhead
from moe import balance, moe8

pytestmark = pytest.mark.gpu


def head_inputs(device, n, v, d, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g).to(torch.bfloat16).to(device.torch)
    head = (torch.randn(v, d, generator=g) * 0.1).to(torch.bfloat16).to(device.torch)
    return x, head, torch.rand(n, generator=g).to(device.torch) + 0.25, g


def teacher(n, k, v, g, device):
    ids = torch.randint(0, v, (n, k), generator=g).int()
    vals = torch.randn(n, k, generator=g) * 3
    vals[torch.rand(n, k, generator=g) < 0.1] = -math.inf
    return ids.to(device.torch), vals.to(device.torch)


def router_inputs(device, batch, rows, width, experts, k, seed):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(batch, rows, width, generator=g) * 2).to(device.torch)
    ids = torch.randint(0, experts + 2, (batch, rows, k), generator=g).to(torch.int16).to(device.torch)
    mask = (torch.rand(batch, rows, generator=g) < 0.7).to(device.torch)
    return logits, ids, mask, (torch.rand(batch, generator=g) + 0.5).to(device.torch)


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
def test_two_layers_share_an_ids_buffer(device, kind):
    """Two layers route into one ids buffer before one backward: each layer's gradient is that of its own picks."""
    g = torch.Generator().manual_seed(1)
    layers = [torch.randn(1, 1, 32, 64, generator=g).to(device.torch).requires_grad_() for _ in range(2)]
    ids = torch.empty(1, 1, 32, 4, dtype=torch.int16, device=device.torch)
    w = torch.empty(1, 1, 32, 4, dtype=torch.bfloat16, device=device.torch)
    total, want = 0.0, []
    for logits in layers:
        moe8.route(logits.detach(), ids, w, 4, kind=kind)
        want.append(balance.balance_loss_grads(logits.detach(), ids, 4, kind=kind)[2])
        total = total + balance.balance_loss(logits, ids, 4, kind=kind)[0].sum()
    total.backward()
    for i, logits in enumerate(layers):
        same(f"layer {i}", logits.grad, want[i])


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("batch, rows, width, experts, k", [
    (1, 1, 1, 1, 1), (1, 64, 32, 32, 4), (1, 65, 32, 32, 4), (3, 100, 130, 97, 2), (300, 40, 41, 40, 4), (2, 70, 600, 513, 16),
    (1, 5000, 128, 128, 4), (1, 8200, 256, 250, 6), (1, 600, 1030, 1000, 8),
])
def test_balance_backward_is_the_one_call(device, kind, batch, rows, width, experts, k):
    """backward() after the ids and the counts were written over: the gradient of the call that gives all at once, by one
    workgroup a batch, by many, and where their sums take a launch of their own."""
    logits, ids, mask, g = router_inputs(device, batch, rows, width, experts, k, batch + rows)
    for m in (None, mask):
        want = balance.balance_loss_grads(logits, ids, k, g, kind=kind, experts=experts, mask=m)
        leaf, mine = logits.clone().requires_grad_(), ids.clone()
        loss, counts = balance.balance_loss(leaf, mine, k, kind=kind, experts=experts, mask=m)
        same("loss", loss.detach(), want[0])
        same("counts", counts, want[1])
        mine.fill_(0), counts.add_(1)
        (loss * g).sum().backward()
        same(f"{kind} {batch} x {rows} x {experts} of {width}", leaf.grad, want[2])


def test_inputs_that_the_library_writes_again(device):
    """What the library writes into a caller's tensor counts for autograd as a change of it: a backward that would read the
    new values where the forward read the old ones is refused."""
    n, d, v = 8, 256, 512
    x, head, _, g = head_inputs(device, n, v, d, 2)
    w, _ = linear.native_weight(device, torch.randn(d, d, generator=g) * 0.1, linear.bfloat8_b)
    buf = torch.empty(1, 1, n, d, dtype=torch.bfloat16, device=device.torch)
    ids = torch.randint(0, v, (n,), generator=g).to(device.torch)
    leaf = head.clone().requires_grad_()
    linear.matmul(x.reshape(1, 1, n, d), w, None, out=buf)
    loss = head_loss.token_loss(buf, leaf, ids)
    loss.sum().backward()  # (nothing in between)
    same("nothing written", leaf.grad, head_loss.token_loss_grads(buf, head, ids)[2])
    loss = head_loss.token_loss(buf, leaf, ids)
    linear.matmul(x.reshape(1, 1, n, d) * 2, w, None, out=buf)
    raises("x written by a matmul", RuntimeError, lambda: loss.sum().backward())

    slots = torch.zeros(1, 1, n, 4, dtype=torch.int16, device=device.torch)
    weights = torch.ones(1, 1, n, 4, dtype=torch.bfloat16, device=device.torch)
    y = (weights.clone().requires_grad_() * weights).sum()
    moe8.route(torch.randn(1, 1, n, 64, generator=g).to(device.torch), slots, weights, 4)
    raises("weights written by the router", RuntimeError, y.backward)

    token = torch.zeros(1, dtype=torch.int32, device=device.torch)
    one = x[:1].reshape(1, 1, 1, d)
    for rescore in (True, False):
        th = lmhead.DeviceHead(device, head.cpu(), fmt="bf16", chunks=1, k=8, rescore=rescore, device_pick=True)
        th.logits_topk(one, 1, ids_out=token)
        for what, t in (("page", th.picks[1][0, 0, :1, 0]), ("token", token)):
            loss = head_loss.token_loss(x[:1], leaf, t)
            th.logits_topk(one, 1, ids_out=token)
            raises(f"a {what} written by the pick, rescore {rescore}", RuntimeError, lambda: loss.sum().backward())
        th.deallocate()


def test_forward_mode_is_refused(device):
    """A dual tensor's tangent has no rule here: an error, never a loss without it."""
    x, head, w, g = head_inputs(device, 6, 100, 64, 3)
    ids = torch.randint(0, 100, (6,), generator=g).to(device.torch)
    ti, tv = teacher(6, 3, 100, g, device)
    logits, slots, mask, gb = router_inputs(device, 2, 10, 32, 32, 4, 3)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for name, fn in (
            ("x", lambda: head_loss.token_loss(dual(x), head, ids)),
            ("the head", lambda: head_loss.token_loss(x, dual(head), ids)),
            ("x that needs a gradient too", lambda: head_loss.token_loss(dual(x.clone().requires_grad_()), head, ids)),
            ("x of both at once", lambda: head_loss.token_loss_grads(dual(x), head, ids)),
            ("weights", lambda: head_loss.token_loss_grads(x, head, ids, dual(w))),
            ("a teacher's values", lambda: head_loss.distill_loss(x, head, dual(tv), ti)),
            ("a teacher's values, both at once", lambda: head_loss.distill_loss_grads(x, head, dual(tv), ti)),
            ("logits", lambda: balance.balance_loss(dual(logits), slots, 4)),
            ("logits of both at once", lambda: balance.balance_loss_grads(dual(logits), slots, 4)),
            ("weights of batches", lambda: balance.balance_loss_grads(logits, slots, 4, dual(gb))),
        ):
            raises(f"forward mode, {name}", RuntimeError, fn)
        same("nothing dual", head_loss.token_loss(x, head, ids), head_loss.token_loss_grads(x, head, ids)[0])


@pytest.mark.parametrize("n, s, d", [(8, 1024, 4096), (3, 70000, 64), (1, 1024, 4096)])
def test_rows_far_apart(device, n, s, d):
    """The last position of each of a batch's sequences, read where the whole batch lies, at any distance."""
    g = torch.Generator().manual_seed(4)
    hidden = torch.full((n, s, d), float("nan"), dtype=torch.bfloat16, device=device.torch)
    hidden[:, -1] = torch.randn(n, d, generator=g).to(device.torch)
    head = (torch.randn(300, d, generator=g) * 0.1).to(torch.bfloat16).to(device.torch)
    ids = torch.randint(0, 300, (n,), generator=g).to(device.torch)
    x = hidden[:, -1]
    want = head_loss.token_loss_grads(x.contiguous(), head, ids)
    assert n == 1 or x.stride(0) > 1 << 21
    for part, a, b in zip(("loss", "dx", "dhead"), head_loss.token_loss_grads(x, head, ids), want):
        same(part, a, b)
    leaf = x.detach().requires_grad_()
    head_loss.token_loss(leaf, head, ids).sum().backward()
    same("backward", leaf.grad, want[1])
