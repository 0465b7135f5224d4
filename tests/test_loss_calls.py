"""Calls of the losses (lm_head_topk/head_loss.py, moe/balance.py) that a program makes and their operators' own tests do not.
Most compare two calls that mean the same, bit for bit."""

import pytest
import torch

from common.testing import same
from moe import balance, moe8

pytestmark = pytest.mark.gpu


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
