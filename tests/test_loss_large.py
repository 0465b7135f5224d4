"""The LM head's losses where the products take their large tiles (test_loss_calls_host.LARGE holds which): every value within
the bounds of test_head_loss.py, against 64 bits."""

import gc

import pytest
import torch
from test_head_loss import check, expected, inputs, teacher
from test_loss_calls_host import LARGE

from lm_head_topk import head_loss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n, v, valid, d, k, both", [call for call, _ in LARGE])
def test_large_tiles(device, n, v, valid, d, k, both):
    """Ragged rows, tokens and values, a few rows left out, and the sums of two pieces of the vocabulary; alone a backward makes
    its logits again."""
    x, head, w, g = inputs(device, n, v, d, n + v + d + k, spread=0.05)
    kw = dict(valid=valid)
    if k:
        ids, vals = teacher(n, k, valid, g, device)
        ids[0], vals[1] = -1, -torch.inf
        args, kw["temperature"] = (vals, ids), 1.5
    else:
        ids, vals = torch.randint(0, valid, (n,), generator=g).to(device.torch), None
        ids[0], ids[1], ids[2] = -100, valid, valid - 1
        args = (ids,)
    x[:1] = torch.nan
    if both:
        out = (head_loss.distill_loss_grads if k else head_loss.token_loss_grads)(x, head, *args, w, **kw)
    else:
        leaves = x.clone().requires_grad_(), head.clone().requires_grad_()
        loss = (head_loss.distill_loss if k else head_loss.token_loss)(*leaves, *args, **kw)
        (loss * w).sum().backward()
        out = loss.detach(), leaves[0].grad, leaves[1].grad
    check(f"{n} x {v} ({valid}) x {d}, {k} entries", out, expected(x, head, ids, vals, kw.get("temperature", 1.0), valid, w))
    gc.collect()
    torch.cuda.empty_cache()  # (the 64-bit logits)
