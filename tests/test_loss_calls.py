"""Calls of the losses (lm_head_topk/head_loss.py, moe/balance.py) that a program makes and their operators' own tests do not.
Most compare two calls that mean the same, bit for bit."""

import ctypes
import math
import threading

import pytest
import torch
from torch.autograd import forward_ad

from common import device as cdev
from common.testing import raises, same
from dense_reader import _lib, linear
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


def test_one_row_is_read_where_it_lies(device):
    """The last position of one sequence takes no copy, whatever its batch's stride."""
    x, head, _, g = head_inputs(device, 1, 300, 64, 7)
    ids = torch.zeros(1, dtype=torch.int64, device=device.torch)
    want = head_loss.token_loss(x, head, ids)
    for stride in (1, 12, 1 << 22):
        view = x.as_strided((1, 64), (stride, 1))
        assert head_loss._Call(view, head, ids, None, 1.0, None).x.data_ptr() == x.data_ptr(), stride
        same(f"stride {stride}", head_loss.token_loss(view, head, ids), want)


def laid(t, ld, fill):
    """t's rows ld apart, what lies between them filled: (the memory, a check that it still holds that)."""
    wide = torch.full((t.shape[0], ld), fill, dtype=t.dtype, device=t.device)
    wide[:, : t.shape[1]] = t
    gap = wide[:, t.shape[1] :].clone()

    def untouched(what):
        got = wide[:, t.shape[1] :]
        assert torch.equal(torch.nan_to_num(got.double(), 3.0), torch.nan_to_num(gap.double(), 3.0)), f"{what}: between its rows"

    return wide, untouched


@pytest.mark.parametrize("n, v, valid, d, k", [
    (5, 300, 299, 64, 0), (40, 900, 890, 136, 0), (300, 2100, 2100, 264, 0), (1100, 5000, 4999, 800, 0),
    (5, 300, 299, 64, 3), (40, 900, 890, 136, 16), (300, 2100, 2100, 264, 5), (1100, 5000, 4999, 800, 2),
])
def test_head_loss_rows_at_any_distance(device, n, v, valid, d, k):
    """Every operand of the C entry with rows further apart than they are long: what the packed ones give, alone and with the
    gradients, and nothing between the rows is read into a sum or written."""
    x, head, g, gen = head_inputs(device, n, v, d, n + k)
    if k:
        ids, vals = teacher(n, k, valid, gen, device)
    else:
        ids, vals = torch.randint(-20, valid, (n, 1), generator=gen).to(device.torch), None
    m = max(1, k)
    lib, dt = _lib.lib(), device.torch
    wx, _ = laid(x, d + 24, math.nan)
    wh, _ = laid(head, d + 8, math.nan)
    wi, _ = laid(ids, m + 3, 1)  # (a token of the vocabulary: read as a row's target it would change the loss)
    wv, _ = laid(vals, m + 2, 100.0) if k else (None, None)

    def call(what, far):
        loss, lse, logits = torch.empty(n, device=dt), torch.empty(n, device=dt), torch.empty(n, m, device=dt)
        dx, dxu = laid(torch.full((n, d), 7.0, dtype=torch.bfloat16, device=dt), d + 16 if far else d, 7.0)
        dh, dhu = laid(torch.full((v, d), 7.0, dtype=torch.bfloat16, device=dt), d + 32 if far else d, 7.0)
        X, H, I, V = (wx, wh, wi, wv) if far else (x, head, ids, vals)
        A = _lib.HeadLoss()
        A.x, A.ldx, A.head, A.ld_head = X.data_ptr(), X.stride(0), H.data_ptr(), H.stride(0)
        A.rows, A.dim, A.vocab, A.valid = n, d, v, valid
        A.ids, A.ld_ids, A.ids64, A.k = I.data_ptr(), I.stride(0), int(I.dtype == torch.int64), m
        if k:
            A.vals, A.ld_vals = V.data_ptr(), V.stride(0)
        A.temperature = 1.0
        A.loss, A.lse, A.logits, A.g = loss.data_ptr(), lse.data_ptr(), logits.data_ptr(), g.data_ptr()
        if what & _lib.DR_LOSS_BACKWARD:
            A.dx, A.ld_dx, A.dhead, A.ld_dhead = dx.data_ptr(), dx.stride(0), dh.data_ptr(), dh.stride(0)
        need = lib.dr_head_loss_workspace_bytes(ctypes.byref(A), what)
        assert need > 0
        ws = torch.empty(need, dtype=torch.uint8, device=dt)
        A.workspace, A.workspace_bytes, A.stream = ws.data_ptr(), need, cdev.raw_stream(dt)
        assert lib.dr_head_loss_run(ctypes.byref(A), what) == _lib.DR_OK
        torch.cuda.synchronize()
        dxu("dx"), dhu("dhead")
        return loss, lse, logits, dx[:, :d], dh[:, :d]

    for what in (_lib.DR_LOSS_FORWARD, _lib.DR_LOSS_FORWARD | _lib.DR_LOSS_BACKWARD):
        for part, a, b in zip(("loss", "lse", "logits", "dx", "dhead"), call(what, True), call(what, False)):
            same(f"{what}: {part}", a, b)


@pytest.mark.parametrize("batch, rows, width, experts, k", [(2, 33, 70, 64, 4), (1, 3000, 128, 100, 8), (1, 600, 1030, 1000, 3)])
def test_balance_rows_at_any_distance(device, batch, rows, width, experts, k):
    logits, ids, mask, g = router_inputs(device, batch, rows, width, experts, k, rows)
    want = balance.balance_loss_grads(logits, ids, k, g, experts=experts, mask=mask)
    dt = device.torch
    for more in (1, 4):
        wl, _ = laid(logits.reshape(-1, width), width + more, math.nan)
        wi, _ = laid(ids.reshape(-1, k), k + 3, 1)
        d, untouched = laid(torch.full((batch * rows, width), 7.0, device=dt), width + more, 7.0)
        loss, counts = torch.empty(batch, device=dt), torch.empty(batch, experts, dtype=torch.int32, device=dt)
        A = _lib.Balance()
        A.logits, A.ld_logits, A.batch, A.rows, A.experts, A.width = wl.data_ptr(), width + more, batch, rows, experts, width
        A.ids, A.ld_ids, A.k, A.mask = wi.data_ptr(), k + 3, k, mask.data_ptr()
        A.loss, A.counts, A.g, A.dlogits, A.ld_dlogits = loss.data_ptr(), counts.data_ptr(), g.data_ptr(), d.data_ptr(), width + more
        need = _lib.lib().dr_moe_balance_workspace_bytes(ctypes.byref(A), _lib.DR_BALANCE_GRAD)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dt)
        A.workspace, A.workspace_bytes, A.stream = ws.data_ptr(), need, cdev.raw_stream(dt)
        assert _lib.lib().dr_moe_balance(ctypes.byref(A), _lib.DR_BALANCE_GRAD) == _lib.DR_OK
        torch.cuda.synchronize()
        untouched("dlogits")
        same("loss", loss, want[0])
        same("counts", counts, want[1])
        same("dlogits", d[:, :width].reshape(want[2].shape), want[2])


@pytest.mark.parametrize("n", [1, 5, 32, 33, 300])
@pytest.mark.parametrize("others", [0.0, 0.5])
def test_infinite_weights(device, n, others):
    """A row of infinite weight gives dhead infinities of the sign of its dz x, whatever the number of rows and with weights of
    0 beside it: no NaN, as the formula has none (every p above 0, no x of 0)."""
    x, head, w, g = head_inputs(device, n, 300, 64, 5)
    x = torch.where(x == 0, torch.ones_like(x), x)
    ids = torch.randint(0, 300, (n,), generator=g).to(device.torch)
    w.fill_(others)
    w[n // 2] = math.inf
    dhead = head_loss.token_loss_grads(x, head, ids, w)[2]
    sign = torch.ones(300, 1, dtype=torch.float64, device=device.torch)
    sign[ids[n // 2]] = -1  # (p - 1 at the row's own token)
    same(f"{n} rows", dhead.double(), math.inf * sign * x[n // 2].double().sign())


@pytest.mark.parametrize("n", [5, 40, 300])
def test_neither_gradient(device, n):
    """Asked for no gradient, the calls of both give the loss alone."""
    x, head, w, g = head_inputs(device, n, 900, 800, 6)
    ids = torch.randint(-100, 900, (n,), generator=g).to(device.torch)
    ti, tv = teacher(n, 5, 900, g, device)
    for loss, got in (
        (head_loss.token_loss(x, head, ids), head_loss.token_loss_grads(x, head, ids, w, x_grad=False, head_grad=False)),
        (head_loss.distill_loss(x, head, tv, ti), head_loss.distill_loss_grads(x, head, tv, ti, w, x_grad=False, head_grad=False)),
    ):
        assert got[1] is None and got[2] is None
        same("loss", got[0], loss)


def test_empty_batches_in_autograd(device):
    """No rows, and no batches: gradients of the leaves' shapes, zeros where there is anything."""
    x, head, _, _ = head_inputs(device, 4, 300, 64, 8)
    leaf, weight = x[:0].clone().requires_grad_(), head.clone().requires_grad_()
    loss = head_loss.token_loss(leaf, weight, torch.empty(0, dtype=torch.int64, device=device.torch))
    loss.sum().backward()
    assert loss.shape == (0,) and leaf.grad.shape == (0, 64) and not weight.grad.any()
    for shape in ((2, 0, 32), (0, 5, 32)):
        logits = torch.empty(shape, device=device.torch).requires_grad_()
        ids = torch.empty(*shape[:2], 4, dtype=torch.int16, device=device.torch)
        loss, counts = balance.balance_loss(logits, ids, 4)
        loss.sum().backward()
        assert loss.shape == shape[:1] and counts.shape == (shape[0], 32) and not counts.any() and logits.grad.shape == shape


def test_one_vector(device):
    """x of rank 1, a target of rank 0, teacher's entries of rank 1."""
    x, head, _, g = head_inputs(device, 1, 300, 64, 9)
    ids = torch.randint(0, 300, (1,), generator=g).to(device.torch)
    ti, tv = teacher(1, 5, 300, g, device)
    for got, want in ((head_loss.token_loss_grads(x[0], head, ids[0]), head_loss.token_loss_grads(x, head, ids)),
                      (head_loss.distill_loss_grads(x[0], head, tv[0], ti[0]), head_loss.distill_loss_grads(x, head, tv, ti))):
        assert got[0].shape == () and got[1].shape == (64,)
        for part, a, b in zip(("loss", "dx", "dhead"), got, want):
            same(part, a.reshape(b.shape), b)


def test_backward_twice_and_on_another_stream(device):
    """One graph's backward twice, the second time with the caller on another stream than the forward's."""
    x, head, w, g = head_inputs(device, 200, 900, 136, 10)
    ids = torch.randint(-50, 900, (200,), generator=g).to(device.torch)
    logits, slots, mask, gb = router_inputs(device, 3, 70, 64, 60, 4, 10)
    want = head_loss.token_loss_grads(x, head, ids, w)
    more = balance.balance_loss_grads(logits, slots, 4, gb, experts=60, mask=mask[:, :1].expand(3, 70))
    xl, hl, ll = (t.clone().requires_grad_() for t in (x, head, logits))
    loss = head_loss.token_loss(xl, hl, ids)
    bal, _ = balance.balance_loss(ll, slots, 4, experts=60, mask=mask[:, :1].expand(3, 70))
    total = (loss * w).sum() + (bal * gb).sum()
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            grads = torch.autograd.grad(total, (xl, hl, ll), retain_graph=True)
        torch.cuda.current_stream().wait_stream(stream)
        for part, a, b in zip(("dx", "dhead", "dlogits"), grads, (want[1], want[2], more[2])):
            same(part, a, b)


def test_two_threads(device):
    """Two threads at once, a stream each, of few rows and of many: what one alone gives."""
    calls = []
    for n in (40, 500):
        x, head, w, g = head_inputs(device, n, 2000, 264, n)
        ids = torch.randint(-50, 2000, (n,), generator=g).to(device.torch)
        logits, slots, mask, gb = router_inputs(device, 2, n, 64, 64, 4, n)
        calls.append(lambda x=x, head=head, ids=ids, w=w, logits=logits, slots=slots, gb=gb: (
            *head_loss.token_loss_grads(x, head, ids, w), *balance.balance_loss_grads(logits, slots, 4, gb)))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = [calls[i]() for _ in range(20)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs, ref in zip(got, want):
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, ref))
