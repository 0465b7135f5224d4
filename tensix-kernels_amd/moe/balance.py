"""balance.py: the MoE router's balance loss and each expert's count on MI355X, with the gradient of the router's logits.
The reference (XylolabsInc/tensix-kernels) has no counterpart; logits and ids are moe8.route's (its moe/moe8.py:1139-1253).

  moe8.route(logits, ids, w, k)                              # the picks
  loss, counts = balance_loss(logits, ids, k)                # differentiable in the logits
  loss, counts, dlogits = balance_loss_grads(logits, ids, k, g)

Over the rows t of a batch (the second last dim; the dims before it are batches, each with a loss of its own: a sequence's,
or with one batch the whole step's): p[t] = softmax(logits[t]), or with kind "sigmoid" sigmoid(logits[t]) over its sum;
counts[e] = the slots that chose expert e; loss = sum over e of E counts[e] / sum(counts) * mean over t of p[t][e], which is
1 where every expert is chosen alike. (A row with no logit above -inf, or whose sigmoids are all 0 in float32, has p 0.) The
counts have no gradient (a choice has none); a backward takes them as its forward made them, so one ids buffer serves several
layers, and reads the logits and the mask again. mask: the rows that count (a padded batch); the others enter nothing, whatever
their logits and ids hold, and get zeros. An id at or past E chooses no expert.

The kernels are dr_moe_balance's of libdense_reader.so (include/moe.h); nothing goes to the host, and the memory of a call
is torch's, on the current stream, so a HIP graph can hold balance_loss and balance_loss_grads (autograd's backward refuses
to be captured, as lm_head_topk.head_loss's does).
"""

import ctypes
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from common import device as dev  # noqa: E402
from dense_reader import _lib  # noqa: E402

MAX_E = 1024  # experts at most, as moe8.route's
KINDS = {"softmax": 0, "sigmoid": 1}


def _weights(g, batch, device):
    """The batches' weights as the launch takes them (None: ones)."""
    if g is None:
        return None
    dev.no_tangents("balance", g)
    # (a number filled in: a copy from the host could not be captured)
    gs = g if isinstance(g, torch.Tensor) else torch.full((batch,), float(g), device=device)
    assert gs.device == device, (gs.device, device)
    assert gs.numel() in (1, batch), f"balance: {gs.numel()} weights for {batch} batches"
    if gs.dtype != torch.float32 or gs.numel() != batch or not gs.is_contiguous():
        gs = gs.detach().reshape(-1).to(torch.float32).expand(batch).contiguous()
    return gs


def _launch(A, what, device):
    ref = ctypes.byref(A)
    A.stream = dev.raw_stream(device)
    lib = _lib.lib()
    if device.index == torch.cuda.current_device():
        st = lib.dr_moe_balance(ref, what)
    else:  # (a launch goes to the current device)
        with torch.cuda.device(device):
            st = lib.dr_moe_balance(ref, what)
    if st != _lib.DR_OK:
        _lib.check(st, "dr_moe_balance")


def _run(logits, ids, k, g, kind, ids32, experts, mask, grad, keep=False):
    """(loss, counts, dlogits or None, what a backward takes or None)."""
    dev.no_tangents("balance", logits)
    assert kind in KINDS, f"balance: kind {kind!r}"
    assert logits.is_cuda and logits.dtype == torch.float32 and logits.dim() >= 2, (logits.device, logits.dtype)
    *lead, R, W = logits.shape
    E = W if experts is None else int(experts)
    assert 1 <= E <= min(W, MAX_E) and 1 <= k <= 16, (E, W, k)
    batch = 1
    for n in lead:
        batch *= n
    want = (torch.int32, torch.uint32) if ids32 else (torch.int16, torch.uint16)
    assert ids.dtype in want, f"balance: ids are {ids.dtype}, ids32={ids32} wants {want[0]} or {want[1]}"
    assert ids.device == logits.device and ids.is_contiguous(), (ids.device, ids.is_contiguous())
    ld = ids.shape[-1]
    assert ld >= k and ids.numel() == batch * R * ld, (tuple(ids.shape), tuple(logits.shape), k)
    lg = logits.contiguous()
    m = None
    if mask is not None:
        assert mask.device == logits.device and mask.dtype in (torch.bool, torch.uint8), (mask.device, mask.dtype)
        assert mask.numel() == batch * R, (tuple(mask.shape), tuple(logits.shape))
        m = mask.contiguous()
    device = logits.device
    gs = _weights(g, batch, device) if grad else None
    loss = torch.empty(lead, dtype=torch.float32, device=device)
    counts = torch.empty((*lead, E), dtype=torch.int32, device=device)
    dlogits = torch.empty_like(lg) if grad else None
    kept = torch.empty((batch, 1 + E), dtype=torch.int32, device=device) if keep else None
    if batch * R == 0:
        loss.zero_(), counts.zero_()
        return loss, counts, dlogits, kept
    ptr = torch.Tensor.data_ptr
    A = _lib.Balance(
        ptr(lg), W, batch, R, E, W, ptr(ids), ld, bool(ids32), k, KINDS[kind], None if m is None else ptr(m), ptr(loss),
        ptr(counts), None if kept is None else ptr(kept), None if gs is None else ptr(gs),
        None if dlogits is None else ptr(dlogits), W)
    ref = ctypes.byref(A)
    what = _lib.DR_BALANCE_GRAD if grad else _lib.DR_BALANCE_LOSS
    lib = _lib.lib()
    need = lib.dr_moe_balance_workspace_bytes(ref, what)
    _lib.check(_lib.DR_EINVAL if need < 0 else _lib.DR_OK, "dr_moe_balance_workspace_bytes")
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        A.workspace, A.workspace_bytes = ptr(ws), need
    _launch(A, what, device)
    return loss, counts, dlogits, kept


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, k, kind, ids32, experts, mask):
        # (the counts kept, not the ids: the next layer's router may write into the same buffer before this backward)
        loss, counts, _, kept = _run(logits, ids, k, None, kind, ids32, experts, mask, False, keep=True)
        ctx.save_for_backward(logits, mask, kept)
        ctx.kind = kind
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("balance: a HIP graph captures balance_loss_grads, not backward()")
        logits, mask, kept = ctx.saved_tensors
        lg, m = logits.contiguous(), None if mask is None else mask.contiguous()
        R, W = lg.shape[-2:]
        batch, E = kept.shape[0], kept.shape[1] - 1
        dlogits = torch.empty_like(lg)
        if lg.numel():
            gs = _weights(g, batch, lg.device)
            A = _lib.Balance(logits=lg.data_ptr(), ld_logits=W, batch=batch, rows=R, experts=E, width=W, ld_ids=1, k=1,
                             kind=KINDS[ctx.kind], mask=None if m is None else m.data_ptr(), kept=kept.data_ptr(),
                             g=gs.data_ptr(), dlogits=dlogits.data_ptr(), ld_dlogits=W)
            _launch(A, _lib.DR_BALANCE_BACKWARD, lg.device)
        return dlogits, None, None, None, None, None, None


def balance_loss(logits, ids, k, *, kind="softmax", ids32=False, experts=None, mask=None):
    """(loss, counts): logits [..., R, W] float32 on the GPU, ids [..., R, >= k] (uint16, or uint32 with ids32: moe8.route's,
    contiguous; the first k of a row), loss float32 and counts int32 [..., E] for each batch of R rows. experts (default W):
    the logits' columns 0 .. E - 1. mask [..., R] bool: the rows that count (default all). The loss is differentiable in the
    logits."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Balance.apply(logits, ids, k, kind, ids32, experts, mask)
    return _run(logits, ids, k, None, kind, ids32, experts, mask, False)[:2]


def balance_loss_grads(logits, ids, k, g=None, *, kind="softmax", ids32=False, experts=None, mask=None):
    """balance_loss and, in the same call, the gradient of the sum over batches of g * loss: (loss, counts, dlogits), dlogits
    of the logits' shape (zeros past E). g: each batch's weight, one number for all, or None for ones."""
    return _run(logits, ids, k, g, kind, ids32, experts, mask, True)[:3]
