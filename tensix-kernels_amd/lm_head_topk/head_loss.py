"""head_loss.py: the LM head's losses on MI355X, with their gradients: the cross entropy of the head's logits against each
row's token, and the divergence from a teacher's best logits of each row. The reference (XylolabsInc/tensix-kernels) has no
counterpart; the head is head_pick.head_rows' table (its lm_head_topk/head_pick.py:43-52), a teacher's logits what
linear.topk_merge leaves of its top-k records (its dense_reader/linear.py:747-768).

  rows = head_rows(device, weight)                              # the bf16 head [1, 1, vocab, dim], one row a token
  loss = token_loss(x, rows, targets)                           # float32, one a row; differentiable in x and rows
  loss, dx, drows = token_loss_grads(x, rows, targets, g)       # the same and its gradients in one call
  vals, ids = linear.topk_merge(records, nrows, k, k_out=16)    # a teacher's best logits and their ids
  loss, dx, drows = distill_loss_grads(x, student_rows, vals, ids, g, temperature=2.0)

The logits x . rows^T (float32 sums) go by in pieces, and backward computes them again; a call of both directions whose rows
times tokens are few enough (the logits 2 GiB, their gradient 1 GiB) keeps them in its workspace instead, which is faster for
few rows and from 768 values a row on. No call has more of them in memory. A row whose target lies
outside 0 .. valid - 1 (a padded or ignored position; -100, say), or that holds no teacher entry, is left out: its loss and
its dx are 0 and it adds nothing to drows, whatever x, the teacher's values or g hold there; it costs next to nothing where
there are many rows. dx and drows are bf16, summed in float32 from the logits' gradient rounded to bf16 (up to 32 rows, from
that and what the rounding leaves): past 32 rows a row of drows or dx that one token's gradient dominates is off by up to half
a bf16 step twice.

Nothing goes to the host. Memory comes from torch's allocator each call, on the current stream, so calls on several streams,
threads or captured graphs never share any. In a HIP graph, capture token_loss, distill_loss or the *_grads calls; autograd's
backward refuses to be captured (the gradient's accumulation into a leaf may run on another stream than the capture's, which
ends the process).

The kernels are dr_head_loss_run's of libdense_reader.so (include/lm_head.h).
"""

import ctypes
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from common import device as dev  # noqa: E402
from dense_reader import _lib  # noqa: E402
from lm_head_topk import head_pick  # noqa: E402

MAX_K = _lib.DR_LOSS_MAX_K  # teacher entries a row at most
MAX_LD = _lib.DR_LOSS_MAX_LD  # values from a row of x to the next at most, else it is copied


class _Call:
    """One call's inputs, checked, and the launch of it."""

    def __init__(self, x, rows_t, ids, vals, temperature, valid):
        dev.no_tangents("head_loss", x, rows_t, vals)
        dim = x.shape[-1]
        device = self.device = x.device
        assert x.is_cuda and x.dtype == torch.bfloat16, (x.device, x.dtype)
        assert dim % 8 == 0, f"head_loss: dim {dim} is not a multiple of 8"
        head_pick.check_rows(rows_t, dim)
        self.vocab = vocab = rows_t.shape[-2]
        self.valid = vocab if valid is None else int(valid)
        assert 1 <= self.valid <= vocab, (valid, rows_t.shape)
        if x.dim() != 2:
            x = x.reshape(-1, dim)
        n = self.n = x.shape[0]
        # (past MAX_LD the offsets in a tile pass the kernels' 32 bits: a few positions of long sequences, say)
        if x.stride(-1) != 1 or x.data_ptr() % 16 or (n > 1 and (x.stride(0) % 8 or not dim <= x.stride(0) <= MAX_LD)):
            x = x.clone(memory_format=torch.contiguous_format)
        self.x, self.rows_t, self.dim = x, rows_t, dim
        self.vals = None
        if vals is None:
            assert ids.dtype in (torch.int32, torch.int64), ids.dtype
            assert ids.numel() == n, f"head_loss: {ids.numel()} targets for {n} rows"
            self.shape, self.k = ids.shape, 1
        else:
            assert ids.dtype == torch.int32, ids.dtype
            assert vals.device == device and vals.dtype == torch.float32 and vals.shape == ids.shape and vals.dim() >= 1, (
                vals.device, vals.dtype, vals.shape, ids.shape)
            self.shape, self.k = ids.shape[:-1], ids.shape[-1]
            assert 1 <= self.k <= MAX_K, f"head_loss: 1 to {MAX_K} teacher entries a row, not {self.k}"
            assert ids.numel() == n * self.k, f"head_loss: teacher entries {tuple(ids.shape)} for {n} rows"
            self.vals = vals.contiguous()
        assert ids.device == device and rows_t.device == device, (ids.device, rows_t.device, device)
        self.ids = ids.contiguous()
        self.temperature = float(temperature)
        assert 2.0**-20 <= self.temperature < math.inf, f"head_loss: temperature {temperature}"

    def empty(self, *shape, dtype=torch.float32):
        return torch.empty(*shape or ((),), dtype=dtype, device=self.device)

    def outputs(self):
        """(loss, lse, logits) to be filled, and kept for a backward pass."""
        return self.empty(self.n), self.empty(self.n), self.empty(self.n, self.k)

    def grads(self, x_grad, head_grad):
        dx = self.empty(self.n, self.dim, dtype=torch.bfloat16) if x_grad else None
        return dx, self.empty(self.vocab, self.dim, dtype=torch.bfloat16) if head_grad else None

    def weights(self, g):
        """The rows' weights as the launch takes them (None: ones)."""
        if g is None:
            return None
        dev.no_tangents("head_loss", g)
        if not isinstance(g, torch.Tensor):
            return self.empty(self.n).fill_(float(g))  # (a copy from the host could not be captured)
        assert g.device == self.device, (g.device, self.device)
        if g.dtype == torch.float32 and g.numel() == self.n and g.is_contiguous():
            return g
        assert g.numel() in (1, self.n), f"head_loss: {g.numel()} weights for {self.n} rows"
        return g.detach().reshape(-1).to(torch.float32).expand(self.n).contiguous()

    def run(self, what, loss, lse=None, logits=None, g=None, dx=None, dhead=None):
        """The launch; lse and logits lie in its own memory unless given."""
        n, k, dim = self.n, self.k, self.dim
        if n == 0:
            if dhead is not None:
                dhead.zero_()
            return

        def ptr(t):
            return None if t is None else t.data_ptr()

        A = _lib.HeadLoss(
            self.x.data_ptr(), self.x.stride(0) if n > 1 else dim, self.rows_t.data_ptr(), dim, n, dim, self.vocab,
            self.valid, self.ids.data_ptr(), k, self.ids.dtype == torch.int64, k, ptr(self.vals), k, self.temperature,
            ptr(loss), ptr(lse), ptr(logits), ptr(g), ptr(dx), dim, ptr(dhead), dim)
        ref = ctypes.byref(A)
        lib = _lib.lib()
        need = lib.dr_head_loss_workspace_bytes(ref, what)
        _lib.check(_lib.DR_EINVAL if need < 0 else _lib.DR_OK, "dr_head_loss_workspace_bytes")
        own = 0 if lse is not None else 4 * n * (1 + k)
        ws = self.empty(need + own, dtype=torch.uint8)
        A.workspace, A.workspace_bytes = ws.data_ptr(), need
        if own:
            A.lse, A.logits = A.workspace + need, A.workspace + need + 4 * n
        A.stream = dev.raw_stream(self.device)
        if self.device.index == torch.cuda.current_device():
            st = lib.dr_head_loss_run(ref, what)
        else:  # (a launch goes to the current device)
            with torch.cuda.device(self.device):
                st = lib.dr_head_loss_run(ref, what)
        if st != _lib.DR_OK:
            _lib.check(st, "dr_head_loss_run")


class _Loss(torch.autograd.Function):
    """The loss of each row, differentiable in x and the head's rows; backward computes the logits again."""

    @staticmethod
    def forward(ctx, x, rows_t, ids, vals, temperature, valid):
        c = _Call(x, rows_t, ids, vals, temperature, valid)
        loss, lse, logits = c.outputs()
        c.run(_lib.DR_LOSS_FORWARD, loss, lse, logits)
        ctx.save_for_backward(x, rows_t, ids, vals, lse, logits)
        ctx.settings = temperature, valid
        return loss.reshape(c.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("head_loss: a HIP graph captures token_loss_grads or distill_loss_grads, not backward()")
        x, rows_t, ids, vals, lse, logits = ctx.saved_tensors
        c = _Call(x, rows_t, ids, vals, *ctx.settings)
        dx, dhead = c.grads(*ctx.needs_input_grad[:2])
        c.run(_lib.DR_LOSS_BACKWARD, None, lse, logits, c.weights(g), dx, dhead)
        return (None if dx is None else dx.reshape(x.shape), None if dhead is None else dhead.reshape(rows_t.shape),
                None, None, None, None)


def _loss(x, rows_t, ids, vals, temperature, valid):
    if torch.is_grad_enabled() and (x.requires_grad or rows_t.requires_grad):
        return _Loss.apply(x, rows_t, ids, vals, temperature, valid)
    c = _Call(x, rows_t, ids, vals, temperature, valid)
    loss = c.empty(*c.shape)
    c.run(_lib.DR_LOSS_FORWARD, loss)
    return loss


def _grads(x, rows_t, ids, vals, temperature, valid, g, x_grad, head_grad):
    c = _Call(x, rows_t, ids, vals, temperature, valid)
    loss = c.empty(*c.shape)
    dx, dhead = c.grads(x_grad, head_grad)
    c.run(_lib.DR_LOSS_FORWARD | _lib.DR_LOSS_BACKWARD, loss, g=c.weights(g), dx=dx, dhead=dhead)
    return (loss, None if dx is None else dx.reshape(x.shape), None if dhead is None else dhead.reshape(rows_t.shape))


def token_loss(x, rows_t, targets, valid=None):
    """Per row of x [..., dim] bf16 the cross entropy of the head's logits against its target: float32 of the targets'
    shape, differentiable in x and rows_t (head_rows' table, [vocab, dim] or [1, 1, vocab, dim] bf16). targets: int64 or
    int32, one a row; one outside 0 .. valid - 1 leaves its row out. valid: a padded head's real vocabulary (the rows past
    it enter nothing and get zeros; default all)."""
    return _loss(x, rows_t, targets, None, 1.0, valid)


def token_loss_grads(x, rows_t, targets, g=None, valid=None, x_grad=True, head_grad=True):
    """token_loss and, in the same call, the gradients of the sum over rows of g * loss: (loss, dx, drows), bf16 in the
    shapes of x and rows_t (None for one not asked for: a frozen head's, say). g: each row's weight (float32, the targets'
    shape), one number for all, or None for ones."""
    return _grads(x, rows_t, targets, None, 1.0, valid, g, x_grad, head_grad)


def distill_loss(x, rows_t, vals, ids, temperature=1.0, valid=None):
    """Per row of x the divergence sum q log(q / p) of the head's softmax p over the vocabulary, at the temperature, from a
    teacher's q = softmax(vals / temperature) over the row's entries: float32, differentiable in x and rows_t. vals [..., k]
    float32 and ids [..., k] int32, k to 64: as linear.topk_merge leaves them (-inf and -1 in empty slots), of a teacher
    of this vocabulary; an id outside 0 .. valid - 1 is an empty slot too, one that comes twice counts twice, and a row of
    empty slots is left out. temperature: from 2^-20 on (a probability is off by |logit| / temperature * 2^-23 of itself)."""
    return _loss(x, rows_t, ids, vals, temperature, valid)


def distill_loss_grads(x, rows_t, vals, ids, g=None, temperature=1.0, valid=None, x_grad=True, head_grad=True):
    """distill_loss and its gradients in one call, as token_loss_grads."""
    return _grads(x, rows_t, ids, vals, temperature, valid, g, x_grad, head_grad)
