"""grads.py: a model's gradients as a whole on MI355X: their global norm, and clipping by it. The reference (XylolabsInc/
tensix-kernels) has no counterpart; the gradients are those of dense_reader.gated, lm_head_topk.head_loss and moe.balance beside torch's
own.

  norm = global_norm(p.grad for p in params)                  # float32, on the device
  norm = clip_((p.grad for p in params), max_norm=1.0)        # in place, by min(1, max_norm / (norm + 1e-6))
  norm, out = clipped(grads, 1.0, dtype=torch.float32)        # the same into tensors of their own (or out=)

  total = global_norm(mine).square_()                         # gradients that lie on several ranks:
  dist.all_reduce(total)
  clip_(mine, 1.0, norm=total.sqrt_())                        # clipped by the norm of all

The tensors are float32, bfloat16 or float16 on one GPU, in any mix and of any shapes (None is passed over). Squares and their sums are
float64, so that no float32 gradient overflows; a clipped value is the float32 product with the factor, rounded once. A NaN among them
makes the norm and all that is clipped NaN, an infinity the norm infinite and the clipped values 0 (its own NaN): look at the norm. An
infinite max_norm is no limit: all stays as it is, infinities too, but for a NaN's. A tensor whose memory is dense in another order of
its dims (a transposed gradient) is taken as it lies; any other strided one is read from a copy, and refused in place.

Nothing goes to the host and nothing is differentiable. Memory comes from torch's allocator each call, on the current stream, so calls
on several streams, threads or captured graphs never share any; the addresses are the launches' arguments, so a captured graph goes on
with the tensors that it saw.

The kernels are dr_grads_norm's and dr_grads_clip's of libdense_reader.so (include/grads.h).
"""

import ctypes
import sys
from array import array
from operator import attrgetter
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from common import device as dev  # noqa: E402
from dense_reader import _lib  # noqa: E402

_data_ptr, _numel, _contiguous = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous
_dtype, _requires_grad = attrgetter("dtype"), attrgetter("requires_grad")
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _order(t):
    """The dims of t by falling stride, if its memory is dense in that order (None otherwise)."""
    dims = sorted(range(t.dim()), key=lambda d: (t.stride(d), t.shape[d]), reverse=True)
    return dims if t.permute(dims).is_contiguous() else None


def _tensors(grads):
    """The tensors among them, checked, and their device."""
    ts = [t for t in grads if t is not None]
    if not ts:
        raise ValueError("grads: no gradients")
    dev.no_tangents("grads", *ts)
    device = ts[0].device
    assert device.type == "cuda", device
    assert set(map(torch.Tensor.get_device, ts)) == {device.index}, f"grads: not all on {device}"
    assert not (torch.is_grad_enabled() and any(map(_requires_grad, ts))), (
        "grads: no derivative (detach them, or call under torch.no_grad())")
    return ts, device


def _types(ts):
    kinds = list(map(TYPES.get, map(_dtype, ts)))
    assert None not in kinds, set(map(_dtype, ts))
    return array("i", kinds)


class _Call:
    """The tensors' values, and the launch over them. (The lists are arrays of the standard library, each made of a list, which is
    faster than of an iterator: what the call's host time goes by is how often each tensor is asked for something.)"""

    def __init__(self, ts, device, sizes=None):
        self.device, self.held = device, ts
        self.norm = torch.empty((), dtype=torch.float32, device=device)
        self.ins, self.sizes, self.types = array("Q", list(map(_data_ptr, ts))), array("q", sizes or list(map(_numel, ts))), _types(ts)
        self.A = _lib.Grads(len(ts), *(a.buffer_info()[0] for a in (self.ins, self.sizes, self.types)))

    def run(self, fn, workspace):
        A, device = self.A, self.device
        if workspace:
            ws = torch.empty(-(-A.count // _lib.DR_GRADS_LIST) * _lib.DR_GRADS_LIST_BYTES, dtype=torch.uint8, device=device)
            A.workspace, A.workspace_bytes = ws.data_ptr(), ws.numel()
        A.norm = self.norm.data_ptr()
        A.stream = dev.raw_stream(device)
        if device.index == torch.cuda.current_device():
            st = fn(ctypes.byref(A))
        else:  # (a launch goes to the current device)
            with torch.cuda.device(device):
                st = fn(ctypes.byref(A))
        if st != _lib.DR_OK:
            _lib.check(st, "dr_grads_norm" if fn is _lib.lib().dr_grads_norm else "dr_grads_clip")

    def clip(self, outs, max_norm, norm):
        A = self.A
        at, types = (self.ins, self.types) if outs is self.held else (array("Q", list(map(_data_ptr, outs))), _types(outs))
        A.out, A.out_types = at.buffer_info()[0], types.buffer_info()[0]
        assert not isinstance(max_norm, torch.Tensor), "grads: max_norm is a number of the host's"
        A.max_norm = float(max_norm)
        assert A.max_norm >= 0, f"grads: max_norm {max_norm}"
        if norm is not None:
            dev.no_tangents("grads", norm)
            assert norm.device == self.device and norm.dtype == torch.float32 and norm.numel() == 1, (norm.device, norm.dtype, norm.shape)
            assert not norm.is_neg(), "grads: a norm is no negative view"
            assert not (torch.is_grad_enabled() and norm.requires_grad), "grads: no derivative by the norm (detach it)"
            self.norm, A.given = norm, 1
        self.run(_lib.lib().dr_grads_clip, norm is None)
        return self.norm


def global_norm(grads):
    """The 2-norm of all values of the gradients (an iterable of tensors or None): float32 [] on their device."""
    ts, device = _tensors(grads)
    c = _Call([t if t.is_contiguous() or _order(t) else t.contiguous() for t in ts], device)
    c.run(_lib.lib().dr_grads_norm, True)
    return c.norm


def clip_(grads, max_norm, norm=None):
    """The gradients times min(1, max_norm / (their global norm + 1e-6)), in place; the norm before that, float32 []. norm: take this
    one instead (float32, one value on their device). Tensors that share memory are refused (ValueError)."""
    ts, device = _tensors(grads)
    assert all(t.is_contiguous() or _order(t) for t in ts), "grads: in place, a gradient's memory is dense"
    norm = _Call(ts, device).clip(ts, max_norm, norm)
    dev.written(*ts)
    return norm


def clipped(grads, max_norm, out=None, dtype=None, norm=None):
    """(norm, clipped): clip_'s norm, and the clipped gradients in tensors of their own, of `dtype` (default each one's own), or in `out`,
    a list of contiguous tensors of as many values (None where a gradient is). No tensor of out may share memory with another, nor with
    a gradient but its own as a whole (ValueError)."""
    grads = list(grads)
    ts, device = _tensors(grads)
    sizes = list(map(_numel, ts))
    if out is None:
        assert dtype is None or dtype in TYPES, dtype
        out = [None if t is None else torch.empty(t.shape, dtype=dtype or t.dtype, device=device) for t in grads]
        outs = [o for o in out if o is not None]
    else:
        assert dtype is None, "grads: dtype is out's"
        out = list(out)
        outs, where = _tensors(out)
        assert where == device and all(map(_contiguous, outs)), "grads: out is contiguous, on the gradients' device"
        if len(ts) < len(grads) or len(outs) < len(out):
            assert [t is None for t in grads] == [o is None for o in out], "grads: out has a tensor where there is a gradient"
        assert list(map(_numel, outs)) == sizes, "grads: out has as many values of each"
    if not all(map(_contiguous, ts)):
        ts = [t.contiguous() for t in ts]
    if 1 in sizes:  # (the only contiguous memory that can stand for its negative: a value of a conjugate's imaginary part)
        assert not any(o.is_neg() for o in outs), "grads: out is a negative view"
        ts = [t.resolve_neg() for t in ts]
    norm = _Call(ts, device, sizes).clip(outs, max_norm, norm)
    dev.written(*outs)
    return norm, out
