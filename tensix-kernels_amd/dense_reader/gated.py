"""gated.py: the gated feed-forward block in training on MI355X, with its gradients: h = a(x . w_gate^T) * (x . w_up^T), for bf16
weights as a linear layer holds them ([width, dim], one row an output). It is what linear(activation="swiglu" or "geglu") computes of
packed weights, which are not trained; the reference (XylolabsInc/tensix-kernels, its dense_reader/linear.py:568-744) has no
counterpart.

  h = gated(x, w_gate, w_up)                                 # bf16 [..., width]; differentiable in x and both weights
  h = gated(x, w_gate, w_up, "geglu", keep=False)            # the same, keeping nothing for backward but its inputs
  h, kept = gated_keep(x, w_gate, w_up)                      # a step without autograd, in a HIP graph say
  dx, dw_gate, dw_up = gated_grads(x, w_gate, w_up, dh, kept=kept)

Sums are float32; h and the gradients bf16, rounded once. The gradients' products take dg and du, the gradients of both
projections' outputs, rounded to bf16: a value of dx or of a weight's gradient that one of theirs dominates is off by up to half a
bf16 step twice. What the forward pass keeps is both projections' outputs, g and u, in 24 bits each (float32 without the last 8 of
the mantissa), 6 bytes an output and row; with keep=False, or kept=None, they are computed again instead.

Nothing goes to the host. Memory comes from torch's allocator each call, on the current stream, so calls on several streams, threads
or captured graphs never share any. In a HIP graph, capture gated, gated_keep and gated_grads; autograd's backward refuses to be
captured (the gradient's accumulation into a leaf may run on another stream than the capture's, which ends the process).

The kernels are dr_gated_run's of libdense_reader.so (include/gated.h).
"""

import ctypes
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from common import device as dev  # noqa: E402
from dense_reader import _lib  # noqa: E402

ACTIVATIONS = {"swiglu": 0, "geglu": 1}
MAX_LD = _lib.DR_GATED_MAX_LD  # values from a row of x or a weight to the next at most, else it is copied
PANEL = 256  # outputs of a panel of what is kept


def _rows(t, dim):
    """t [..., dim] as rows the kernels read where they lie (itself, or a copy), and the values from one to the next."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, dim
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    if t.stride(-1) != 1 or t.data_ptr() % 16 or (t.shape[0] > 1 and (t.stride(0) % 8 or not dim <= t.stride(0) <= MAX_LD)):
        t = t.clone(memory_format=torch.contiguous_format)
    return t, (t.stride(0) if t.shape[0] > 1 else dim)


class _Call:
    """One call's inputs, checked, and the launch of it."""

    def __init__(self, x, w_gate, w_up, activation):
        dev.no_tangents("gated", x, w_gate, w_up)
        assert activation in ACTIVATIONS, f"gated: activation {activation!r}"
        device, bf16 = x.device, torch.bfloat16
        assert x.is_cuda and x.dtype is bf16 and x.dim() >= 1, (device, x.dtype, x.shape)
        assert w_gate.dtype is bf16 and w_up.dtype is bf16, (w_gate.dtype, w_up.dtype)
        assert w_gate.device == device and w_up.device == device, (w_gate.device, w_up.device, device)
        shape = w_gate.shape
        assert len(shape) == 2 and shape == w_up.shape, (shape, w_up.shape)
        self.width, self.dim = width, dim = shape
        self.device, self.shape = device, x.shape
        assert self.shape[-1] == dim, (x.shape, shape)
        assert dim % 8 == 0 and width % 8 == 0 and dim and width, f"gated: [{width}, {dim}] weights: not multiples of 8"
        n = self.n = x.numel() // dim
        x, ldx = _rows(x, dim)
        gate, ld_gate = _rows(w_gate, dim)
        up, ld_up = _rows(w_up, dim)
        self.held = x, gate, up
        self.A = _lib.Gated(x.data_ptr(), ldx, gate.data_ptr(), ld_gate, up.data_ptr(), ld_up, n, dim, width,
                            ACTIVATIONS[activation])

    def run(self, what):
        A, device = self.A, self.device
        ref = ctypes.byref(A)
        lib = _lib.lib()
        if what == _lib.DR_GATED_BACKWARD:
            need = lib.dr_gated_workspace_bytes(ref, what)
            _lib.check(_lib.DR_EINVAL if need < 0 else _lib.DR_OK, "dr_gated_workspace_bytes")
            ws = torch.empty(need, dtype=torch.uint8, device=device)
            A.workspace, A.workspace_bytes = ws.data_ptr(), need
        A.stream = dev.raw_stream(device)
        if device.index == torch.cuda.current_device():
            st = lib.dr_gated_run(ref, what)
        else:  # (a launch goes to the current device)
            with torch.cuda.device(device):
                st = lib.dr_gated_run(ref, what)
        if st != _lib.DR_OK:
            _lib.check(st, "dr_gated_run")

    def kept_shape(self):
        return 3, -(-self.width // PANEL), self.n, PANEL

    def forward(self, keep):
        A, x = self.A, self.held[0]
        h = x.new_empty((*self.shape[:-1], self.width))
        kept = x.new_empty(self.kept_shape(), dtype=torch.int16) if keep else None
        if self.n:
            A.h, A.ld_h = h.data_ptr(), self.width
            if keep:
                A.kept = kept.data_ptr()
            self.run(_lib.DR_GATED_FORWARD)
        return h, kept

    def backward(self, dh, kept, x_grad, gate_grad, up_grad):
        width, dim, A = self.width, self.dim, self.A
        x, gate, _ = self.held
        dx = x.new_empty(self.shape) if x_grad else None
        dgate, dup = (gate.new_empty((width, dim)) if asked else None for asked in (gate_grad, up_grad))
        if self.n == 0:
            for t in (dgate, dup):
                if t is not None:
                    t.zero_()
            return dx, dgate, dup
        dh, A.ld_dh = _rows(dh, width)
        A.dh, A.ld_dx, A.ld_dgate, A.ld_dup = dh.data_ptr(), dim, dim, dim
        A.kept, A.dx, A.dgate, A.dup = [None if t is None else t.data_ptr() for t in (kept, dx, dgate, dup)]
        self.run(_lib.DR_GATED_BACKWARD)
        return dx, dgate, dup

    def check_grads(self, dh, kept):
        dev.no_tangents("gated", dh, kept)
        assert dh.device == self.device and dh.dtype is torch.bfloat16, (dh.device, dh.dtype)
        assert dh.shape == (*self.shape[:-1], self.width), (dh.shape, self.shape, self.width)
        if kept is not None:
            assert kept.device == self.device and kept.dtype is torch.int16, (kept.device, kept.dtype)
            assert kept.shape == self.kept_shape(), (kept.shape, self.kept_shape())
            assert kept.is_contiguous() and kept.data_ptr() % 16 == 0, "gated: kept as gated_keep gave it"


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation, keep):
        h, kept = _Call(x, w_gate, w_up, activation).forward(keep)
        ctx.save_for_backward(x, w_gate, w_up, kept)
        ctx.activation = activation
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("gated: a HIP graph captures gated_keep and gated_grads, not backward()")
        x, w_gate, w_up, kept = ctx.saved_tensors
        c = _Call(x, w_gate, w_up, ctx.activation)
        c.check_grads(dh, kept)
        return (*c.backward(dh, kept, *ctx.needs_input_grad[:3]), None, None)


def gated(x, w_gate, w_up, activation="swiglu", keep=True):
    """h = a(x . w_gate^T) * (x . w_up^T): x [..., dim] bf16 on the GPU, w_gate and w_up [width, dim] bf16, dim and width multiples
    of 8 (to 2^17 and 2^20, to 2^20 rows); h [..., width] bf16, differentiable in all three. activation: "swiglu" (a silu) or "geglu" (gelu's tanh form). keep: hold
    6 bytes an output and row for backward, which otherwise computes both projections again from x."""
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        return _Gated.apply(x, w_gate, w_up, activation, keep)
    return _Call(x, w_gate, w_up, activation).forward(False)[0]


def gated_keep(x, w_gate, w_up, activation="swiglu"):
    """(h, kept): gated's h, and what gated_grads of the same x, weights and activation takes ([3, ceil(width / 256), rows, 256]
    int16: the library's own layout of both projections' outputs)."""
    return _Call(x, w_gate, w_up, activation).forward(True)


def gated_grads(x, w_gate, w_up, dh, activation="swiglu", kept=None, x_grad=True, w_grad=True):
    """The gradients of the sum of dh * h: (dx, dw_gate, dw_up), bf16 in the shapes of x and the weights (None for those not asked
    for: a frozen layer's). dh [..., width] bf16. kept: gated_keep's of the same x, weights and activation, or None: both projections
    again. With kept, x's values count for the weights' gradients alone, the weights' for dx alone."""
    c = _Call(x, w_gate, w_up, activation)
    c.check_grads(dh, kept)
    return c.backward(dh, kept, x_grad, w_grad, w_grad)
