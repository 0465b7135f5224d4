"""A training step's feed-forward block and the norm of its gradients: what is timed and compared.

A case is one pass through an operator, as a training program makes it:

- gated: the gated block act(x . w_gate^T) * (x . w_up^T) of weights in training (dense_reader.gated): the block alone
         (sampling or scoring with the weights that are being trained), with what its gradients need and those (a step),
         or its gradients alone, computed again from x (a step that keeps nothing of the layer);
- norm:  the global norm of a model's gradients (common.grads), alone (a log, or a check);
- clip:  the same and the gradients clipped by it, into the buffers that an optimizer reads.

Rows are standard normal with a few channels far larger, weights as an initialised or trained layer has them. A model's
gradients are a list: for each layer two norms' vectors, the attention's four matrices and the block's three, then the
embedding; some of them have no part in a step and are zero, and their sizes differ by orders of magnitude.
"""

import math
import sys
from pathlib import Path

import torch

own = False
PKG = str(Path(__file__).resolve().parents[1] / "tensix-kernels_amd")


def listed():
    return [
        # one token sampled with a small draft's weights: launch and host time count
        {"name": "block_token", "kind": "gated", "n": 1, "d": 1024, "f": 4096, "act": "swiglu", "mode": "alone"},
        # a decode step of a batch with a large layer's training weights: their bytes bound it
        {"name": "block_rows", "kind": "gated", "n": 32, "d": 4096, "f": 14336, "act": "swiglu", "mode": "alone"},
        # a ragged batch scored
        {"name": "block_score", "kind": "gated", "n": 2047, "d": 2880, "f": 2880, "act": "geglu", "mode": "alone"},
        # a small step of a draft
        {"name": "train_small", "kind": "gated", "n": 48, "d": 1024, "f": 4096, "act": "swiglu", "mode": "step"},
        # fine-tuning on a ragged batch
        {"name": "train_ragged", "kind": "gated", "n": 1003, "d": 2048, "f": 5632, "act": "geglu", "mode": "step"},
        # a training step of a large layer
        {"name": "train_large", "kind": "gated", "n": 8192, "d": 4096, "f": 14336, "act": "swiglu", "mode": "step"},
        # the backward pass of a layer that kept nothing, its weights frozen
        {"name": "train_frozen", "kind": "gated", "n": 4096, "d": 4096, "f": 14336, "act": "swiglu", "mode": "again",
         "weights": False},
        # a small model's gradients
        {"name": "norm_small", "kind": "norm", "layers": 2, "d": 96, "f": 250, "v": 0, "type": "float32"},
        # a model's gradients as its backward pass left them
        {"name": "norm_model", "kind": "norm", "layers": 16, "d": 1024, "f": 4096, "v": 8192, "type": "bfloat16"},
        # a draft's gradients of odd sizes, for an optimizer of weights of their own type
        {"name": "clip_draft", "kind": "clip", "layers": 4, "d": 500, "f": 1333, "v": 8192, "type": "bfloat16",
         "out": "bfloat16"},
        # gradients of one type and the float32 that an optimizer of float32 weights takes
        {"name": "clip_wide", "kind": "clip", "layers": 6, "d": 1024, "f": 2880, "v": 32000, "type": "bfloat16",
         "out": "float32"},
        # accumulated float32 gradients of wide layers and a large embedding
        {"name": "clip_large", "kind": "clip", "layers": 4, "d": 2048, "f": 5632, "v": 50257, "type": "float32",
         "out": "float32"},
    ]


# --- drawn cases ------------------------------------------------------------------------------------------------------


def _log(rng, lo, hi, step=1):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step))


def draw(rng):
    kind = rng.choice(("gated", "gated", "gated", "norm", "clip"))
    if kind == "gated":
        case = {"kind": kind, "n": _log(rng, 1, 8192), "d": _log(rng, 256, 4096, 8), "f": _log(rng, 512, 14336, 8),
                "act": rng.choice(("swiglu", "geglu")), "mode": rng.choice(("alone", "step", "step", "again"))}
        return case if case["mode"] == "alone" else {**case, "weights": rng.choice((True, True, False))}
    layers = _log(rng, 1, 16 if kind == "norm" else 6)
    case = {"kind": kind, "layers": layers, "d": _log(rng, 64, 1024), "f": _log(rng, 100, 4096),
            "v": rng.choice((0, 1000, 8192, 32000)), "type": rng.choice(("float32", "bfloat16", "float16"))}
    return case if kind == "norm" else {**case, "out": rng.choice((case["type"], "float32"))}


def _shapes(case):
    d, f, kv = case["d"], case["f"], max(1, case["d"] // 4)
    layer = [(d,), (d,), (d, d), (kv, d), (kv, d), (d, d), (f, d), (f, d), (d, f)]
    return layer * case["layers"] + ([(case["v"], d)] if case["v"] else [])


# --- inputs -----------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    if case["kind"] == "gated":
        n, d, f = case["n"], case["d"], case["f"]
        x = randn(n, d)
        x[:, :4] *= 8
        bf16 = lambda t: t.to(torch.bfloat16)
        state = {"case": case, "x": bf16(x), "gate": bf16(randn(f, d) / d**0.5), "up": bf16(randn(f, d) / d**0.5)}
        if case["mode"] != "alone":
            state["dh"] = bf16(randn(n, f) / n)
        return state
    shapes, kind = _shapes(case), getattr(torch, case["type"])
    # how large each tensor's gradients are, over a range of 1000, one in sixteen none at all; the norm about 0.2 to 20
    scale = 10 ** -(3 * torch.rand(len(shapes), generator=g, device="cuda"))
    scale = torch.where(torch.arange(len(shapes), device="cuda") % 16 == 11, 0.0, scale)
    total = sum(math.prod(s) for s in shapes)
    scale = (scale * 10 ** (2 * torch.rand(1, generator=g, device="cuda") - 0.5) / (total / 10) ** 0.5).tolist()
    state = {"case": case, "grads": [(randn(*s) * c).to(kind) for s, c in zip(shapes, scale)]}
    if case["kind"] == "clip":
        state["out"] = [torch.empty(s, dtype=getattr(torch, case["out"]), device="cuda") for s in shapes]
    return state


# --- the operators ----------------------------------------------------------------------------------------------------


def _own(s):
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    case = s["case"]
    if case["kind"] != "gated":
        from common import grads

        if case["kind"] == "norm":
            return grads.global_norm(s["grads"])
        norm, out = grads.clipped(s["grads"], 1.0, out=s["out"])
        return [norm, *out]
    from dense_reader import gated

    x, gate, up, act = s["x"], s["gate"], s["up"], case["act"]
    if case["mode"] == "alone":
        return gated.gated(x, gate, up, act)
    weights = case.get("weights", True)
    if case["mode"] == "again":
        out = gated.gated_grads(x, gate, up, s["dh"], act, w_grad=weights)
    else:
        h, kept = gated.gated_keep(x, gate, up, act)
        out = (h, *gated.gated_grads(x, gate, up, s["dh"], act, kept=kept, w_grad=weights))
    return [t for t in out if t is not None]


def _plain_grads(s):
    case = s["case"]
    squares = torch.stack([t.float().square().sum() for t in s["grads"]])
    norm = squares.double().sum().sqrt()
    if case["kind"] == "norm":
        return norm.float()
    factor = (1.0 / (norm + 1e-6)).clamp(max=1.0).float()
    return [norm.float(), *[out.copy_(t.float() * factor) for t, out in zip(s["grads"], s["out"])]]


def _plain(s):
    case = s["case"]
    if case["kind"] != "gated":
        return _plain_grads(s)
    x, gate, up = s["x"].float(), s["gate"].float(), s["up"].float()
    g, u = x @ gate.T, x @ up.T
    if case["act"] == "swiglu":
        p = 1 / (1 + (-g).exp())
        slope = p * (1 + g * (1 - p))
    else:
        c = 2 * math.sqrt(2 / math.pi)
        p = 1 / (1 + (-c * (g + 0.044715 * g**3)).exp())
        slope = p * (1 + g * (1 - p) * c * (1 + 3 * 0.044715 * g * g))
    a = g * p
    h = (a * u).to(torch.bfloat16)
    if case["mode"] == "alone":
        return h
    dh = s["dh"].float()
    dg, du = dh * u * slope, dh * a
    out = [] if case["mode"] == "again" else [h]
    out.append((dg @ gate + du @ up).to(torch.bfloat16))
    if case.get("weights", True):
        out += [(dg.T @ x).to(torch.bfloat16), (du.T @ x).to(torch.bfloat16)]
    return out


def run(state):
    return _own(state) if own else _plain(state)


# --- what a pass cannot do without ------------------------------------------------------------------------------------


def work(case):
    if case["kind"] != "gated":
        size = lambda t: 4 if t == "float32" else 2
        total = sum(math.prod(s) for s in _shapes(case))
        if case["kind"] == "norm":
            return {"bytes": total * size(case["type"]) + 4, "flops": 2 * total}
        return {"bytes": total * (size(case["type"]) + size(case["out"])) + 4, "flops": 3 * total}
    n, d, f, weights = case["n"], case["d"], case["f"], case.get("weights", True)
    moved, products = 2 * n * d + 4 * f * d, 2
    if case["mode"] != "again":
        moved += 2 * n * f
    if case["mode"] != "alone":
        moved += 2 * n * f + 2 * n * d + (4 * f * d if weights else 0)
        products += 4 if weights else 2
    return {"bytes": moved, "flops": 2 * products * n * d * f}


# --- the definition in 64 bits ----------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] != "gated":
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(t.double()) for t in s["grads"]]))
        if case["kind"] == "norm":
            return norm
        return [norm, *[t.double() * torch.minimum(norm.new_ones(()), 1.0 / (norm + 1e-6)) for t in s["grads"]]]
    weights = case.get("weights", True)
    x = s["x"].double().requires_grad_()
    gate, up = (s[k].double().requires_grad_(weights) for k in ("gate", "up"))
    act = torch.nn.functional.silu if case["act"] == "swiglu" else lambda t: torch.nn.functional.gelu(t, approximate="tanh")
    h = act(torch.nn.functional.linear(x, gate)) * torch.nn.functional.linear(x, up)
    if case["mode"] == "alone":
        return h.detach()
    out = list(torch.autograd.grad(h, [x, gate, up] if weights else [x], s["dh"].double()))
    return out if case["mode"] == "again" else [h.detach(), *out]
