"""The training losses of the LM head and of the router, each with its gradients: what is timed and compared.

A case is one pass through an operator, as a training, distillation or scoring program makes it:

- token:   the cross entropy of the head's logits against each row's token (lm_head_topk.head_loss), alone (scoring a
           text) or with the gradients of the rows and of the head (training), the logits never in memory;
- distill: the same head against a teacher's best logits of each row (head_loss, in the form linear.topk_merge leaves
           them), forward and backward, of the rows alone (a frozen head) or of both;
- balance: the router's balance loss and each expert's count (moe.balance), with the gradient of the router's logits.

Head rows are N(0, 0.05); a row of x is standard normal with a few channels far larger plus a share of its own token's
head row, so that tokens are known anywhere from not at all to well, as a model in training knows them.
"""

import math
import sys
from pathlib import Path

import torch

own = False


def listed():
    return [
        # the score of one token under a small draft's head: launch and host time count
        {"name": "score_token", "kind": "token", "n": 1, "v": 8192, "valid": 8192, "d": 1024, "counted": 1.0,
         "grads": "none"},
        # the scores of a batch's next tokens under a large head: the head's bytes bound it
        {"name": "score_rows", "kind": "token", "n": 32, "v": 128256, "valid": 128256, "d": 4096, "counted": 1.0,
         "grads": "none"},
        # a small step of a draft's head, a few rows padding
        {"name": "token_small", "kind": "token", "n": 48, "v": 8192, "valid": 8192, "d": 1024, "counted": 0.9,
         "grads": "both"},
        # fine-tuning on answers: most rows are a prompt's and count nothing; the head padded past its real vocabulary
        {"name": "token_answers", "kind": "token", "n": 1003, "v": 50304, "valid": 50257, "d": 2880, "counted": 0.4,
         "grads": "both"},
        # a training step of a large head
        {"name": "token_large", "kind": "token", "n": 8192, "v": 128256, "valid": 128256, "d": 4096, "counted": 1.0,
         "grads": "both"},
        # a draft's head distilled from what a decode step of its teacher left
        {"name": "distill_draft", "kind": "distill", "n": 64, "v": 8192, "valid": 8192, "d": 1024, "k": 8, "t": 1.0,
         "counted": 1.0, "grads": "both"},
        # a ragged batch against a teacher's best sixteen, softened
        {"name": "distill_rows", "kind": "distill", "n": 2047, "v": 128256, "valid": 128256, "d": 2048, "k": 16,
         "t": 2.0, "counted": 0.9, "grads": "both"},
        # the body trained through a frozen head against the best sixty-four
        {"name": "distill_frozen", "kind": "distill", "n": 4096, "v": 32000, "valid": 32000, "d": 4096, "k": 64,
         "t": 1.0, "counted": 1.0, "grads": "x"},
        # the router of a small batch
        {"name": "balance_rows", "kind": "balance", "b": 1, "r": 32, "e": 32, "k": 4, "score": "softmax",
         "counted": 1.0},
        # a batch of padded sequences, a loss for each, many experts scored by sigmoid
        {"name": "balance_batch", "kind": "balance", "b": 8, "r": 4096, "e": 256, "k": 8, "score": "sigmoid",
         "counted": 0.8},
        # one long flat batch
        {"name": "balance_flat", "kind": "balance", "b": 1, "r": 20011, "e": 128, "k": 4, "score": "softmax",
         "counted": 1.0},
    ]


# --- drawn cases ------------------------------------------------------------------------------------------------------


def _log(rng, lo, hi, step=1):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step))


def draw(rng):
    kind = rng.choice(("token", "token", "distill", "distill", "balance"))
    counted = rng.choice((1.0, 1.0, 0.9, 0.4))
    if kind == "balance":
        e = 32 * rng.randint(1, 8)
        b = rng.choice((1, 1, 2, 5, 8))
        return {"kind": kind, "b": b, "r": _log(rng, 1, 32768 // b), "e": e, "k": rng.randint(1, 8),
                "score": rng.choice(("softmax", "sigmoid")), "counted": counted}
    v = _log(rng, 1000, 128256)
    case = {"kind": kind, "n": _log(rng, 1, 8192), "v": v, "valid": v - rng.choice((0, 0, 1, 47)),
            "d": _log(rng, 512, 4096, 8), "counted": counted}
    if kind == "token":
        return {**case, "grads": rng.choice(("none", "both", "both", "x"))}
    return {**case, "k": rng.randint(1, 64), "t": rng.choice((1.0, 1.0, 2.0, 0.7)),
            "grads": rng.choice(("none", "both", "both", "x"))}


# --- inputs -----------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    randint = lambda hi, *s: torch.randint(0, hi, s, generator=g, device="cuda")
    if case["kind"] == "balance":
        b, r, e, k = case["b"], case["r"], case["e"], case["k"]
        logits = randn(b, r, e) * 1.5 + randn(e)  # (some experts liked more than others)
        ids = logits.topk(k, dim=-1).indices.to(torch.int16)
        # sequences of different lengths, padded to the longest
        lengths = (r * (case["counted"] + (1 - case["counted"]) * (rand(b) - 0.5))).ceil().clamp(1, r)
        mask = None if case["counted"] == 1.0 else torch.arange(r, device="cuda") < lengths[:, None]
        return {"case": case, "logits": logits, "ids": ids, "mask": mask, "g": 0.5 + rand(b)}
    n, v, valid, d = case["n"], case["v"], case["valid"], case["d"]
    head = (randn(v, d) * 0.05).to(torch.bfloat16)
    targets = randint(valid, n)
    x = randn(n, d)
    x[:, :4] *= 8
    x += (6 * rand(n, 1) / (d * 0.0025)) * head[targets].float()
    x = x.to(torch.bfloat16)
    counts = rand(n) < case["counted"]
    counts[0] = True
    state = {"case": case, "x": x, "head": head, "g": torch.full((n,), 1.0 / n, device="cuda")}
    if case["kind"] == "token":
        state["targets"] = torch.where(counts, targets, -100)
        return state
    # a teacher's best k, in decreasing order: other ids than each other, some rows with fewer than k of them
    k = case["k"]
    gaps = 1 + (rand(n, k) * (valid // k - 1)).long()
    ids = (targets[:, None] + gaps.cumsum(1) - gaps[:, :1]) % valid
    vals = 12.0 - (rand(n, k) * 0.8).cumsum(1)
    fewer = torch.where(rand(n) < 0.1, randint(k, n) + 1, k)
    held = (torch.arange(k, device="cuda") < fewer[:, None]) & counts[:, None]
    state["ids"] = torch.where(held, ids, -1).to(torch.int32)
    state["vals"] = torch.where(held, vals, -math.inf)
    return state


# --- the operators ----------------------------------------------------------------------------------------------------


def _own(s):
    sys.path[:0] = [p for p in [str(Path(__file__).resolve().parents[1] / "tensix-kernels_amd")] if p not in sys.path]
    case = s["case"]
    if case["kind"] == "balance":
        from moe import balance

        return balance.balance_loss_grads(s["logits"], s["ids"], case["k"], g=s["g"], kind=case["score"],
                                          mask=s["mask"])
    from lm_head_topk import head_loss

    grads = case["grads"]
    if case["kind"] == "token":
        if grads == "none":
            return head_loss.token_loss(s["x"], s["head"], s["targets"], valid=case["valid"])
        out = head_loss.token_loss_grads(s["x"], s["head"], s["targets"], g=s["g"], valid=case["valid"],
                                         head_grad=grads == "both")
    else:
        if grads == "none":
            return head_loss.distill_loss(s["x"], s["head"], s["vals"], s["ids"], temperature=case["t"],
                                          valid=case["valid"])
        out = head_loss.distill_loss_grads(s["x"], s["head"], s["vals"], s["ids"], g=s["g"], temperature=case["t"],
                                           valid=case["valid"], head_grad=grads == "both")
    return [t for t in out if t is not None]


def _plain_balance(s):
    case, logits, ids = s["case"], s["logits"].float(), s["ids"].long()
    b, r, e = logits.shape
    m = torch.ones(b, r, device=logits.device) if s["mask"] is None else s["mask"].float()
    if case["score"] == "softmax":
        z = (logits - logits.amax(-1, keepdim=True)).exp()
        p = z / z.sum(-1, keepdim=True)
        inner = p
    else:
        sg = 1 / (1 + (-logits).exp())
        p = sg / sg.sum(-1, keepdim=True)
        inner = p * (1 - sg)
    counts = torch.zeros(b, e, device=logits.device).scatter_add_(1, ids.reshape(b, -1), m.repeat_interleave(ids.shape[-1], 1))
    rows = m.sum(1)[:, None].clamp(min=1)
    f = e * counts / counts.sum(1, keepdim=True).clamp(min=1)
    loss = (f * (p * m[..., None]).sum(1) / rows).sum(1)
    mean = (p * f[:, None]).sum(-1, keepdim=True)
    dlogits = (s["g"][:, None] / rows * m)[..., None] * inner * (f[:, None] - mean)
    return loss, counts.to(torch.int32), dlogits


def _plain(s):
    case = s["case"]
    if case["kind"] == "balance":
        return _plain_balance(s)
    x, head, g = s["x"].float(), s["head"][: case["valid"]].float(), s["g"]
    t = case.get("t", 1.0)
    z = (x @ head.T) / t
    top = z.amax(1, keepdim=True)
    lse = (z - top).exp().sum(1, keepdim=True).log() + top
    if case["kind"] == "token":
        counts = s["targets"] >= 0
        ids = s["targets"].clamp(min=0)[:, None]
        q = counts.float()[:, None]
        loss = torch.where(counts, (lse - z.gather(1, ids))[:, 0], 0.0)
    else:
        held = s["ids"] >= 0
        counts = held.any(1)
        ids = s["ids"].clamp(min=0).long()
        vals = torch.where(held, s["vals"] / t, -math.inf)
        best = vals.amax(1, keepdim=True).clamp(min=-1e30)
        e = (vals - best).exp()
        total = e.sum(1, keepdim=True).clamp(min=1e-30)
        q = e / total
        logq = torch.where(held, vals - best - total.log(), 0.0)
        loss = (q * (logq - z.gather(1, ids) + lse)).sum(1)
    if case["grads"] == "none":
        return loss
    dz = (z - lse).exp() * counts[:, None]
    dz.scatter_add_(1, ids, -q)
    dz *= (g / t)[:, None]
    dx = (dz @ head).to(torch.bfloat16)
    if case["grads"] == "x":
        return [loss, dx]
    dhead = torch.zeros_like(s["head"])
    dhead[: case["valid"]] = (dz.T @ x).to(torch.bfloat16)
    return [loss, dx, dhead]


def run(state):
    return _own(state) if own else _plain(state)


# --- what a pass cannot do without ------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "balance":
        rows = case["b"] * case["r"]
        return {"bytes": rows * (8 * case["e"] + 2 * case["k"]) + 4 * case["b"] * case["e"],
                "flops": 12 * rows * case["e"]}
    n, v, d = case["n"], case["valid"], case["d"]
    rows = max(1, round(n * case["counted"]))
    products = {"none": 1, "x": 2, "both": 3}[case["grads"]]
    moved = 2 * v * d + 2 * rows * d + n * (12 * case["k"] if case["kind"] == "distill" else 8) + 4 * n
    if products > 1:
        moved += 2 * n * d
    if products > 2:
        moved += 2 * case["v"] * d
    return {"bytes": moved, "flops": 2 * products * rows * v * d}


# --- the definition in 64 bits ----------------------------------------------------------------------------------------


def _exact_balance(s):
    case = s["case"]
    losses, counts, grads = [], [], []
    for b in range(case["b"]):
        logits = s["logits"][b].double().requires_grad_()
        on = torch.ones(case["r"], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"][b]
        kept = logits[on]
        p = torch.softmax(kept, 1) if case["score"] == "softmax" else torch.sigmoid(kept)
        p = p / p.sum(1, keepdim=True)
        c = torch.bincount(s["ids"][b][on].long().flatten(), minlength=case["e"])
        loss = case["e"] * (c.double() / c.sum()) @ p.mean(0)
        grads.append(torch.autograd.grad(loss * s["g"][b].double(), logits)[0])
        losses.append(loss.detach())
        counts.append(c.to(torch.int32))
    return torch.stack(losses), torch.stack(counts), torch.stack(grads)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "balance":
        return _exact_balance(s)
    t, v = case.get("t", 1.0), case["valid"]
    if case["kind"] == "token":
        on = s["targets"] >= 0
        want = torch.zeros(case["n"], 1, dtype=torch.float64, device="cuda")
        want[on] = 1.0
        ids = s["targets"][:, None].clamp(min=0)
        entropy = 0.0
    else:
        on = (s["ids"] >= 0).any(1)
        ids = s["ids"].long().clamp(min=0)
        want = torch.softmax((s["vals"].double() / t)[on], 1)
        want = torch.zeros(case["n"], case["k"], dtype=torch.float64, device="cuda").index_put_((on,), want)
        entropy = torch.special.entr(want).sum(1)
    x, head = s["x"].double(), s["head"][:v].double()
    logp = torch.log_softmax(x @ head.T / t, 1)
    loss = -(want * logp.gather(1, ids)).sum(1) - entropy
    if case["grads"] == "none":
        return loss
    dz = logp.exp_()
    dz[~on] = 0.0
    dz.scatter_add_(1, ids, -want)
    dz *= (s["g"].double() / t)[:, None]
    out = [loss, dz @ head]
    if case["grads"] == "both":
        dhead = torch.zeros(case["v"], case["d"], dtype=torch.float64, device="cuda")
        dhead[:v] = dz.T @ x
        out.append(dhead)
    return out
