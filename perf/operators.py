"""Cases of the operators at the end of a training step, for timing and for comparison with their plain forms.

* ``loss``: cross entropy of a language-model head taken from the hidden states, the head's weight and the targets, with
  the gradients of both (``ops.functional.linear_cross_entropy``), or without a gradient as per-token scores.
* ``clip``: the norm over a list of gradient tensors and their scaling to a maximum norm, in place
  (``ops.functional.clip_grad_norm_``).

``own`` is false for the plain forms (elementary torch operations in 32 bits, rounded once at the end) and true for the
calls of this framework.
"""
import math
import random

import torch

own = False

IGNORE = -100


def listed():
    return [
        # --- the loss of one micro-batch of a training step, with its gradients
        # four sequences of 4096 tokens of the benchmark's model; the last position of a sequence has no target
        {"name": "loss_16384x2048x50304", "op": "loss", "mode": "mean", "tokens": 16384, "hidden": 2048, "vocab": 50304, "ignored": 4 / 16384},
        # one sequence of it
        {"name": "loss_4096x2048x50304", "op": "loss", "mode": "mean", "tokens": 4096, "hidden": 2048, "vocab": 50304, "ignored": 1 / 4096},
        # the widest head among the model families
        {"name": "loss_4096x7168x129280", "op": "loss", "mode": "mean", "tokens": 4096, "hidden": 7168, "vocab": 129280, "ignored": 1 / 4096},
        # a ragged batch: a third of the positions is padding, no size is a multiple of a tile; a summed loss
        {"name": "loss_1037x1000x32001", "op": "loss", "mode": "sum", "tokens": 1037, "hidden": 1000, "vocab": 32001, "ignored": 1 / 3},
        # per-token weights on the losses (a gradient for every row of its own)
        {"name": "loss_weighted_2048x4096x128256", "op": "loss", "mode": "weighted", "tokens": 2048, "hidden": 4096, "vocab": 128256, "ignored": 0.0},
        # the model of a quick test: launches and host time count
        {"name": "loss_512x512x1024", "op": "loss", "mode": "mean", "tokens": 512, "hidden": 512, "vocab": 1024, "ignored": 2 / 512},
        # scoring without a gradient: a document, and a single token
        {"name": "score_2000x2048x50304", "op": "loss", "mode": "score", "tokens": 2000, "hidden": 2048, "vocab": 50304, "ignored": 0.0},
        {"name": "score_1x4096x128256", "op": "loss", "mode": "score", "tokens": 1, "hidden": 4096, "vocab": 128256, "ignored": 0.0},
        # --- clipping before the optimizer's update
        # a dense model of 1.2e9 parameters in bf16, one gradient for each of its 147 tensors
        {"name": "clip_dense_16x2048", "op": "clip", "layout": "dense", "layers": 16, "hidden": 2048, "inter": 8192, "vocab": 50304, "experts": 0, "norm": "l2"},
        # experts held as modules of their own: many small tensors
        {"name": "clip_experts_4x64", "op": "clip", "layout": "dense", "layers": 4, "hidden": 2048, "inter": 1024, "vocab": 50304, "experts": 64, "norm": "l2"},
        # the model of a quick test: everything fits in the cache, launches and host time count
        {"name": "clip_dense_2x512", "op": "clip", "layout": "dense", "layers": 2, "hidden": 512, "inter": 1024, "vocab": 1024, "experts": 0, "norm": "l2"},
        # bf16 and fp32 gradients of any length that start at any element of their buffers, largest absolute value
        {"name": "clip_odd_300", "op": "clip", "layout": "odd", "count": 300, "largest": 1000003, "sizes": 5, "norm": "inf"},
    ]


MOST_LOSS = 4096 * 7168 * 129280 / 4  # tokens x hidden x vocabulary of the costliest drawn loss
MOST_CLIP = 200_000_000               # elements of the largest drawn list of gradients


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.6:
        mode = rng.choice(["mean", "mean", "sum", "weighted", "score"])
        hidden, vocab, tokens = 8 * _log(rng, 4, 700), _log(rng, 40, 131072), _log(rng, 1, 12000)
        tokens = max(1, min(tokens, int(MOST_LOSS / (hidden * vocab))))
        ignored = rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.9), 3)])
        return {"op": "loss", "mode": mode, "tokens": tokens, "hidden": hidden, "vocab": vocab, "ignored": ignored}
    norm = rng.choice(["l2", "l2", "l2", "inf"])
    if rng.random() < 0.4:
        hidden = 8 * _log(rng, 8, 256)
        inter = 8 * rng.randrange(hidden // 16, hidden // 2)
        experts = rng.choice([0, rng.randrange(2, 32)])
        vocab = _log(rng, 500, 60000)
        a_layer = 4 * hidden * hidden + 3 * max(1, experts) * hidden * inter
        layers = max(1, min(_log(rng, 1, 24), (MOST_CLIP - 2 * vocab * hidden) // a_layer))
        return {"op": "clip", "layout": "dense", "layers": layers, "hidden": hidden, "inter": inter, "vocab": vocab, "experts": experts, "norm": norm}
    count = _log(rng, 1, 1500)
    largest = max(1, min(_log(rng, 2, 3_000_000), MOST_CLIP // count))
    return {"op": "clip", "layout": "odd", "count": count, "largest": largest, "sizes": rng.randrange(1 << 20), "norm": norm}


# ------------------------------------------------------------------ what a program has in hand
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _n_ignored(case):
    return min(case["tokens"] - 1, int(round(case["tokens"] * case["ignored"])))


def _prepare_loss(case, seed):
    g = _generator(seed)
    T, H, V = case["tokens"], case["hidden"], case["vocab"]
    # a head as it is initialised, and hidden states behind a norm that lean towards their targets: a loss between that
    # of a new model and that of a trained one; frequent tokens have low numbers, as a tokenizer gives them
    weight = torch.empty((V, H), dtype=torch.bfloat16, device="cuda").normal_(0.0, 0.02, generator=g)
    x = torch.randn((T, H), device="cuda", generator=g)
    targets = (V * torch.rand(T, device="cuda", generator=g).double().pow(4)).long().clamp_(max=V - 1)
    towards = weight[targets].float()
    x = x + 5.0 * towards / towards.square().sum(1, keepdim=True)
    order = torch.randperm(T, device="cuda", generator=g)
    targets[order[:_n_ignored(case)]] = IGNORE
    state = {"op": "loss", "mode": case["mode"], "x": x.to(torch.bfloat16), "weight": weight, "targets": targets}
    if case["mode"] == "weighted":
        state["row_grad"] = torch.rand(T, device="cuda", generator=g) / T
    if case["mode"] != "score":
        state["x"].requires_grad_()
        state["weight"].requires_grad_()
    return state


def _shapes(case):
    """(numel, dtype, element offset modulo 64) of every gradient."""
    if case["layout"] == "odd":
        r = random.Random(case["sizes"])
        return [(int(round(math.exp(r.uniform(0.0, math.log(case["largest"]))))), torch.float32 if r.random() < 0.3 else torch.bfloat16,
                 r.randrange(64)) for _ in range(case["count"])]
    H, inter, V = case["hidden"], case["inter"], case["vocab"]
    sizes = [V * H]
    for _ in range(case["layers"]):
        sizes += [H * H] * 4 + [H] * 2
        if case["experts"]:
            sizes += [case["experts"] * H]
        sizes += [inter * H] * (3 * max(1, case["experts"]))
    sizes += [H, V * H]
    return [(n, torch.bfloat16, 0) for n in sizes]


def _prepare_clip(case, seed):
    g, r = _generator(seed), random.Random(seed)
    todo = _shapes(case)
    total = sum(n for n, _, _ in todo)
    room = {torch.bfloat16: 0, torch.float32: 0}
    places = []
    for n, dtype, shift in todo:  # one buffer for each type, and the gradients as pieces of it: allocators give multiples of 64 elements
        at = (room[dtype] + 63) // 64 * 64 + shift
        places.append((dtype, at, n))
        room[dtype] = at + n
    flats = {t: torch.zeros(max(1, n), dtype=t, device="cuda") for t, n in room.items()}
    grads = []
    for k, (dtype, at, n) in enumerate(places):
        piece = flats[dtype][at:at + n]
        # layers differ in scale; an expert or a row that saw no token has a gradient of zeros
        if k == 0 or r.random() > 0.03:
            piece.normal_(0.0, 6.0 / math.sqrt(total) * math.exp(r.gauss(0.0, 0.7)), generator=g)
        grads.append(piece)
    # a norm of about six (for the largest value: about 1e-3 of its own) against the limit
    limit = 1.0 if case["norm"] == "l2" else 6.0 / math.sqrt(total)
    return {"op": "clip", "norm": case["norm"], "grads": grads, "flats": list(flats.values()), "limit": limit}


def prepare(case, seed):
    return _prepare_loss(case, seed) if case["op"] == "loss" else _prepare_clip(case, seed)


# ------------------------------------------------------------------ one pass
def _plain_loss(state):
    mode, targets = state["mode"], state["targets"]
    x, w = state["x"].detach().float(), state["weight"].detach().float()
    logits = x @ w.t()
    valid = targets >= 0
    column = targets.clamp(min=0)[:, None]
    top = logits.amax(1, keepdim=True)
    at_target = logits.gather(1, column) - top
    e = (logits - top).exp_()
    z = e.sum(1, keepdim=True)
    losses = torch.where(valid, (z.log() - at_target)[:, 0], 0.0)
    if mode == "score":
        return {"losses": losses}
    count = valid.sum()
    if mode == "weighted":
        row = state["row_grad"]
    else:
        row = (1.0 / count if mode == "mean" else torch.ones((), device=x.device)).expand(targets.shape)
    row = torch.where(valid, row, 0.0)[:, None]
    d = e.mul_(row / z)
    d.scatter_add_(1, column, -row)
    dx, dw = (d @ w).to(torch.bfloat16), (d.t() @ x).to(torch.bfloat16)
    if mode == "weighted":
        return {"losses": losses, "dx": dx, "dw": dw}
    loss = losses.sum()
    return {"loss": loss / count if mode == "mean" else loss, "dx": dx, "dw": dw}


def _plain_clip(state, limit):
    grads = state["grads"]
    if state["norm"] == "l2":
        norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    else:
        norm = torch.stack([g.float().abs().max() for g in grads]).max()
    factor = (limit / (norm + 1e-6)).clamp(max=1.0)
    for g in grads:
        g.copy_(g.float() * factor)
    return norm


def run(state):
    if own:
        from optimus_lm_b200.ops import functional as OF
    if state["op"] == "loss":
        if not own:
            with torch.no_grad():
                return _plain_loss(state)
        x, w, targets, mode = state["x"], state["weight"], state["targets"], state["mode"]
        if mode == "score":
            with torch.no_grad():
                return {"losses": OF.linear_cross_entropy(x, w, targets, reduction="none")}
        if mode == "weighted":
            losses = OF.linear_cross_entropy(x, w, targets, reduction="none")
            dx, dw = torch.autograd.grad(losses, (x, w), state["row_grad"])
            return {"losses": losses.detach(), "dx": dx, "dw": dw}
        loss = OF.linear_cross_entropy(x, w, targets, reduction=mode)
        dx, dw = torch.autograd.grad(loss, (x, w))
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    # clipping works in place: the limit falls from pass to pass, so that every pass has something to clip
    limit = state["limit"]
    state["limit"] = limit * 0.999
    if own:
        norm = OF.clip_grad_norm_(state["grads"], limit, norm_type=2.0 if state["norm"] == "l2" else math.inf)
    else:
        norm = _plain_clip(state, limit)
    return {"norm": norm, "grads": state["flats"]}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "loss":
        T, H, V = case["tokens"], case["hidden"], case["vocab"]
        rows = T - _n_ignored(case)
        once = 2 * T * H + 2 * V * H + 8 * T  # hidden states, weight, targets
        if case["mode"] == "score":
            return {"bytes": once + 4 * T, "flops": 2 * rows * H * V}
        return {"bytes": once + 2 * T * H + 2 * V * H, "flops": 6 * rows * H * V}
    todo = _shapes(case)
    size = sum(n * (2 if t == torch.bfloat16 else 4) for n, t, _ in todo)
    return {"bytes": 2 * size, "flops": 3 * sum(n for n, _, _ in todo)}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "clip":
        if case["norm"] == "l2":
            norm = math.sqrt(math.fsum(torch.linalg.vector_norm(g.double()).item() ** 2 for g in state["grads"]))
        else:
            norm = max(g.abs().max().item() for g in state["grads"])
        factor = min(1.0, state["limit"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [f.double() * factor for f in state["flats"]]}
    x, w, t, mode = state["x"].detach().double(), state["weight"].detach().double(), state["targets"], state["mode"]
    weight_of = torch.ones(len(t), dtype=torch.float64, device=x.device)
    if mode == "mean":
        weight_of /= int((t != IGNORE).sum())
    elif mode == "weighted":
        weight_of = state["row_grad"].double()
    losses, dx, dw = [], [], torch.zeros_like(w) if mode != "score" else None
    for lo in range(0, len(t), 2048):
        xs, ts, gs = x[lo:lo + 2048], t[lo:lo + 2048], weight_of[lo:lo + 2048]
        logp = torch.log_softmax(xs @ w.T, dim=1)
        rows = torch.nonzero(ts != IGNORE)[:, 0]
        loss = torch.zeros(len(ts), dtype=torch.float64, device=x.device)
        loss[rows] = -logp[rows, ts[rows]]
        losses.append(loss)
        if mode == "score":
            continue
        d = torch.zeros_like(logp)
        d[rows] = logp[rows].exp()
        d[rows, ts[rows]] -= 1.0
        d *= gs[:, None]
        dx.append(d @ w)
        dw += d.T @ xs
    losses = torch.cat(losses)
    if mode == "score":
        return {"losses": losses}
    if mode == "weighted":
        return {"losses": losses, "dx": torch.cat(dx), "dw": dw}
    return {"loss": (losses * weight_of).sum(), "dx": torch.cat(dx), "dw": dw}
