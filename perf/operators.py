"""The operators of a language model's input and output ends, and of its training step, as one program calls them.

  embedding            rows of a token table, scaled                      (mtc_embedding)
  embedding_grad       the table's gradient, token by token               (mtc_embedding_grad)
  cross_entropy        softmax cross entropy of x.W^T + b at the targets  (mtc_linear_cross_entropy)
  cross_entropy_grad   the same with the gradients of x, W and b          (mtc_linear_cross_entropy_grad)
  clip                 gradients scaled to a global norm                  (mtc_clip_global_norm)

A case names its operator in "op".  `run` takes the plain form (elementary torch
operations, float32) or, where `own` is true, the calls of minitensor_cpp_b200.abi.
"""
import math

import torch

own = False

DEVICE = "cuda"
IGNORE = -100  # target of a position that has no loss (a prompt's tokens, padding)
PADDING = 0    # token of a padded position


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # one generated token's row: a decoding step, launch latency only
        {"name": "embedding one token", "op": "embedding", "vocab": 32000, "dim": 1024, "tokens": 1, "padding": False},
        # a ragged batch of prompts, wide rows
        {"name": "embedding prompts", "op": "embedding", "vocab": 32000, "dim": 4096, "tokens": 4099, "padding": True},
        # a small training step: as many positions as half the vocabulary
        {"name": "embedding grad step", "op": "embedding_grad", "vocab": 32000, "dim": 1024, "tokens": 16384,
         "padding": False},
        # a large training step with padded sequences; frequent tokens own thousands of positions
        {"name": "embedding grad large", "op": "embedding_grad", "vocab": 131072, "dim": 2048, "tokens": 65536,
         "padding": True},
        # the log-probability of one token: scoring while decoding
        {"name": "loss one token", "op": "cross_entropy", "vocab": 32000, "dim": 1024, "rows": 1, "ignored": 0.0,
         "bias": False},
        # evaluation of a batch, prompts without loss
        {"name": "loss evaluation", "op": "cross_entropy", "vocab": 32000, "dim": 1024, "rows": 4096, "ignored": 0.25,
         "bias": False},
        # the output layer of the spiral MLP (64 -> 3, 300 points): the smallest training step of this repository
        {"name": "loss grad spiral", "op": "cross_entropy_grad", "vocab": 3, "dim": 64, "rows": 300, "ignored": 0.0,
         "bias": True},
        # odd sizes everywhere: nothing is a multiple of a tile or of 16 bytes
        {"name": "loss grad odd", "op": "cross_entropy_grad", "vocab": 50003, "dim": 771, "rows": 1031, "ignored": 0.1,
         "bias": True},
        # the output layer of the wide MLP (8192 -> 1000) at its global batch
        {"name": "loss grad wide MLP", "op": "cross_entropy_grad", "vocab": 1000, "dim": 8192, "rows": 65536,
         "ignored": 0.0, "bias": True},
        # a training step over a large vocabulary, a quarter of the positions without loss
        {"name": "loss grad large", "op": "cross_entropy_grad", "vocab": 131072, "dim": 2048, "rows": 8192,
         "ignored": 0.25, "bias": False},
        # the spiral MLP's parameters (2 -> 64 -> 64 -> 3): six small tensors
        {"name": "clip spiral", "op": "clip", "layout": "2,64,64,3", "tensors": 6, "elements": 4547, "over": 4.0},
        # the wide MLP's parameters (1024 -> 8192 x 3 -> 1000): eight tensors, 0.6 GB
        {"name": "clip wide MLP", "op": "clip", "layout": "1024,8192,8192,8192,1000", "tensors": 8,
         "elements": 150823912, "over": 4.0},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["embedding", "embedding_grad", "cross_entropy", "cross_entropy_grad", "clip"])
    if op in ("embedding", "embedding_grad"):
        return {"op": op, "vocab": _log_int(rng, 1000, 131072), "dim": _log_int(rng, 64, 4096),
                "tokens": _log_int(rng, 1, 32768), "padding": rng.random() < 0.5}
    if op in ("cross_entropy", "cross_entropy_grad"):
        case = {"op": op, "vocab": _log_int(rng, 3, 131072), "dim": _log_int(rng, 64, 4096),
                "rows": _log_int(rng, 1, 16384), "ignored": rng.choice([0.0, 0.1, 0.25, 0.9]),
                "bias": rng.random() < 0.5}
        most = 8192 * 131072 * 2048
        while case["vocab"] * case["dim"] * case["rows"] > most:
            case["rows"] = (case["rows"] + 1) // 2
        return case
    tensors = _log_int(rng, 1, 400)
    return {"op": op, "layout": "", "tensors": tensors, "elements": _log_int(rng, 100 * tensors, 150000000),
            "over": rng.choice([0.5, 4.0, 100.0])}


# ----------------------------------------------------------------- inputs --

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _token_rates(vocab):
    """Zipf-Mandelbrot frequencies, the law that word counts follow."""
    rate = 1.0 / (torch.arange(vocab, dtype=torch.float64, device=DEVICE) + 2.7)
    return rate / rate.sum()


def _tokens(vocab, count, padding, g):
    edges = _token_rates(vocab).cumsum(0)
    at = torch.rand(count, dtype=torch.float64, device=DEVICE, generator=g)
    rank = torch.searchsorted(edges, at).clamp_(max=vocab - 1)
    order = torch.randperm(vocab, device=DEVICE, generator=g)  # frequency is no order of a tokenizer's ids
    tokens = order[rank]
    if padding:
        tokens = torch.where(torch.rand(count, device=DEVICE, generator=g) < 0.1, PADDING, tokens)
    return tokens


def _layers(case):
    """The shapes of a dense MLP's weights and biases."""
    widths = [int(w) for w in case["layout"].split(",")]
    return [s for a, b in zip(widths, widths[1:]) for s in ((b, a), (b,))]


def _pieces(case):
    """Sizes of many parameters, large and small in turn, that share one buffer."""
    share = [1.0 if i % 3 else 40.0 for i in range(case["tensors"])]
    return [max(1, int(case["elements"] * s / sum(share))) for s in share]


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    state = {"op": op, "case": case}
    if op in ("embedding", "embedding_grad"):
        state["tokens"] = _tokens(case["vocab"], case["tokens"], case["padding"], g)
        state["scale"] = math.sqrt(case["dim"])
        state["padding"] = PADDING if case["padding"] else None
        rows = case["vocab"] if op == "embedding" else case["tokens"]
        state["x"] = torch.randn(rows, case["dim"], device=DEVICE, generator=g) * 0.02
    elif op in ("cross_entropy", "cross_entropy_grad"):
        n, v, d = case["rows"], case["vocab"], case["dim"]
        # logits of a half-trained model: spread 2, the target's raised by 6
        w = torch.randn(v, d, device=DEVICE, generator=g) * (2.0 / math.sqrt(d))
        t = _tokens(v, n, False, g)
        x = torch.randn(n, d, device=DEVICE, generator=g)
        x += 3.0 * w[t] / w[t].norm(dim=1, keepdim=True)
        if case["ignored"] > 0:
            keep = torch.rand(n, device=DEVICE, generator=g) >= case["ignored"]
            keep[n // 2] = True
            t = torch.where(keep, t, IGNORE)
        count = (t != IGNORE).sum().clamp(min=1)
        state["x"], state["w"], state["t"] = x, w, t
        state["b"] = torch.randn(v, device=DEVICE, generator=g) * 0.5 if case["bias"] else None
        state["dloss"] = (1.0 / count.float()).reshape(1).expand(n)  # of the mean over the positions with a loss
    else:
        if case["layout"]:
            state["grads"] = [torch.randn(s, device=DEVICE, generator=g) * 1e-3 for s in _layers(case)]
        else:  # views of one buffer, back to back: a gradient bucket
            flat = torch.randn(sum(_pieces(case)), device=DEVICE, generator=g) * 1e-3
            state["grads"] = list(flat.split(_pieces(case)))
        norm = 1e-3 * math.sqrt(sum(t.numel() for t in state["grads"]))
        state["max_norm"] = norm / case["over"]
    return state


# -------------------------------------------------------------- the calls --

def _plain(state):
    op = state["op"]
    if op == "embedding":
        out = state["x"][state["tokens"]] * state["scale"]
        if state["padding"] is not None:
            out = out * (state["tokens"] != state["padding"]).unsqueeze(1)
        return out
    if op == "embedding_grad":
        d = state["x"] * state["scale"]
        if state["padding"] is not None:
            d = d * (state["tokens"] != state["padding"]).unsqueeze(1)
        table = torch.zeros(state["case"]["vocab"], d.shape[1], device=d.device)
        return table.index_add_(0, state["tokens"], d)
    if op in ("cross_entropy", "cross_entropy_grad"):
        x, w, t, b = state["x"], state["w"], state["t"], state["b"]
        keep = t != IGNORE
        at = torch.where(keep, t, 0)
        row = torch.arange(t.numel(), device=t.device)
        z = x @ w.t()
        if b is not None:
            z = z + b
        top = z.amax(dim=1, keepdim=True)
        zt = z[row, at]
        e = torch.exp(z - top)
        s = e.sum(dim=1, keepdim=True)
        lse = (top + torch.log(s)).squeeze(1)
        loss = torch.where(keep, lse - zt, 0.0)
        if op == "cross_entropy":
            return {"loss": loss, "lse": lse * keep}
        g = e / s
        g[row, at] -= 1.0
        g *= (state["dloss"] * keep).unsqueeze(1)
        out = {"loss": loss, "dx": g @ w, "dw": g.t() @ x}
        if b is not None:
            out["db"] = g.sum(dim=0)
        return out
    norm = torch.stack([(t * t).sum() for t in state["grads"]]).sum().sqrt()
    scale = torch.clamp(state["max_norm"] / norm, max=1.0)
    outs = [t * scale for t in state["grads"]]
    return {"norm": norm, "grads": outs if state["case"]["layout"] else torch.cat(outs)}


def _own(state):
    from minitensor_cpp_b200 import abi

    view = abi.View.of
    op = state["op"]
    if op == "embedding":
        table, tokens = state["x"], state["tokens"]
        out = torch.empty(tokens.numel(), table.shape[1], device=table.device)
        abi.embedding(view(table), view(tokens), view(out), scale=state["scale"], padding_token=state["padding"])
        return out
    if op == "embedding_grad":
        d, tokens = state["x"], state["tokens"]
        table = torch.empty(state["case"]["vocab"], d.shape[1], device=d.device)
        abi.embedding_grad(view(d), view(tokens), view(table), scale=state["scale"], padding_token=state["padding"])
        return table
    if op in ("cross_entropy", "cross_entropy_grad"):
        x, w, t, b = state["x"], state["w"], state["t"], state["b"]
        bias = None if b is None else view(b)
        loss = torch.empty(t.numel(), device=x.device)
        if op == "cross_entropy":
            lse = torch.empty(t.numel(), device=x.device)
            abi.linear_cross_entropy(view(x), view(w), view(t), view(loss), bias=bias, lse=view(lse),
                                     ignore_target=IGNORE)
            return {"loss": loss, "lse": lse}
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        db = None if b is None else torch.empty_like(b)
        abi.linear_cross_entropy_grad(view(x), view(w), view(t), view(state["dloss"]), dx=view(dx), dweight=view(dw),
                                      bias=bias, dbias=None if b is None else view(db), loss=view(loss),
                                      ignore_target=IGNORE)
        out = {"loss": loss, "dx": dx, "dw": dw}
        if b is not None:
            out["db"] = db
        return out
    if state["case"]["layout"]:
        bucket = outs = [torch.empty_like(t) for t in state["grads"]]
    else:
        bucket = torch.empty(sum(t.numel() for t in state["grads"]), device=DEVICE)
        outs = bucket.split([t.numel() for t in state["grads"]])
    norm = torch.empty((), device=DEVICE)
    abi.clip_global_norm([view(t) for t in state["grads"]], state["max_norm"], view(norm), outs=[view(t) for t in outs])
    return {"norm": norm, "grads": bucket}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------ what it cannot do without --

def work(case):
    op = case["op"]
    if op in ("embedding", "embedding_grad"):
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        if op == "embedding_grad":  # every gradient row read, the whole table written
            return {"bytes": 4.0 * n * d + 8.0 * n + 4.0 * v * d, "flops": 1.0 * n * d}
        rate = 1.0 / (torch.arange(v, dtype=torch.float64) + 2.7)
        seen = float((1.0 - (1.0 - rate / rate.sum()) ** n).sum())  # distinct tokens, expected
        return {"bytes": 4.0 * seen * d + 8.0 * n + 4.0 * n * d, "flops": 1.0 * n * d}
    if op in ("cross_entropy", "cross_entropy_grad"):
        n, v, d = case["rows"], case["vocab"], case["dim"]
        live = max(1.0, n * (1.0 - case["ignored"]))  # a position without a loss needs no product
        read = 4.0 * (live * d + v * d + (v if case["bias"] else 0)) + 8.0 * n
        if op == "cross_entropy":
            return {"bytes": read + 8.0 * n, "flops": 2.0 * live * v * d}
        wrote = 4.0 * (n * d + v * d + (v if case["bias"] else 0) + n)
        return {"bytes": read + wrote + 4.0, "flops": 6.0 * live * v * d}
    return {"bytes": 8.0 * case["elements"] + 4.0, "flops": 3.0 * case["elements"]}


# ------------------------------------------------- the definitions, in 64 bits --

def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "embedding":
        out = state["x"].double().index_select(0, state["tokens"]).mul_(state["scale"])
        if state["padding"] is not None:
            out[state["tokens"] == state["padding"]] = 0.0
        return out
    if op == "embedding_grad":
        live = torch.ones_like(state["tokens"], dtype=torch.bool)
        if state["padding"] is not None:
            live = state["tokens"] != state["padding"]
        out = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device=DEVICE)
        out.index_put_((state["tokens"][live],), state["x"][live].double() * state["scale"], accumulate=True)
        return out
    if op in ("cross_entropy", "cross_entropy_grad"):
        n = case["rows"]
        w = state["w"].double()
        b = 0.0 if state["b"] is None else state["b"].double()
        loss = torch.zeros(n, dtype=torch.float64, device=DEVICE)
        lse = torch.zeros_like(loss)
        grads = op == "cross_entropy_grad"
        dx = torch.zeros(n, case["dim"], dtype=torch.float64, device=DEVICE) if grads else None
        dw = torch.zeros_like(w) if grads else None
        db = torch.zeros(case["vocab"], dtype=torch.float64, device=DEVICE)
        live = (state["t"] != IGNORE).nonzero().squeeze(1)
        for rows in live.split(2048):
            x = state["x"][rows].double()
            logp = torch.addmm(b, x, w.t()) if state["b"] is not None else torch.mm(x, w.t())
            total = torch.logsumexp(logp, dim=1)
            logp -= total.unsqueeze(1)
            t = state["t"][rows].unsqueeze(1)
            loss[rows] = -logp.gather(1, t).squeeze(1)
            lse[rows] = total
            if not grads:
                continue
            g = logp.exp_()
            g.scatter_add_(1, t, torch.full_like(t, -1.0, dtype=torch.float64))
            g *= state["dloss"][rows].double().unsqueeze(1)
            dx[rows] = g.mm(w)
            dw.addmm_(g.t(), x)
            db += g.sum(dim=0)
        if not grads:
            return {"loss": loss, "lse": lse}
        out = {"loss": loss, "dx": dx, "dw": dw}
        if state["b"] is not None:
            out["db"] = db
        return out
    norm = math.sqrt(sum(float(t.double().pow(2).sum()) for t in state["grads"]))
    scale = state["max_norm"] / norm if norm > state["max_norm"] else 1.0
    outs = [t.double() * scale for t in state["grads"]]
    return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": outs if case["layout"] else torch.cat(outs)}
