"""The operators of a training step on given answers, as one program calls them: scoring, its gradient, the update.

  log_probs       log probabilities of given tokens, entropy, top alternatives  (mtc_token_log_probs)
  log_probs_grad  the logits' gradient of both                                  (mtc_token_log_probs_grad)
  orthogonalize   updates of weight matrices by Newton-Schulz products          (mtc_orthogonalize)

A case names its operator in "op".  `run` takes the plain form (elementary torch
operations, float32) or, where `own` is true, the calls of minitensor_cpp_b200.abi.
"""
import math

import torch

own = False

DEVICE = "cuda"
IGNORE = -100  # token of a position that is not scored (a prompt's tokens, padding)
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # of X, (X X^T) X and (X X^T)^2 X
STEPS = 5
EPS = 1e-7


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # one generated token's row with its alternatives: a decoding step, launch latency only
        {"name": "log probs one token", "op": "log_probs", "rows": 1, "vocab": 32000, "top": 20, "scale": 1.0,
         "ignored": 0.0, "masked": 0.0},
        # the wide MLP's answers (1000 classes) at its global batch, with the five best
        {"name": "log probs wide MLP", "op": "log_probs", "rows": 65536, "vocab": 1000, "top": 5, "scale": 1.0,
         "ignored": 0.0, "masked": 0.0},
        # evaluation of a batch with alternatives, prompts not scored
        {"name": "log probs evaluation", "op": "log_probs", "rows": 4096, "vocab": 32000, "top": 20, "scale": 1.0,
         "ignored": 0.25, "masked": 0.0},
        # odd sizes, a temperature, classes that a mask excludes
        {"name": "log probs odd", "op": "log_probs", "rows": 1031, "vocab": 50003, "top": 7, "scale": 1.0 / 0.7,
         "ignored": 0.1, "masked": 0.5},
        # scoring of sampled answers before a training step, no alternatives
        {"name": "log probs large", "op": "log_probs", "rows": 16384, "vocab": 32000, "top": 0, "scale": 1.0,
         "ignored": 0.0, "masked": 0.0},
        # the spiral MLP's output (3 classes, 300 points): the smallest training step of this repository
        {"name": "log probs grad spiral", "op": "log_probs_grad", "rows": 300, "vocab": 3, "scale": 1.0,
         "ignored": 0.0, "masked": 0.0},
        # odd sizes, a temperature, classes that a mask excludes
        {"name": "log probs grad odd", "op": "log_probs_grad", "rows": 1031, "vocab": 50003, "scale": 1.0 / 0.7,
         "ignored": 0.1, "masked": 0.5},
        # a training step over a large vocabulary, a quarter of the positions not scored
        {"name": "log probs grad large", "op": "log_probs_grad", "rows": 8192, "vocab": 131072, "scale": 1.0,
         "ignored": 0.25, "masked": 0.0},
        # the spiral MLP's weights (2 -> 64 -> 64 -> 3)
        {"name": "orthogonalize spiral", "op": "orthogonalize", "shapes": "64x2,64x64,3x64"},
        # a batch of odd matrices and a single tall one: nothing is a multiple of a tile or of 16 bytes
        {"name": "orthogonalize odd", "op": "orthogonalize", "shapes": "3x771x1031,1500x333"},
        # weights of a few layers of width 1024
        {"name": "orthogonalize layers", "op": "orthogonalize", "shapes": "4x1024x1024,4096x1024,1024x4096"},
        # the wide MLP's weights (1024 -> 8192 x 3 -> 1000)
        {"name": "orthogonalize wide MLP", "op": "orthogonalize",
         "shapes": "8192x1024,8192x8192,8192x8192,1000x8192"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["log_probs", "log_probs_grad", "orthogonalize"])
    if op == "orthogonalize":
        shapes, spent = [], 0.0
        for _ in range(_log_int(rng, 1, 12)):
            shape = (_log_int(rng, 1, 64) if rng.random() < 0.3 else 1, _log_int(rng, 1, 8192), _log_int(rng, 1, 8192))
            cost = _flops(shape)
            if shapes and spent + cost > 5e12 or cost > 1.2e13:
                continue
            spent += cost
            shapes.append("x".join(str(s) for s in (shape if shape[0] > 1 else shape[1:])))
        return {"op": op, "shapes": ",".join(shapes) if shapes else "100x77"}
    vocab = _log_int(rng, 3, 131072)
    case = {"op": op, "rows": _log_int(rng, 1, 65536), "vocab": vocab, "scale": rng.choice([1.0, 1.0 / 0.7, 0.5]),
            "ignored": rng.choice([0.0, 0.1, 0.25, 0.9]), "masked": rng.choice([0.0, 0.0, 0.5, 0.99])}
    most = 16384 * 32000 if op == "log_probs" else 8192 * 131072
    while case["rows"] * vocab > most:
        case["rows"] = (case["rows"] + 1) // 2
    if op == "log_probs":
        case["top"] = min(vocab, rng.choice([0, 1, 2, 5, 8, 20, 32]))
    return case


def _shapes(case):
    """[(count, rows, columns, whether the tensor has a leading axis)]"""
    out = []
    for text in case["shapes"].split(","):
        s = [int(v) for v in text.split("x")]
        out.append((s[0], s[1], s[2], True) if len(s) == 3 else (1, s[0], s[1], False))
    return out


# ----------------------------------------------------------------- inputs --

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _matrix(count, rows, cols, g):
    """A gradient's momentum: a few strong directions over noise."""
    rank = min(8, rows, cols)
    strong = torch.randn(count, rows, rank, device=DEVICE, generator=g)
    t = torch.bmm(strong, torch.randn(count, rank, cols, device=DEVICE, generator=g))
    t += torch.randn(count, rows, cols, device=DEVICE, generator=g)
    return t.mul_(1e-3)


def prepare(case, seed):
    g = _generator(seed)
    state = {"op": case["op"], "case": case}
    if case["op"] == "orthogonalize":
        state["updates"] = [t if lead else t[0] for count, rows, cols, lead in _shapes(case)
                            for t in [_matrix(count, rows, cols, g)]]
        return state
    n, v = case["rows"], case["vocab"]
    # logits of a half-trained model: spread 2, common classes likelier, the given token's raised by 6
    logits = torch.randn(n, v, device=DEVICE, generator=g).mul_(2.0)
    rate = torch.log(torch.arange(v, device=DEVICE, dtype=torch.float32) + 2.7)
    logits -= 0.5 * rate[torch.randperm(v, device=DEVICE, generator=g)]
    tokens = torch.randint(0, v, (n,), device=DEVICE, generator=g)
    row = torch.arange(n, device=DEVICE)
    logits[row, tokens] += 6.0
    if case["masked"] > 0:
        for rows in row.split(1024):
            out = torch.rand(rows.numel(), v, device=DEVICE, generator=g) < case["masked"]
            out[:, :32] = False  # control tokens stay
            out[torch.arange(rows.numel(), device=DEVICE), tokens[rows]] = False
            logits[rows[0]:rows[-1] + 1].masked_fill_(out, -math.inf)
    if case["ignored"] > 0:
        keep = torch.rand(n, device=DEVICE, generator=g) >= case["ignored"]
        keep[n // 2] = True
        tokens = torch.where(keep, tokens, IGNORE)
    state["logits"], state["tokens"] = logits, tokens
    if case["op"] == "log_probs_grad":
        count = (tokens != IGNORE).sum().clamp(min=1).float()
        state["dlog_probs"] = -torch.randn(n, device=DEVICE, generator=g) / count  # advantages of a mean
        state["dentropy"] = (-0.01 / count).reshape(1).expand(n)                   # a bonus on the mean entropy
    return state


# -------------------------------------------------------------- the calls --

def _plain_log_probs(state):
    case, logits, tokens = state["case"], state["logits"], state["tokens"]
    keep = tokens != IGNORE
    at = torch.where(keep, tokens, 0)
    z = logits * case["scale"]
    top = z.amax(dim=1, keepdim=True)
    d = z - top
    e = torch.exp(d)
    s = e.sum(dim=1, keepdim=True)
    lse = top + torch.log(s)
    zt = z[torch.arange(at.numel(), device=z.device), at].unsqueeze(1)
    entropy = torch.log(s) - (torch.where(e > 0, d, 0.0) * e).sum(dim=1, keepdim=True) / s
    out = {"log_probs": torch.where(keep, (zt - lse).squeeze(1), 0.0), "lse": torch.where(keep, lse.squeeze(1), 0.0),
           "entropy": torch.where(keep, entropy.squeeze(1), 0.0)}
    if case["top"] > 0:
        # whole numbers that order as the logits do and, where these are equal, against the index
        bits = (logits + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 32
        key += torch.arange(z.shape[1] - 1, -1, -1, device=z.device)
        best = key.topk(case["top"], dim=1).indices
        out["top_log_probs"] = torch.where(keep.unsqueeze(1), z.gather(1, best) - lse, 0.0)
        out["top_tokens"] = torch.where(keep.unsqueeze(1), best, -1)
    return out


def _plain_log_probs_grad(state):
    case, logits, tokens = state["case"], state["logits"], state["tokens"]
    keep = tokens != IGNORE
    at = torch.where(keep, tokens, 0)
    z = logits * case["scale"]
    d = z - z.amax(dim=1, keepdim=True)
    e = torch.exp(d)
    p = e / e.sum(dim=1, keepdim=True)
    d = torch.where(e > 0, d, 0.0)
    mean = (p * d).sum(dim=1, keepdim=True)
    dlp = (state["dlog_probs"] * keep * case["scale"]).unsqueeze(1)
    dent = (state["dentropy"] * keep * case["scale"]).unsqueeze(1)
    g = -p * (dlp + dent * (d - mean))
    g[torch.arange(at.numel(), device=z.device), at] += dlp.squeeze(1)
    return {"dlogits": g}


def _plain_orthogonalize(state):
    a, b, c = COEFFICIENTS
    outs = []
    for t in state["updates"]:
        tall = t.shape[-2] > t.shape[-1]
        x = t.transpose(-1, -2) if tall else t
        x = x / ((x * x).sum(dim=(-1, -2), keepdim=True).sqrt() + EPS)
        for _ in range(STEPS):
            s = x @ x.transpose(-1, -2)
            x = a * x + (b * s + c * (s @ s)) @ x
        outs.append(x.transpose(-1, -2) if tall else x)
    return {"updates": outs}


def _own(state):
    from minitensor_cpp_b200 import abi

    view = abi.View.of
    if state["op"] == "orthogonalize":
        outs = [torch.empty_like(t) for t in state["updates"]]
        abi.orthogonalize([view(t) for t in state["updates"]], outs=[view(t) for t in outs],
                          coefficients=[COEFFICIENTS] * STEPS, eps=EPS)
        return {"updates": outs}
    case, logits, tokens = state["case"], state["logits"], state["tokens"]
    if state["op"] == "log_probs_grad":
        dlogits = torch.empty_like(logits)
        abi.token_log_probs_grad(view(logits), view(dlogits), tokens=view(tokens), dlog_probs=view(state["dlog_probs"]),
                                 dentropy=view(state["dentropy"]), scale=case["scale"], ignore_token=IGNORE)
        return {"dlogits": dlogits}
    n, k = tokens.numel(), case["top"]
    out = {name: torch.empty(n, device=logits.device) for name in ("log_probs", "lse", "entropy")}
    if k > 0:
        out["top_log_probs"] = torch.empty(n, k, device=logits.device)
        out["top_tokens"] = torch.empty(n, k, dtype=torch.int64, device=logits.device)
    abi.token_log_probs(view(logits), tokens=view(tokens), scale=case["scale"], ignore_token=IGNORE,
                        **{name: view(t) for name, t in out.items()})
    return out


def run(state):
    if own:
        return _own(state)
    if state["op"] == "log_probs":
        return _plain_log_probs(state)
    if state["op"] == "log_probs_grad":
        return _plain_log_probs_grad(state)
    return _plain_orthogonalize(state)


# ------------------------------------------------------ what it cannot do without --

def _flops(shape):
    """Of one tensor (count, rows, columns): both products of a step that are symmetric count half."""
    count, m, n = shape[0], min(shape[1:3]), max(shape[1:3])
    return float(STEPS) * count * (m * (m + 1.0) * n + m * m * (m + 1.0) + 2.0 * m * m * n)


def work(case):
    if case["op"] == "orthogonalize":
        shapes = _shapes(case)
        return {"bytes": sum(8.0 * s[0] * s[1] * s[2] for s in shapes), "flops": sum(_flops(s) for s in shapes)}
    n, v = case["rows"], case["vocab"]
    live = max(1.0, n * (1.0 - case["ignored"]))  # a position that is not scored need not be read
    read = 4.0 * live * v + 8.0 * n
    if case["op"] == "log_probs":
        return {"bytes": read + n * (12.0 + 12.0 * case["top"]), "flops": 6.0 * live * v}
    return {"bytes": read + 4.0 * n * v + 4.0 * n, "flops": 9.0 * live * v}


# ------------------------------------------------- the definitions, in 64 bits --

def _exact_rows(case, state):
    n, v = case["rows"], case["vocab"]
    grad = case["op"] == "log_probs_grad"
    k = 0 if grad else case["top"]
    new = lambda *s: torch.zeros(*s, dtype=torch.float64, device=DEVICE)
    log_probs, lse, entropy, top = new(n), new(n), new(n), new(n, k)
    best = torch.full((n, k), -1, dtype=torch.int64, device=DEVICE)
    dlogits = new(n, v) if grad else None
    live = (state["tokens"] != IGNORE).nonzero().squeeze(1)
    for rows in live.split(max(1, 2 ** 26 // v)):
        raw = state["logits"][rows]
        t = state["tokens"][rows].unsqueeze(1)
        logp = raw.double().mul_(case["scale"])
        total = torch.logsumexp(logp, dim=1, keepdim=True)
        logp -= total
        p = logp.exp()
        h = -torch.special.xlogy(p, p).sum(dim=1, keepdim=True)
        if grad:
            g = torch.zeros_like(p).scatter_(1, t, 1.0).sub_(p).mul_(state["dlog_probs"][rows].double().unsqueeze(1))
            slope = (torch.special.xlogy(p, p) + p * h).mul_(state["dentropy"][rows].double().unsqueeze(1))
            dlogits[rows] = g.sub_(slope).mul_(case["scale"])
            continue
        log_probs[rows] = logp.gather(1, t).squeeze(1)
        lse[rows], entropy[rows] = total.squeeze(1), h.squeeze(1)
        if k > 0:
            order = raw.sort(dim=1, descending=True, stable=True).indices[:, :k]
            best[rows] = order
            top[rows] = logp.gather(1, order)
    if grad:
        return {"dlogits": dlogits}
    out = {"log_probs": log_probs, "lse": lse, "entropy": entropy}
    if k > 0:
        out["top_log_probs"], out["top_tokens"] = top, best
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] != "orthogonalize":
        return _exact_rows(case, state)
    a, b, c = COEFFICIENTS
    outs = []
    for t in state["updates"]:
        x = t.double()
        x = x / (torch.linalg.matrix_norm(x, keepdim=True) + EPS)
        for _ in range(STEPS):  # the polynomial of the shorter side's products, by Horner's rule
            if t.shape[-2] > t.shape[-1]:
                s = x.mT @ x
                x = a * x + (b * x + c * (x @ s)) @ s
            else:
                s = x @ x.mT
                x = a * x + s @ (b * x + c * (s @ x))
        outs.append(x)
    return {"updates": outs}
