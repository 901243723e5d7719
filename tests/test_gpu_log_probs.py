"""Log probabilities of given tokens, their entropy, alternatives and gradient on the GPU
against their definitions in float64.

Tolerances are worst-case rounding bounds, U = 2^-24 being half a step of float32.  With
d = scale (x - max), p = exp(d) / S and E = sum p |d|:
 - d is off by 3 U |d| (the difference, the product, the factor in base 2);
 - an exponential by another 2^-22 = 4 U of itself (the hardware's 2^x), so a sum of them
   by 3 U |d| + 4 U each, and by its additions: a thread adds V / 256 of them at most, rescales
   them once for each 32 and twice when threads join (5 U each, beside the 3 U |d| that
   count the parts of d), and 10 steps join the threads: S - 1, whose largest terms are
   exactly 1, by eps (S - 1) with eps = (V / 200 + 64) U, and by 3 U sum |d| exp(d) = 3 U S E;
 - log S = log1p(S - 1) by that over S, eps (S - 1) / S + 3 U E, and 4 U of itself;
 - E by the same of each |d| p: sum p |d| (3 U |d| + 8 U) + 2 (eps + 3 U E) E;
 - p by 3 U |d| + 4 U (the exponential) + eps (S - 1) / S + 3 U E + 2 U of itself, and where
   the token is the largest logit 1 - p = (S - 1) / S by eps + 4 U of itself and 3 U E.
"""
import ctypes
import math

import pytest
from test_gpu_lm_operators import U, view, within

from minitensor_cpp_b200 import abi

pytestmark = pytest.mark.gpu

IGNORE = -100
INF = math.inf
LOWEST = -3.4028234663852886e38


def f32(x):
    return ctypes.c_float(x).value


def reference(x, t, scale, k=0):
    """{name: (value, bound)} in float64 of rows [N, V] with finite maxima, and what the gradient needs."""
    import torch

    n, vocab = x.shape
    live = torch.ones(n, dtype=torch.bool, device=x.device) if t is None else t != IGNORE
    z = x.double() * f32(scale)
    top = z.amax(1, keepdim=True)
    empty = top == -INF
    d = torch.where(empty, -INF, z - torch.where(empty, 0.0, top))
    e = d.exp()
    s = e.sum(1, keepdim=True)
    ones = (z == top).sum(1, keepdim=True).double()
    others = torch.where(z == top, 0.0, e).sum(1, keepdim=True) + (ones - 1.0).clamp(min=0.0)
    s = torch.where(empty, 1.0, 1.0 + others)
    p = e / s
    da = torch.where(e > 0, d.abs(), 0.0)
    spread = (p * da).sum(1, keepdim=True)
    log_s = torch.log1p(others)
    eps = (vocab / 200 + 64) * U
    dlog_s = eps * others / s + 3 * U * spread + 4 * U * log_s
    dspread = (p * da * (3 * U * da + 8 * U)).sum(1, keepdim=True) + 2 * (eps + 3 * U * spread) * spread
    lse = torch.where(empty, -INF, top + log_s)
    logp = torch.where(empty, -INF, d - log_s)
    dlogp = 3 * U * d.abs() + dlog_s + U * (d.abs() + log_s)
    out = {"lse": (lse.squeeze(1), (dlog_s + U * (top + log_s).abs()).squeeze(1)),
           "entropy": ((log_s + spread).masked_fill(empty, 0.0).squeeze(1),
                       (dlog_s + dspread + U * (log_s + spread)).squeeze(1))}
    if t is not None:
        at = torch.where(live, t, 0).unsqueeze(1)
        out["log_probs"] = (logp.gather(1, at).squeeze(1), dlogp.gather(1, at).squeeze(1))
    for name, (v, b) in out.items():
        out[name] = (torch.where(live, v, 0.0), b.nan_to_num(nan=0.0, posinf=0.0) * live)
    if k:
        order = (x + 0.0).sort(dim=1, descending=True, stable=True).indices[:, :k]
        out["top_tokens"] = (torch.where(live.unsqueeze(1), order, -1), None)
        out["top_log_probs"] = (torch.where(live.unsqueeze(1), logp.gather(1, order), 0.0),
                                dlogp.gather(1, order).nan_to_num(nan=0.0, posinf=0.0) * live.unsqueeze(1))
    rest = {"live": live, "empty": empty, "p": p, "d": torch.where(e > 0, d, 0.0), "da": da, "spread": spread,
            "dspread": dspread, "eps": eps, "share": others / s, "is_top": z == top}
    return out, rest


def grad_reference(x, t, dlp, dent, scale):
    import torch

    _, r = reference(x, t, scale)
    zero = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    on = (r["live"] & ~r["empty"].squeeze(1)).double() * f32(scale)
    a = (zero if dlp is None else dlp.double() * on).unsqueeze(1)
    b = (zero if dent is None else dent.double() * on).unsqueeze(1)
    p = r["p"].nan_to_num(nan=0.0)
    own = b * (r["d"] + r["spread"])
    g = -p * (a + own)
    rel = 3 * U * r["da"] + 6 * U + r["eps"] * r["share"] + 3 * U * r["spread"]
    tol = p * rel * (a.abs() + own.abs()) + p * b.abs() * (3 * U * r["da"] + r["dspread"] + U * (r["da"] + r["spread"]))
    if t is not None and dlp is not None:
        hot = torch.zeros_like(p).scatter_(1, torch.where(r["live"], t, 0).unsqueeze(1), 1.0)
        left = torch.where(r["is_top"], r["share"], 1.0 - p)
        g = g + hot * (a * (p + torch.where(r["is_top"], r["share"], 1.0 - p)))
        # (p and 1 - p of the token together: what is left of 1)
        g = torch.where(hot > 0, a * left - p * own, g)
        tol = tol + hot * a.abs() * torch.where(r["is_top"], (r["eps"] + 4 * U) * left + 3 * U * r["spread"], U)
    return g, tol + 5 * U * g.abs() + 1e-40


def run(x, t, scale=1.0, k=0, stream=None, **skip):
    import torch

    lead = x.shape[:-1]
    out = {n: torch.full(lead, 99.0, device=x.device) for n in ("log_probs", "lse", "entropy") if n not in skip}
    if t is None:
        del out["log_probs"]
    if k:
        out["top_log_probs"] = torch.full((*lead, k), 99.0, device=x.device)
        out["top_tokens"] = torch.full((*lead, k), 99, dtype=torch.int64, device=x.device)
    abi.token_log_probs(view(x), tokens=None if t is None else view(t), scale=scale, ignore_token=IGNORE, stream=stream,
                        **{n: view(v) for n, v in out.items()})
    return out


def run_grad(x, t, dlp, dent, scale=1.0, to=None, stream=None):
    import torch

    to = torch.full_like(x, 99.0) if to is None else to
    abi.token_log_probs_grad(view(x), view(to), tokens=None if t is None else view(t),
                             dlog_probs=None if dlp is None else view(dlp),
                             dentropy=None if dent is None else view(dent), scale=scale, ignore_token=IGNORE, stream=stream)
    return to


def same_or_within(got, want, tol, what):
    """`within`, infinities and NaN being where they should be."""
    import torch

    want = torch.where(want.abs() > -LOWEST, want.sign() * INF, want)  # (NaN stays)
    special = ~want.isfinite()
    assert torch.equal(got[special].double().nan_to_num(nan=7.0), want[special].nan_to_num(nan=7.0)), what
    within(torch.where(special, 0.0, got), torch.where(special, 0.0, want), tol, what)


def check(x, t, dlp, dent, scale=1.0, k=0):
    """Both entry points; x [.., V]."""
    import torch

    got = run(x, t, scale, k)
    got["dlogits"] = run_grad(x, t, dlp, dent, scale)
    abi.check_device_errors(0)
    vocab = x.shape[-1]
    flat = lambda v: None if v is None else v.reshape(-1)
    want, _ = reference(x.reshape(-1, vocab), flat(t), scale, k)
    want["dlogits"] = grad_reference(x.reshape(-1, vocab), flat(t), flat(dlp), flat(dent), scale)
    for name, v in got.items():
        value, tol = want[name]
        what = f"{name} of {tuple(x.shape)}, k {k}"
        if tol is None:
            assert torch.equal(v.reshape(value.shape), value), what
        else:
            same_or_within(v.reshape(value.shape), value, tol + 1e-42, what)
    return got


def data(n, vocab, seed, ignored=0.0, spread=2.0, masked=0.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, vocab, device="cuda", generator=g) * spread
    t = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    if masked:
        x[torch.rand(n, vocab, device="cuda", generator=g) < masked] = -INF
    if ignored:
        t[torch.rand(n, device="cuda", generator=g) < ignored] = IGNORE
    dlp, dent = (torch.randn(n, device="cuda", generator=g) for _ in range(2))
    return x, t, dlp, dent


# the sizes where the path, the number of a thread's elements or the vectors' ends change
VOCABS = [1, 2, 3, 5, 31, 32, 33, 127, 128, 129, 511, 512, 513, 1000, 1023, 1024, 1025, 1026, 1027, 1028, 2047, 4099, 8191,
          8192, 8193, 8199, 16384, 16385, 32000, 50003, 65536, 131072, 200003]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("n, ignored, scale", [(1, 0.0, 1.0), (7, 0.3, 1.0 / 0.7), (67, 0.1, 0.25)])
def test_against_float64(cuda, vocab, n, ignored, scale):
    for k in sorted({1, min(vocab, 5), min(vocab, 32)}):
        check(*data(n, vocab, vocab + n, ignored), scale, k)


@pytest.mark.parametrize("rows", [300, 5000])
@pytest.mark.parametrize("vocab", [3, 1000, 2000])
def test_many_rows(cuda, rows, vocab):
    check(*data(rows, vocab, rows, 0.25), 1.0, 3)


@pytest.mark.parametrize("vocab", [3, 40, 700, 1024, 1500, 9001, 32000])
@pytest.mark.parametrize("masked", [0.5, 0.97, 1.0])
def test_masks(cuda, vocab, masked):
    """-inf leaves a part of a row, a few of it, or nothing (with fewer left than alternatives are wanted)."""
    x, t, dlp, dent = data(33, vocab, 5, 0.1, masked=masked)
    x[3], x[4] = -INF, -INF
    x[4, vocab // 2] = 1.5
    got = check(x, t, dlp, dent, 0.8, min(vocab, 32))
    t3 = t[3].item()
    if t3 != IGNORE:
        assert got["lse"][3] == -INF and got["log_probs"][3] == -INF and got["entropy"][3] == 0
        assert got["top_tokens"][3].tolist() == list(range(min(vocab, 32))) and (got["dlogits"][3] == 0).all()
    if t[4].item() != IGNORE:
        assert got["lse"][4] == f32(f32(0.8) * 1.5) and got["entropy"][4] == 0 and got["top_tokens"][4, 0] == vocab // 2


@pytest.mark.parametrize("vocab", [7, 512, 1024, 1025, 20000, 140001])
def test_equal_logits_go_to_the_lowest_index(cuda, vocab):
    import torch

    k = min(vocab, 32)
    x = torch.stack([torch.full((vocab,), 2.5, device=cuda), torch.full((vocab,), LOWEST, device=cuda),
                     torch.arange(vocab, device=cuda).float() // 9, -(torch.arange(vocab, device=cuda).float() // 9),
                     torch.where(torch.arange(vocab, device=cuda) % 2 == 0, 0.0, -0.0),  # zeros of both signs are equal
                     torch.arange(vocab, device=cuda).flip(0) % 3 * 1.0])
    t = torch.tensor([0, vocab - 1, 0, vocab // 2, vocab - 1, 1], device=cuda)
    got = check(x, t, torch.ones(6, device=cuda), torch.ones(6, device=cuda), 1.0, k)
    for row in (0, 1, 4):
        assert got["top_tokens"][row].tolist() == list(range(k))


@pytest.mark.parametrize("vocab, threads", [(140001, 512), (8000, 256), (1024, 32), (700, 32)])
@pytest.mark.parametrize("many", [1, 3, 60])
def test_likeliest_that_crowd(cuda, vocab, threads, many):
    """The largest logits lie where few threads read them: more than a list of candidates holds."""
    import torch

    x, t, dlp, dent = data(5, vocab, many)
    of = torch.arange(vocab, device=cuda)
    of = of // 4 % threads if vocab > 1024 else of % threads
    x[:, (of >= 9) & (of < 9 + many)] += 50.0
    x[3] = x[3].round()
    for k in (1, 3, 32):
        check(x, t, dlp, dent, 1.0, k)


@pytest.mark.parametrize("vocab", [3, 100, 1000, 30000])
def test_sorted_rows(cuda, vocab):
    import torch

    x, t, dlp, dent = data(4, vocab, 1)
    x[0], x[1] = x[0].sort().values, x[1].sort(descending=True).values
    x[2] = torch.linspace(-80.0, 80.0, vocab, device=cuda)  # every batch raises the maximum
    x[3] = torch.linspace(3e38, -3e38, vocab, dtype=torch.float64, device=cuda).float()  # (float32 steps overflow)
    check(x, t, dlp, dent, 1.0, min(vocab, 20))


def test_rows_that_are_sure_keep_the_digits_of_what_is_left(cuda):
    """p of the token 1 - 1e-9: log p, the entropy and the gradient are of the size of what is left."""
    import torch

    for vocab in (5, 1000, 3000, 32000):
        x, t, dlp, dent = data(40, vocab, 2, spread=0.5)
        x[torch.arange(40, device=cuda), t] = torch.linspace(18, 60, 40, device=cuda)
        got = check(x, t, dlp, dent, 1.0, 2)
        assert (got["log_probs"] < 0).all() and (got["entropy"] > 0).all()
        assert (got["dlogits"].gather(1, t.unsqueeze(1)) != 0).all()


@pytest.mark.parametrize("vocab", [5, 900, 5000])
def test_nan_and_infinity_stay_in_their_rows(cuda, vocab):
    import torch

    k = 3
    x, t, dlp, dent = data(8, vocab, 3)
    x[1, 2], x[2, vocab - 1], x[2, 0] = float("nan"), float("nan"), INF
    x[3, 1], x[4, 1], x[4, 4] = INF, INF, INF
    x[5, 3], t[6] = float("nan"), IGNORE
    x[6] = float("nan")  # a row that is not scored may hold anything
    sign = torch.tensor([0xFFC00000 - 2 ** 32], dtype=torch.int32, device=cuda).view(torch.float32)
    x[5, 0] = sign[0]  # a NaN with its sign set
    got = run(x, t, 1.0, k)
    got["dlogits"] = run_grad(x, t, dlp, dent)
    abi.check_device_errors(0)
    for name in ("log_probs", "lse", "entropy", "top_log_probs", "dlogits"):
        v = got[name].reshape(8, -1)
        assert v[1:6].isnan().all(), name
        assert v[[0, 7]].isfinite().all() and (v[6] == 0).all(), name
    assert got["top_tokens"][:, 0].tolist()[1:7] == [2, vocab - 1, 1, 1, 0, -1]
    assert got["top_tokens"][2, 1] == 0 and got["top_tokens"][4, 1] == 4 and got["top_tokens"][5, 1] == 3
    fine = torch.tensor([0, 7], device=cuda)
    want, _ = reference(x[fine], t[fine], 1.0, k)
    assert torch.equal(got["top_tokens"][fine], want["top_tokens"][0])


@pytest.mark.parametrize("vocab", [6, 600, 3000])
def test_lowest_and_largest_values(cuda, vocab):
    """Masks of the type's lowest value, and differences that overflow."""
    import torch

    x, t, dlp, dent = data(6, vocab, 4)
    x[0, 1:], x[1], x[2, ::2] = LOWEST, LOWEST, LOWEST
    x[3], x[3, 0] = LOWEST, -LOWEST
    x[4] = torch.where(torch.arange(vocab, device=cuda) % 2 == 0, LOWEST, -INF)
    t[0], t[3] = 0, 1
    check(x, t, dlp, dent, 1.0, min(vocab, 9))


def test_views(cuda):
    """Leading axes of any number, gaps, transposed and broadcast operands, offsets without alignment."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(9)
    rnd = lambda *s: torch.randn(*s, device=cuda, generator=g)
    for vocab in (37, 1000, 2001):
        tok = lambda *s: torch.randint(0, vocab, s, device=cuda, generator=g)
        check(rnd(vocab), tok(), rnd(()), rnd(()), 1.0, 3)                                    # no leading axis
        check(rnd(2, 3, 5, vocab), tok(2, 3, 5), rnd(2, 3, 5), rnd(2, 3, 5), 1.0, 3)
        check(rnd(1, 1, 2, 1, 2, 1, 2, vocab), tok(1, 1, 2, 1, 2, 1, 2), rnd(1, 1, 2, 1, 2, 1, 2),
              rnd(1, 1, 2, 1, 2, 1, 2), 1.0, 1)
        check(rnd(vocab, 11).t(), tok(11), rnd(11), rnd(11), 1.0, 5)                           # classes apart
        check(rnd(4, 6, 2 * vocab)[1:, ::2, ::2], tok(3, 3), rnd(3, 3), rnd(1, 1).expand(3, 3), 1.0, 5)
        check(rnd(6, 4, vocab).transpose(0, 1), tok(6, 4).t(), rnd(4, 6), rnd(6, 4).t(), 1.0, 5)
        check(rnd(1, vocab).expand(5, vocab), tok(5), rnd(5), rnd(5), 1.0, 2)                  # one row for all
        check(rnd(9, vocab), tok(1).expand(9), rnd(1).expand(9), rnd(9), 1.0, 2)
        for offset in (1, 2, 3):
            check(rnd(5 * (vocab + 1) + offset)[offset:].view(5, vocab + 1)[:, :vocab], tok(5), rnd(5), rnd(5), 1.0, 4)


@pytest.mark.parametrize("vocab", [50, 1000, 1777, 9000])
def test_written_views(cuda, vocab):
    """Outputs with gaps and offsets: what lies between and behind them stays as it was."""
    import torch

    x, t, dlp, dent = data(12, vocab, 6, 0.2)
    want = run(x, t, 1.0, 4)
    want["dlogits"] = run_grad(x, t, dlp, dent)
    held = {"log_probs": torch.full((30,), 7.0, device=cuda), "lse": torch.full((30,), 7.0, device=cuda),
            "entropy": torch.full((30,), 7.0, device=cuda), "top_log_probs": torch.full((15, 13), 7.0, device=cuda),
            "top_tokens": torch.full((9, 15), 7, device=cuda), "dlogits": torch.full((14, 2 * vocab + 3), 7.0, device=cuda)}
    part = {"log_probs": held["log_probs"][3:27:2], "lse": held["lse"][1:13], "entropy": held["entropy"][2::2][:12],
            "top_log_probs": held["top_log_probs"][1:13, 2:10:2], "top_tokens": held["top_tokens"][2:6, 1:13].t(),
            "dlogits": held["dlogits"][1:13, 1:2 * vocab:2]}
    abi.token_log_probs(view(x), tokens=view(t), ignore_token=IGNORE,
                        **{n: view(v) for n, v in part.items() if n != "dlogits"})
    run_grad(x, t, dlp, dent, to=part["dlogits"])
    for offset in (0, 1, 2, 3):
        to = torch.full((12 * vocab + 5,), 7.0, device=cuda)
        run_grad(x, t, dlp, dent, to=to[offset:offset + 12 * vocab].view(12, vocab))
        assert torch.equal(to[offset:offset + 12 * vocab].view(12, vocab), want["dlogits"])
        assert (to[:offset] == 7).all() and (to[offset + 12 * vocab:] == 7).all()
    torch.cuda.synchronize()
    for n, v in part.items():
        assert torch.equal(v, want[n]), n
        v.fill_(7)
        assert (held[n] == 7).all(), n


def test_each_output_alone(cuda):
    import torch

    for vocab in (9, 800, 6001):
        x, t, dlp, dent = data(20, vocab, 8, 0.3)
        want = run(x, t, 1.3, 6)
        for name, v in want.items():
            got = torch.full_like(v, 99)
            tokens = view(t)
            abi.token_log_probs(view(x), tokens=tokens, scale=1.3, ignore_token=IGNORE, **{name: view(got)})
            assert torch.equal(got, v), name
        free = run(x, None, 1.3, 6)  # without tokens every row counts
        scored = t != IGNORE
        for name, v in free.items():
            assert torch.equal(v[scored], want[name][scored]), name
            assert name == "top_tokens" or v.isfinite().all()
        within(run_grad(x, t, dlp, None, 1.3), *grad_reference(x, t, dlp, None, 1.3), "of log_probs alone")
        within(run_grad(x, t, None, dent, 1.3), *grad_reference(x, t, None, dent, 1.3), "of the entropy alone")
        within(run_grad(x, None, None, dent, 1.3), *grad_reference(x, None, None, dent, 1.3), "without tokens")


@pytest.mark.parametrize("vocab", [3, 1000, 1025, 32000, 131072])
def test_gradient_in_place(cuda, vocab):
    import torch

    x, t, dlp, dent = data(21, vocab, 10, 0.2)
    want = run_grad(x, t, dlp, dent)
    run_grad(x, t, dlp, dent, to=x)
    assert torch.equal(x, want)


@pytest.mark.parametrize("vocab", [5, 700, 4000])
def test_gradient_against_differences(cuda, vocab):
    """Along random directions v, (f(x + h v) - f(x - h v)) / 2h = g . v + O(h^2), f in float64.
    With |f'''| <= 20 sum |weights| |v|^3 (derivatives of softmax and of p log p are sums of at
    most 6 products of p, [v = t] and log p + H with p |log p + H| < 1 ...) and h = 1e-4, h^2
    leaves 1e-7 of the weights; the gradient itself has float32's digits."""
    import torch

    x, t, dlp, dent = data(6, vocab, 11, spread=1.0)
    g = run_grad(x, t, dlp, dent, 1.2).double()

    def f(z):
        logp = torch.log_softmax(z * f32(1.2), 1)
        h = -(logp.exp() * logp).sum(1)
        return logp.gather(1, t.unsqueeze(1)).squeeze(1) * dlp.double() + h * dent.double()

    for seed in range(3):
        v = torch.randn(6, vocab, device=cuda, generator=torch.Generator(device="cuda").manual_seed(seed)).double()
        v /= v.abs().amax(1, keepdim=True)
        h = 1e-4
        want = (f(x.double() + h * v) - f(x.double() - h * v)) / (2 * h)
        tol = (dlp.abs() + dent.abs()).double() * (1e-6 + 2 ** -18 * v.abs().amax(1))
        within((g * v).sum(1), want, tol, "directional derivative")


def test_tokens_outside_the_classes_are_reported(cuda):
    import torch

    for vocab in (10, 3000):
        for bad in (vocab, -1, 2 ** 40):
            x, t, dlp, dent = data(4, vocab, 12)
            t[2] = bad
            got = run(x, t, 1.0, 3)
            with pytest.raises(IndexError, match=str(bad)):
                abi.check_device_errors(0)
            g = run_grad(x, t, dlp, dent)
            with pytest.raises(IndexError, match=str(bad)):
                abi.check_device_errors(0)
            assert all((got[n][2] == 0).all() for n in ("log_probs", "lse", "entropy", "top_log_probs"))
            assert (got["top_tokens"][2] == -1).all() and (g[2] == 0).all()
            want, _ = reference(x[:2], t[:2], 1.0, 3)
            assert torch.equal(got["top_tokens"][:2], want["top_tokens"][0])
    abi.check_device_errors(0)


def test_beyond_32_bits(cuda):
    """2.2e9 logits: rows behind 2^31 elements are read and written where they are."""
    import torch

    n, vocab = 16500, 131072
    x = torch.zeros(n, vocab, device=cuda)
    t = torch.full((n,), IGNORE, device=cuda)
    some = torch.tensor([0, 1, 8191, 16383, 16384, 16385, n - 1], device=cuda)
    small, token, dlp, dent = data(7, vocab, 13)
    x[some], t[some] = small, token
    want, wantg = run(small, token, 1.0, 5), run_grad(small, token, dlp, dent)
    got = run(x, t, 1.0, 5)
    for name, v in want.items():
        assert torch.equal(got[name][some], v), name
    a, b = torch.zeros(n, device=cuda), torch.zeros(n, device=cuda)
    a[some], b[some] = dlp, dent
    run_grad(x, t, a, b, to=x)
    assert torch.equal(x[some], wantg)
    x[some] = 0.0
    assert x.count_nonzero() == 0


@pytest.mark.parametrize("vocab", [3, 1000, 20011])
def test_recorded_and_replayed_next_to_eager_calls(cuda, vocab):
    """Two graphs and eager calls on other streams at once; new inputs in the same places."""
    import torch

    st = ctypes.c_void_p()
    abi.check(abi.lib().mtc_stream_create(0, ctypes.byref(st)))
    x, t, dlp, dent = data(50, vocab, 14, 0.2)
    buffers = [run(x, t, 1.0, 3), run(x, t, 1.0, 3)]
    grads = [torch.empty_like(x), torch.empty_like(x)]
    graphs = []
    torch.cuda.synchronize()
    for out, g in zip(buffers, grads):
        abi.check(abi.lib().mtc_capture_begin(0, st))
        abi.token_log_probs(view(x), tokens=view(t), ignore_token=IGNORE, stream=st.value,
                            **{n: view(v) for n, v in out.items()})
        run_grad(x, t, dlp, dent, to=g, stream=st.value)
        graph = ctypes.c_void_p()
        abi.check(abi.lib().mtc_capture_end(1, ctypes.byref(graph)))
        graphs.append(graph)
    for seed in (15, 16):
        y, u, a, b = data(50, vocab, seed, 0.2)
        x.copy_(y), t.copy_(u), dlp.copy_(a), dent.copy_(b)
        for v in [*buffers[0].values(), *buffers[1].values(), *grads]:
            v.fill_(55)
        torch.cuda.synchronize()
        for graph in graphs:
            abi.check(abi.lib().mtc_graph_launch(graph))
        want, wantg = run(y, u, 1.0, 3), run_grad(y, u, a, b)  # meanwhile
        abi.check(abi.lib().mtc_stream_synchronize(st))
        torch.cuda.synchronize()
        for out, g in zip(buffers, grads):
            assert all(torch.equal(out[n], want[n]) for n in want) and torch.equal(g, wantg)
    for graph in graphs:
        abi.check(abi.lib().mtc_graph_destroy(graph))
    abi.check(abi.lib().mtc_stream_destroy(0, st))


def test_in_a_graph_of_torch(cuda):
    """No workspace is needed, so a stream that torch captures is fine."""
    import torch

    x, t, dlp, dent = data(40, 5000, 17, 0.2)
    want, wantg = run(x, t, 1.0, 3), run_grad(x, t, dlp, dent)
    out, g = {n: torch.zeros_like(v) for n, v in want.items()}, torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        abi.token_log_probs(view(x), tokens=view(t), ignore_token=IGNORE, **{n: view(v) for n, v in out.items()})
        run_grad(x, t, dlp, dent, to=g)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out[n], want[n]) for n in want) and torch.equal(g, wantg)


def test_the_same_inputs_give_the_same_bits(cuda):
    import torch

    for vocab in (1000, 50003):
        x, t, dlp, dent = data(200, vocab, 18, 0.2)
        first, grad = run(x, t, 1.0, 20), run_grad(x, t, dlp, dent)
        for _ in range(5):
            again = run(x, t, 1.0, 20)
            assert all(torch.equal(again[n], first[n]) for n in first)
            assert torch.equal(run_grad(x, t, dlp, dent), grad)


SIGNS = [(1.0, 1.0), (1.0, -1.0), (-1.0, 0.01), (1.0, 0.01), (-0.01, -1.0), (1.0, 100.0)]


@pytest.mark.parametrize("vocab", [5, 1000, 2000, 3001, 32000])
@pytest.mark.parametrize("dlp, dent", SIGNS)
@pytest.mark.parametrize("scale", [1.0, 0.7])
def test_gradient_of_a_sure_token_keeps_the_digits_of_what_is_left(cuda, vocab, dlp, dent, scale):
    """1 - p of the token from 1e-3 to 1e-12, left to all others or to one of them.

    The token being the largest logit, its element is a (1 - p) - p b E with a = scale dlp and b =
    scale dent.  1 - p is off by (eps + 4 U) of itself and 3 U E (above), a by U; b by U, its
    product with E by U, E by `dspread`, p as above with d = 0, the products by U each, the
    difference by U of itself."""
    import torch

    n = 40
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(n, vocab, device=cuda, generator=g) * 0.5
    t = torch.randint(0, vocab, (n,), device=cuda, generator=g)
    row = torch.arange(n, device=cuda)
    left = torch.logspace(-3, -12, n // 2, device=cuda).repeat(2)
    other = (t + 1 + torch.randint(0, vocab - 1, (n,), device=cuda, generator=g)) % vocab
    x[n // 2:], x[row, other] = -INF, torch.randn(n, device=cuda, generator=g)
    x[row, t] = -INF
    x[row, t] = torch.logsumexp(x * scale, 1) / scale - left.log() / scale
    a, b = torch.full((n,), dlp, device=cuda), torch.full((n,), dent, device=cuda)
    got = run_grad(x, t, a, b, scale)[row, t]
    _, r = reference(x, t, scale)
    at = lambda v: v.expand(n, vocab).gather(1, t.unsqueeze(1)).squeeze(1)
    assert at(r["is_top"]).all()
    a, b = abs(f32(dlp) * f32(scale)), abs(f32(dent) * f32(scale))
    share, p, spread, dspread = at(r["share"]), at(r["p"]), at(r["spread"]), at(r["dspread"])
    want = f32(dlp) * f32(scale) * share - p * (f32(dent) * f32(scale)) * spread
    tol = a * ((r["eps"] + 6 * U) * share + 3 * U * spread)
    tol += p * b * (dspread + spread * (9 * U + r["eps"] * share + 3 * U * spread)) + U * want.abs() + 1e-42
    within(got, want, tol, f"{vocab} classes, {dlp}, {dent}")


@pytest.mark.parametrize("vocab", [3, 33, 100, 500, 1000, 1500, 2000, 2001])
@pytest.mark.parametrize("equal", [True, False])
def test_rows_whose_others_are_some_of_the_largest(cuda, vocab, equal):
    """S - 1 from 0.02 to 2: the largest logit's 1 must not take the others' digits, within the bounds above."""
    import torch

    n = 400
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.zeros(n, vocab, device=cuda) if equal else torch.randn(n, vocab, device=cuda, generator=g)
    t = torch.randint(0, vocab, (n,), device=cuda, generator=g)
    row = torch.arange(n, device=cuda)
    x[row, t] = -INF
    x -= (torch.logsumexp(x, 1) - torch.logspace(math.log10(0.02), math.log10(2.0), n, device=cuda).log()).unsqueeze(1)
    x[row, t] = 0.0
    dlp, dent = (torch.randn(n, device=cuda, generator=g) for _ in range(2))
    check(x, t, dlp, dent, 1.0, 2)
    t = (t + 1) % vocab
    check(x, t, dlp, dent, 1.0 / 0.7, 1)


@pytest.mark.parametrize("vocab", [32, 100, 128, 200, 512, 1000, 1004, 2000, 2048, 3000, 9000])
@pytest.mark.parametrize("gap", [0, 1, 2, 3])
def test_a_row_gives_the_same_bits_alone_and_among_others(cuda, vocab, gap):
    """Also where rows of one call lie on 16 bytes and others do not."""
    import torch

    n = 9
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(n * (vocab + gap) + 8, device=cuda, generator=g).mul_(2.0)[4:4 + n * (vocab + gap)]
    x = x.view(n, vocab + gap)[:, :vocab]
    t = torch.randint(0, vocab, (n,), device=cuda, generator=g)
    dlp, dent = (torch.randn(n, device=cuda, generator=g) for _ in range(2))
    check(x, t, dlp, dent, 1.0, 3)
    want, grad = run(x, t, 1.0, 3), run_grad(x, t, dlp, dent)
    for i in range(n):
        one = slice(i, i + 1)
        got = run(x[one], t[one], 1.0, 3)
        assert all(torch.equal(got[name], want[name][one]) for name in want), i
        assert torch.equal(run_grad(x[one], t[one], dlp[one], dent[one]), grad[one]), i
        held = torch.full_like(x[one], 7.0)
        assert torch.equal(run_grad(x[one], t[one], dlp[one], dent[one], to=held), grad[one]), i


@pytest.mark.parametrize("vocab", [6, 600, 3000])
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -60, 1e-3, 0.25, 0.7])
def test_log_probabilities_of_differences_beyond_float32(cuda, vocab, scale):
    """x - max overflows where scale (x - max) does not."""
    import torch

    x, t, dlp, dent = data(5, vocab, 20)
    x[0], x[0, 0] = 3e38, -3e38
    x[1], x[1, 1] = LOWEST, -LOWEST
    x[2, 2], x[2, 3] = 2e38, LOWEST
    x[3, 0], x[3, 1], x[3, 2] = 1e38, -2.5e38, -INF
    t[:4] = torch.tensor([0, 0, 3, 1], device=cuda)
    got = check(x, t, dlp, dent, scale, min(vocab, 32))
    if scale < 0.5:
        assert got["log_probs"][:4].isfinite().all()


# both sides of the classes at which a row goes to other threads (forward: 32, 128, 512, 1024, 2048 to
# more elements of a lane, 4000, 12000, 24000, 100000 to more threads of a CTA; the gradient's CTAs:
# 1024, 3500, 6000, 12000, 24000, 56000), and CTAs of 32 threads with 0 to 3 elements ahead and behind
BORDERS = [2047, 2048, 2049, 2050, 2051, 2301, 2999, 3002, 3499, 3500, 3501, 3999, 4000, 4001, 5999, 6000, 6001, 11999, 12000,
           12001, 23999, 24000, 24001, 55999, 56000, 56001, 99999, 100000, 100001]


@pytest.mark.parametrize("vocab", BORDERS)
def test_borders_of_the_number_of_threads(cuda, vocab):
    import torch

    for n, ignored, scale, k in ((5, 0.0, 1.0, 1), (6, 0.3, 1.0 / 0.7, 32), (41, 0.1, 0.25, 5)):
        check(*data(n, vocab, vocab + n, ignored), scale, k)
    x, t, dlp, dent = data(9, vocab, vocab, masked=0.9)
    x[1], x[2, 3], x[4], x[5, vocab - 1] = -INF, float("nan"), 2.5, INF
    got = run(x, t, 1.0, 20)
    got["dlogits"] = run_grad(x, t, dlp, dent)
    for name in ("lse", "entropy", "dlogits"):
        assert got[name][[2, 5]].isnan().all(), name
    assert got["top_tokens"][[2, 5], 0].tolist() == [3, vocab - 1]
    fine = torch.tensor([0, 1, 3, 4, 6, 7, 8], device=cuda)
    check(x[fine], t[fine], dlp[fine], dent[fine], 1.0, 20)


@pytest.mark.parametrize("vocab, threads, near", [(2051, 32, 9), (3001, 32, 7), (3999, 32, 5), (8001, 64, 5), (20000, 128, 4),
                                                 (50003, 256, 3), (99999, 256, 2), (140001, 512, 2)])
@pytest.mark.parametrize("equal", [True, False])
def test_likeliest_that_crowd_in_a_few_threads(cuda, vocab, threads, near, equal):
    """Neighbouring threads read the largest logits, of which there are more than the 512 of a list."""
    import torch

    x, t, dlp, dent = data(4, vocab, near)
    of = torch.arange(vocab, device=cuda)
    for row in range(4):
        ahead = (-row * vocab) % 4  # of a contiguous row's first vector
        owner = (of - ahead).clamp(min=0) // 4 % threads
        those = (owner >= 9) & (owner < 9 + near) & (of >= ahead)
        assert those.sum() > 512
        x[row, those] = x[row, those].round() + 50.0 if equal else x[row, those] + 50.0
    for k in (1, 3, 32):
        check(x, t, dlp, dent, 1.0, k)
