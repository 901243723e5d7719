"""Embedding, linear cross entropy and gradient clipping on the GPU against their
definitions in float64.

Tolerances are worst-case rounding bounds, u = 2^-24 being half a step of float32
relative to the value:
 - a sum of K float32 products, in whatever order and grouping, each product of
   operands held to 2^-22 (a pair of 16-bit floats of 11 bits each) and each
   addition off by at most a step: |err| <= (K + 16) * 2u * sum |a||b|;
 - exp and log of CUDA are within 2 steps (4u);
 - a logsumexp over V terms: its argument's error, plus (V / 256 + 32) * 2u for
   sums of partial sums, plus a rounding of the result;
 - the softmax gradient d * (p - [v = t]) carries p times the error of its
   exponent, plus 8u of its own size for exp, the subtraction and the product.
"""
import ctypes
import math

import numpy as np
import pytest

from minitensor_cpp_b200 import abi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
IGNORE = -100


def view(t):
    return abi.View.of(t)


def product_bound(k, a_abs_b_abs):
    return (k + 16) * 2 * U * a_abs_b_abs


def within(got, want, tol, what):
    import torch

    got = got.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        ratio = ((got - want).abs() / tol).nan_to_num(nan=float("inf")).max().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {ratio:.3g} bounds, first {at}: "
                             f"{got[tuple(at)].item()} for {want[tuple(at)].item()}")
    torch.cuda.synchronize()


# ---------------------------------------------------------------- embedding --

def make_tokens(n, vocab, seed, hot=0.3):
    """Tokens of which one owns a share `hot` and the others are spread."""
    import torch

    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, vocab, (n,), generator=g)
    t[torch.rand(n, generator=g) < hot] = vocab // 2
    return t.cuda()


EMB_SHAPES = [(1, 5, 1), (1, 1, 7), (7, 3, 4), (33, 10, 64), (256, 30, 48), (257, 100, 65), (300, 77, 30), (60, 500, 142), (1000, 999, 128), (4097, 50, 36),
              (5000, 70001, 20), (9000, 2000, 1100), (65536, 1000, 8), (70001, 3000, 16), (200003, 300000, 5), (2048, 70000, 24), (2049, 3000, 24),
              (700, 1 << 24, 1)]


@pytest.mark.parametrize("n, vocab, dim", EMB_SHAPES)
@pytest.mark.parametrize("padding", [None, 2])
def test_embedding_rows(cuda, n, vocab, dim, padding):
    import torch

    torch.manual_seed(n + dim)
    table = torch.randn(vocab, dim, device=cuda)
    tok = make_tokens(n, vocab, n)
    if padding is not None:
        tok[:: 3] = padding
        if vocab <= padding:  # a padding token outside the table is no error
            tok.clamp_(max=padding)
    out = torch.full((n, dim), 7.0, device=cuda)
    abi.embedding(view(table), view(tok), view(out), scale=1.7, padding_token=padding)
    abi.check_device_errors(0)
    want = table[tok.clamp(max=vocab - 1)] * torch.tensor(1.7, device=cuda)  # one rounding: the same bits
    if padding is not None:
        want[tok == padding] = 0.0
    assert torch.equal(out, want)


@pytest.mark.parametrize("n, vocab, dim", EMB_SHAPES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_gradient(cuda, n, vocab, dim, accumulate):
    import torch

    torch.manual_seed(n * dim)
    dout = torch.randn(n, dim, device=cuda)
    tok = make_tokens(n, vocab, n + 1)
    padding = vocab // 3
    base = torch.randn(vocab, dim, device=cuda)
    got = base.clone()
    abi.embedding_grad(view(dout), view(tok), view(got), scale=0.3, padding_token=padding, accumulate=accumulate)
    abi.check_device_errors(0)
    live = tok != padding
    scale = float(np.float32(0.3))
    want = torch.zeros(vocab, dim, dtype=torch.float64, device=cuda)
    want.index_put_((tok[live],), dout[live].double() * scale, accumulate=True)
    size = torch.zeros_like(want).index_put_((tok[live],), dout[live].double().abs() * scale, accumulate=True)
    count = torch.bincount(tok[live], minlength=vocab).double().unsqueeze(1)
    tol = (count + 1) * U * 1.01 * size  # one addition a position, one product
    if accumulate:
        want += base.double()
        tol = tol + U * 1.01 * want.abs() + U * tol
    within(got, want, tol + 1e-45, "embedding gradient")
    if not accumulate:  # rows without a position are exact zeros
        assert torch.equal(got[count.squeeze(1) == 0], torch.zeros_like(got[count.squeeze(1) == 0]))
    again = base.clone()
    abi.embedding_grad(view(dout), view(tok), view(again), scale=0.3, padding_token=padding, accumulate=accumulate)
    assert torch.equal(got, again)  # the order of every sum is fixed


def test_embedding_takes_views_of_any_layout(cuda):
    """A transposed table, ragged row strides, an offset that breaks the 16-byte
    alignment, tokens of rank two read backwards; nothing beside the view is written."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(3)
    vocab, dim = 40, 12
    table_t = torch.randn(dim, vocab, device=cuda, generator=g)
    tok = torch.randint(0, vocab, (5, 9), device=cuda, generator=g)
    out_store = torch.full((5 * 9 * 20 + 3,), -3.0, device=cuda)
    out = out_store[3:].as_strided((5, 9, dim), (9 * 20, 20, 1))
    tv = abi.View(view(tok).storage, (5, 9), (-9, -1), 44)
    abi.embedding(view(table_t.t()), tv, view(out), scale=2.0)
    back = tok.flatten().flip(0).reshape(5, 9)
    assert torch.equal(out, table_t.t()[back] * 2.0)
    mask = torch.ones_like(out_store, dtype=torch.bool)
    mask[3:].as_strided((5, 9, dim), (9 * 20, 20, 1)).fill_(False)
    assert (out_store[mask] == -3.0).all()
    # the gradient through the same views, into a table of padded rows
    store = torch.full((vocab, dim + 5), -3.0, device=cuda)
    abi.embedding_grad(view(out), tv, view(store[:, 2:2 + dim]))
    want = torch.zeros(vocab, dim, dtype=torch.float64, device=cuda)
    want.index_put_((back.reshape(-1),), out.reshape(-1, dim).double(), accumulate=True)
    size = torch.zeros_like(want).index_put_((back.reshape(-1),), out.reshape(-1, dim).double().abs(), accumulate=True)
    within(store[:, 2:2 + dim], want, 46 * U * size + 1e-45, "gradient through views")
    assert (store[:, :2] == -3.0).all() and (store[:, 2 + dim:] == -3.0).all()
    # into a transposed table
    gt = torch.full((dim, vocab), 9.0, device=cuda)
    abi.embedding_grad(view(out), tv, view(gt.t()))
    assert torch.equal(gt.t(), store[:, 2:2 + dim])


def test_embedding_reports_tokens_outside_the_table(cuda):
    import torch

    table = torch.randn(10, 8, device=cuda)
    for bad in (10, -1, 2 ** 40):
        tok = torch.tensor([1, bad, 3], device=cuda)
        out = torch.full((3, 8), 5.0, device=cuda)
        abi.embedding(view(table), view(tok), view(out))
        with pytest.raises(IndexError, match=str(bad)):
            abi.check_device_errors(0)
        assert torch.equal(out[[0, 2]], table[[1, 3]]) and (out[1] == 5.0).all()
        grad = torch.empty(10, 8, device=cuda)
        abi.embedding_grad(view(out), view(tok), view(grad))
        with pytest.raises(IndexError, match=str(bad)):
            abi.check_device_errors(0)
        want = torch.zeros(10, 8, device=cuda)
        want[1], want[3] = out[0], out[2]
        assert torch.equal(grad, want)
    abi.check_device_errors(0)


def test_embedding_gradient_of_a_single_token_and_of_nothing(cuda):
    """All positions hold one token (a run over every piece), or only padding, or there is none."""
    import torch

    d = torch.randn(3001, 40, device=cuda)
    tok = torch.full((3001,), 4, device=cuda)
    got = torch.full((6, 40), 8.0, device=cuda)
    abi.embedding_grad(view(d), view(tok), view(got))
    want = torch.zeros(6, 40, dtype=torch.float64, device=cuda)
    want[4] = d.double().sum(0)
    within(got, want, 3002 * U * d.double().abs().sum(0) * torch.tensor([0, 0, 0, 0, 1, 0], device=cuda).unsqueeze(1)
           + 1e-45, "one token")
    abi.embedding_grad(view(d), view(tok), view(got), padding_token=4)
    assert (got == 0).all()
    got.fill_(3.0)
    abi.embedding_grad(view(d[:0]), view(tok[:0]), view(got))
    assert (got == 0).all()
    got.fill_(3.0)
    abi.embedding_grad(view(d[:0]), view(tok[:0]), view(got), accumulate=True)
    assert (got == 3.0).all()


def test_embedding_beyond_32_bits(cuda):
    """A table of 4.7e9 elements: rows behind 2^32 elements are read, summed and cleared."""
    import torch

    vocab, dim = 2300000, 2048
    table = torch.zeros(vocab, dim, device=cuda)
    high = torch.tensor([vocab - 1, 5, vocab - 2, 2 ** 21, 2 ** 21 + 1, vocab - 1], device=cuda)
    table[high] = torch.randn(6, dim, device=cuda)
    out = torch.empty(6, dim, device=cuda)
    abi.embedding(view(table), view(high), view(out), scale=2.0)
    assert torch.equal(out, table[high] * 2.0)
    for tok in (high, high.repeat(60)):  # with and without the sort
        d = torch.randn(tok.numel(), dim, device=cuda)
        table.fill_(3.0)
        abi.embedding_grad(view(d), view(tok), view(table))
        abi.check_device_errors(0)
        for v in high.unique().tolist():
            mine = d[tok == v].double()
            within(table[v], mine.sum(0), (mine.shape[0] + 1) * U * 1.01 * mine.abs().sum(0) + 1e-45, f"row {v}")
            table[v] = 0.0
        assert not table.any()


def test_embedding_of_one_scalar_token(cuda):
    import torch

    table, tok, out = torch.randn(9, 33, device=cuda), torch.tensor(4, device=cuda), torch.empty(33, device=cuda)
    abi.embedding(view(table), view(tok), view(out), scale=0.5)
    assert torch.equal(out, table[4] * 0.5)
    grad = torch.empty(9, 33, device=cuda)
    abi.embedding_grad(view(out), view(tok), view(grad), scale=2.0)
    assert torch.equal(grad[4], out * 2.0) and grad.count_nonzero() == out.count_nonzero()


def test_embedding_keeps_infinities_and_nan_to_their_rows(cuda):
    import torch

    d = torch.randn(64, 16, device=cuda)
    tok = torch.arange(64, device=cuda) % 8
    d[3, 5], d[10, 1] = float("nan"), float("inf")
    tok[20] = 0
    d[20] = float("nan")  # a padded position may hold anything
    got = torch.empty(8, 16, device=cuda)
    abi.embedding_grad(view(d), view(tok), view(got), padding_token=0)
    assert got[3].isnan().nonzero().flatten().tolist() == [5]
    assert got[2].isinf().nonzero().flatten().tolist() == [1]
    rest = torch.ones(8, 16, dtype=torch.bool, device=cuda)
    rest[3, 5] = rest[2, 1] = False
    assert got[rest].isfinite().all() and (got[0] == 0).all()


# ------------------------------------------------------------ cross entropy --

def ce_reference(x, w, b, t, dloss):
    """(loss, lse, dx, dw, db) and their bounds, in float64."""
    import torch

    n, dim = x.shape
    vocab = w.shape[0]
    live = t != IGNORE
    xd, wd = torch.where(live.unsqueeze(1), x.double(), 0.0), w.double()
    bd = torch.zeros(vocab, dtype=torch.float64, device=x.device) if b is None else b.double()
    z = xd @ wd.t() + bd
    dz = product_bound(dim, xd.abs() @ wd.abs().t()) + 2 * U * (z.abs() + bd.abs())
    lse = torch.logsumexp(z, 1)
    at = torch.where(live, t, 0).unsqueeze(1)
    zt = z.gather(1, at).squeeze(1)
    loss = torch.where(live, lse - zt, 0.0)
    p = torch.exp(z - lse.unsqueeze(1))
    top_err = (p * dz).sum(1)  # the logsumexp's derivative in z is p
    dlse = top_err * (1 + 1e-3) + (vocab / 256 + 32) * 2 * U + 4 * U * lse.abs()
    dl = dlse + dz.gather(1, at).squeeze(1) + 4 * U * (lse.abs() + zt.abs())
    lse = torch.where(live, lse, 0.0)
    out = {"loss": (loss, dl), "lse": (lse, dlse)}
    if dloss is None:
        return out
    d = torch.where(live, dloss.double(), 0.0).unsqueeze(1)
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    g = d * (p - hot)
    # exponent: z and lse with their errors, and the rounding of their difference
    e = dz + dlse.unsqueeze(1) + 2 * U * (z.abs() + lse.abs().unsqueeze(1))
    dg = d.abs() * p * (torch.expm1(e) + 8 * U) + 8 * U * g.abs() + 2.0 ** -40 * d.abs().max() * live.unsqueeze(1)
    ax, aw, ag = xd.abs(), wd.abs(), g.abs()
    out["dx"] = (g @ wd, dg @ aw + product_bound(vocab, ag @ aw))
    out["dw"] = (g.t() @ xd, dg.t() @ ax + product_bound(n, ag.t() @ ax))
    out["db"] = (g.sum(0), dg.sum(0) + product_bound(n, ag.sum(0)))
    return out


def ce_data(n, vocab, dim, seed, ignored=0.0, spread=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, dim, device="cuda", generator=g)
    w = torch.randn(vocab, dim, device="cuda", generator=g) * (spread * 2 / math.sqrt(max(dim, 1)))
    b = torch.randn(vocab, device="cuda", generator=g)
    t = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    if ignored:
        t[torch.rand(n, device="cuda", generator=g) < ignored] = IGNORE
    dloss = torch.randn(n, device="cuda", generator=g) / max(n, 1)
    return x, w, b, t, dloss


def run_ce(x, w, b, t, dloss, stream=None):
    import torch

    n, vocab = x.shape[0], w.shape[0]
    loss, lse = (torch.full((n,), 99.0, device=x.device) for _ in range(2))
    bias = None if b is None else view(b)
    if dloss is None:
        abi.linear_cross_entropy(view(x), view(w), view(t), view(loss), bias=bias, lse=view(lse), ignore_target=IGNORE,
                                 stream=stream)
        return {"loss": loss, "lse": lse}
    dx, dw = torch.full_like(x, 99.0), torch.full_like(w, 99.0)
    db = torch.full((vocab,), 99.0, device=x.device)
    abi.linear_cross_entropy_grad(view(x), view(w), view(t), view(dloss), dx=view(dx), dweight=view(dw), bias=bias,
                                  dbias=view(db), loss=view(loss), lse=view(lse), ignore_target=IGNORE, stream=stream)
    return {"loss": loss, "lse": lse, "dx": dx, "dw": dw, "db": db}


def check_ce(x, w, b, t, dloss):
    got = run_ce(x, w, b, t, dloss)
    abi.check_device_errors(0)
    want = ce_reference(x, w, b, t, dloss)
    for name, value in got.items():
        within(value, want[name][0], want[name][1] + 1e-42, f"{name} of {tuple(x.shape)} x {w.shape[0]}")
    return got


# one row and one class; tiles of 64, 128 and 256 met, missed by one and passed by
# one in each direction
CE_SHAPES = [(1, 1, 1), (1, 2, 1), (1, 1000, 64), (2, 3, 5), (5, 257, 63), (64, 64, 64), (65, 63, 66), (127, 129, 128),
             (128, 256, 64), (129, 255, 200), (300, 3, 64), (256, 512, 256), (257, 513, 129), (1000, 1000, 96),
             (513, 5003, 77), (2300, 301, 320), (33, 20011, 257), (4096, 40, 1024), (700, 1500, 1),
             (5000, 3, 300), (3000, 16, 130), (9001, 7, 97), (300, 1, 20000), (70000, 2, 33), (2000, 11, 256),
             (600, 400, 128), (500, 385, 385), (520, 384, 290), (300, 2000, 771), (16, 700, 515), (13, 3001, 640), (3, 5000, 1100), (1, 90001, 50), (17, 900, 400),
             (60, 200, 4096), (17, 17, 5000), (700, 900, 2047), (1300, 1025, 1100), (19, 3000, 1024)]


@pytest.mark.parametrize("n, vocab, dim", CE_SHAPES)
def test_linear_cross_entropy_and_gradients(cuda, n, vocab, dim):
    x, w, b, t, dloss = ce_data(n, vocab, dim, n + vocab + dim, ignored=0.2 if n > 4 else 0.0)
    grads = check_ce(x, w, b, t, dloss)
    alone = check_ce(x, w, b, t, None)
    check_ce(x, w, None, t, dloss)
    import torch

    assert ((grads["loss"] == 0) == (alone["loss"] == 0)).all()
    dead = t == IGNORE
    assert (grads["dx"][dead] == 0).all() and (grads["loss"][dead] == 0).all() and (alone["lse"][dead] == 0).all()
    again = run_ce(x, w, b, t, dloss)
    for k in grads:
        assert torch.equal(grads[k], again[k]), f"{k} differs from run to run"


@pytest.mark.parametrize("n, vocab, dim", [(6, 40, 16), (300, 1000, 80), (1500, 3000, 64), (4000, 6, 200), (9, 3000, 170)])
def test_linear_cross_entropy_takes_views_of_any_layout(cuda, n, vocab, dim):
    """Transposed and padded operands, odd offsets, a broadcast dloss, every second
    target; what lies beside the outputs stays."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 5, ignored=0.1)
    xt = x.t().contiguous().t()
    ws = torch.randn(vocab, dim + 3, device=cuda)
    ws[:, 1:1 + dim] = w
    wv = ws[:, 1:1 + dim]
    ts = torch.stack([t, torch.full_like(t, 10 ** 9)], 1)
    tv = ts[:, 0]
    bs = torch.stack([b, b + 1], 1)
    dl = torch.full((1,), 0.25, device=cuda).expand(n)
    dxs = torch.full((n, dim + 2), 55.0, device=cuda)
    dwt = torch.full((dim, vocab + 1), 55.0, device=cuda)
    lo = torch.full((n + 1, 2), 55.0, device=cuda)
    db = torch.full((vocab, 3), 55.0, device=cuda)
    abi.linear_cross_entropy_grad(view(xt), view(wv), view(tv), view(dl), dx=view(dxs[:, 1:1 + dim]),
                                  dweight=view(dwt[:, 1:].t()), bias=view(bs[:, 0]), dbias=view(db[:, 1]),
                                  loss=view(lo[1:, 0]), ignore_target=IGNORE)
    abi.check_device_errors(0)
    want = ce_reference(x, w, b, t, dl)
    for name, got in (("dx", dxs[:, 1:1 + dim]), ("dw", dwt[:, 1:].t()), ("loss", lo[1:, 0]), ("db", db[:, 1])):
        within(got, want[name][0], want[name][1] + 1e-42, name)
    assert (dxs[:, 0] == 55).all() and (dxs[:, -1] == 55).all() and (dwt[:, 0] == 55).all()
    assert (lo[0] == 55).all() and (lo[:, 1] == 55).all() and (db[:, 0] == 55).all() and (db[:, 2] == 55).all()


@pytest.mark.parametrize("n, vocab, dim", [(40, 30, 20), (600, 1000, 96), (1100, 2048, 256), (3000, 10, 150), (12, 4000, 200)])
def test_ignored_rows_may_hold_anything(cuda, n, vocab, dim):
    """NaN and infinities in rows without a loss reach no output; with all rows
    ignored every gradient is zero."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 8)
    t[::3] = IGNORE
    clean = run_ce(x, w, b, t, dloss)
    x[::6], x[3::6] = float("nan"), float("inf")
    dloss = dloss.clone()
    dloss[::3] = float("nan")
    dirty = run_ce(x, w, b, t, dloss)
    for k in clean:
        assert torch.equal(clean[k], dirty[k]), k
    none = run_ce(x, w, b, torch.full_like(t, IGNORE), dloss)
    for k, v in none.items():
        assert (v == 0).all(), k
    one = torch.full_like(t, IGNORE)
    one[n // 2 + (n // 2) % 3 + 1] = vocab - 1
    x2 = torch.where((one == IGNORE).unsqueeze(1), float("nan"), ce_data(n, vocab, dim, 9)[0])
    check_ce(x2, w, b, one, torch.ones(n, device=cuda))


@pytest.mark.parametrize("n, vocab, dim", [(40, 30, 20), (600, 1000, 96), (3000, 13, 150), (15, 4000, 100)])
def test_targets_outside_the_vocabulary_are_reported(cuda, n, vocab, dim):
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 10)
    for bad in (vocab, -1, 2 ** 33):
        tb = t.clone()
        tb[7] = bad
        got = run_ce(x, w, b, tb, dloss)
        with pytest.raises(IndexError, match=str(bad)):
            abi.check_device_errors(0)
        ti = t.clone()
        ti[7] = IGNORE
        want = run_ce(x, w, b, ti, dloss)
        abi.check_device_errors(0)
        for k in got:
            assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("n, vocab, dim", [(30, 50, 24), (520, 1030, 72), (2200, 12, 170), (10, 3000, 150)])
def test_non_finite_rows_stay_rows(cuda, n, vocab, dim):
    """NaN and infinite x: that row's loss and dx are not finite, the others are as before."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 12)
    want = run_ce(x, w, b, t, dloss)
    bad = x.clone()
    bad[3, 1], bad[9, 0] = float("nan"), float("inf")
    got = run_ce(bad, w, b, t, dloss)
    rows = torch.ones(n, dtype=torch.bool, device=cuda)
    rows[3] = rows[9] = False
    assert torch.equal(got["loss"][rows], want["loss"][rows]) and torch.equal(got["dx"][rows], want["dx"][rows])
    assert not got["loss"][~rows].isfinite().any() and not got["dx"][~rows].isfinite().any()
    assert not got["dw"].isfinite().any()


@pytest.mark.parametrize("n, vocab, dim", [(50, 70, 33), (400, 900, 130), (3000, 9, 160), (7, 2000, 330)])
@pytest.mark.parametrize("sx, sw", [(1e-30, 1.0), (1e25, 1e-25), (1.0, 1e-38), (3e-42, 1.0), (1e30, 1e-38)])
def test_scales_far_from_one(cuda, n, vocab, dim, sx, sw):
    """Operands near the ends of float32's range; the products stay in it."""
    x, w, b, t, dloss = ce_data(n, vocab, dim, 14)
    check_ce(x * sx, w * sw, b, t, dloss)
    check_ce(x, w, b, t, dloss * 1e-30)


def test_scales_that_a_sample_misses(cuda):
    """A few rows far larger than the others, or all others zero: the scale of the 16-bit
    pairs is that of the largest all the same."""
    x, w, b, t, dloss = ce_data(3000, 2500, 80, 24)
    big = x.clone()
    big[1] *= 3e4
    check_ce(big * 1e-3, w, b, t, dloss)
    wide = w.clone()
    wide[3], wide[2401] = wide[3] * 1e3, wide[2401] * 300.0
    check_ce(x * 1e-2, wide, b, t, dloss)
    lone = x * 0.0
    lone[1], lone[2] = x[1], x[2] * 1e-4
    check_ce(lone, w, b, t, dloss)
    check_ce(lone * 0.0, w * 0.0, b, t, dloss)


@pytest.mark.parametrize("n, vocab, dim", [(40, 60, 16), (520, 1300, 100), (3000, 8, 200), (6, 4000, 200)])
def test_confident_rows_keep_small_gradients(cuda, n, vocab, dim):
    """Logits so far apart that p is 1 - 1e-9 at the target and 1e-30 elsewhere: the
    gradient's entries span 30 decades and stay inside their bounds."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 15, spread=6.0)
    x = x + 12.0 * w[t] / w[t].norm(dim=1, keepdim=True)
    got = check_ce(x, w, b, t, torch.ones(n, device=cuda))
    assert got["loss"].min() >= 0


@pytest.mark.parametrize("n, vocab, dim", [(37, 53, 29), (530, 700, 120), (3000, 15, 120), (5, 5000, 180)])
def test_rare_classes_keep_their_precision(cuda, n, vocab, dim):
    """A class of probability 1e-9 in every row: its weight gradient is 1e9 times
    smaller than the others' and still accurate to 1e-4 of itself, as the float32
    product of float32 gradients is (n * 2^-24 and the exponent's rounding, 30 * 2^-24)."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 16, spread=0.5)
    t = t % (vocab - 1)
    b = b.clone()
    b[vocab - 1] = -20.0
    got = run_ce(x, w, b, t, torch.ones(n, device=cuda))
    want = ce_reference(x, w, b, t, torch.ones(n, device=cuda))["dw"][0]
    rel = (got["dw"][-1].double() - want[-1]).norm() / want[-1].norm()
    assert rel <= 1e-4, rel


@pytest.mark.parametrize("n, vocab, dim", [(9, 12, 7), (150, 280, 66)])
def test_gradients_against_differences(cuda, n, vocab, dim):
    """Directional differences of the loss, evaluated in float64 by the definition at
    points around the operands, against the kernel's gradients."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 17, ignored=0.1)
    got = run_ce(x, w, b, t, dloss)

    def total(xx, ww, bb):
        live = t != IGNORE
        z = xx @ ww.t() + bb
        zt = z.gather(1, torch.where(live, t, 0).unsqueeze(1)).squeeze(1)
        return (dloss.double() * live * (torch.logsumexp(z, 1) - zt)).sum().item()

    args = [x.double(), w.double(), b.double()]
    for k, name in enumerate(("dx", "dw", "db")):
        torch.manual_seed(k)
        step = torch.randn_like(args[k])
        h = 1e-4
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + h * step, args[k] - h * step
        diff = (total(*up) - total(*down)) / (2 * h)
        along = (got[name].double() * step).sum().item()
        size = (got[name].double().abs() * step.abs()).sum().item()
        # h^2 of the third derivative (below the first's size times |z step|^2), and float32 rounding
        assert abs(along - diff) <= 1e-4 * size + 1e-12, name


def test_linear_cross_entropy_of_no_rows(cuda):
    import torch

    x, w = torch.empty(0, 8, device=cuda), torch.randn(5, 8, device=cuda)
    t, e = torch.empty(0, dtype=torch.int64, device=cuda), torch.empty(0, device=cuda)
    dw, db = torch.full((5, 8), 4.0, device=cuda), torch.full((5,), 4.0, device=cuda)
    abi.linear_cross_entropy_grad(view(x), view(w), view(t), view(e), dweight=view(dw), dbias=view(db), loss=view(e))
    assert (dw == 0).all() and (db == 0).all()


def test_each_gradient_alone_equals_all_together(cuda):
    """Outputs that are not asked for are not written, and the others do not change."""
    import torch

    for n, vocab, dim in ((40, 60, 16), (300, 900, 70), (3000, 14, 110), (11, 2500, 170)):
        x, w, b, t, dloss = ce_data(n, vocab, dim, 21, ignored=0.2)
        all_ = run_ce(x, w, b, t, dloss)
        for name, shape in (("dx", x.shape), ("dw", w.shape), ("db", b.shape), ("loss", t.shape), ("lse", t.shape)):
            out = torch.full(shape, 77.0, device=cuda)
            kw = {{"dw": "dweight", "db": "dbias"}.get(name, name): view(out)}
            abi.linear_cross_entropy_grad(view(x), view(w), view(t), view(dloss), bias=view(b), ignore_target=IGNORE, **kw)
            assert torch.equal(out, all_[name]), name


@pytest.mark.parametrize("n, vocab, dim", [(40, 90, 16), (6, 3000, 150), (3000, 12, 130), (400, 1700, 96)])
@pytest.mark.parametrize("low", [-math.inf, -3.4028234663852886e38])
def test_classes_masked_by_the_bias(cuda, n, vocab, dim, low):
    """A bias of -inf, or of the type's lowest value, takes classes out, whole tiles of
    them too: the results are those of the other classes alone, and the masked classes'
    gradients are exact zeros."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 19, ignored=0.1)
    masked = torch.rand(vocab, device=cuda) < 0.4
    masked[: vocab // 2] = True
    masked[vocab - 1] = False
    rest = (~masked).nonzero().flatten()
    pick = rest[torch.randint(0, rest.numel(), (n,), device=cuda)]
    t = torch.where(t == IGNORE, t, pick)
    bm = torch.where(masked, low, b)
    got = run_ce(x, w, bm, t, dloss)
    index = torch.full((vocab,), IGNORE, device=cuda)
    index[rest] = torch.arange(rest.numel(), device=cuda)
    tr = torch.where(t == IGNORE, t, index[t.clamp(min=0)])
    want = ce_reference(x, w[rest], b[rest], tr, dloss)
    extra = (vocab / 256 + 32) * 2 * U  # the sums run over all classes
    for k in ("loss", "lse", "dx"):
        scale = 1.0 if k != "dx" else (dloss.abs().max().double() * w.abs().max().double() * vocab)
        within(got[k], want[k][0], want[k][1] + extra * scale, k)
    within(got["dw"][rest], want["dw"][0], want["dw"][1] + extra * x.abs().sum(0).double() * dloss.abs().max(), "dw")
    within(got["db"][rest], want["db"][0], want["db"][1] + extra * dloss.abs().sum(), "db")
    assert (got["dw"][masked] == 0).all() and (got["db"][masked] == 0).all()


def test_linear_cross_entropy_without_columns(cuda):
    """D = 0: the logits are the bias."""
    import torch

    for n, vocab in ((30, 40), (3, 700), (500, 3000), (5000, 7)):
        x, w, b, t, dloss = ce_data(n, vocab, 0, 23, ignored=0.1)
        check_ce(x, w, b, t, dloss)
        check_ce(x, w, None, t, None)


@pytest.mark.parametrize("n, vocab, dim", [(1, 4, 450), (5, 200, 64), (1, 3000, 515), (3, 1000, 64), (16, 700, 128),
                                           (4000, 6, 1024), (9001, 16, 64)])
@pytest.mark.parametrize("gap", [3.0, 11.5, 18.0, 40.0])
def test_rows_sure_of_their_class_keep_the_digits_of_what_is_left(cuda, n, vocab, dim, gap):
    """Logits that float32 holds exactly, one far above the others: 1 - p is lost in 1, and is
    the gradient.  The logarithm of a probability is rounded once beside its value, and an
    exponential is off by that and two units more."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 26)
    steps = torch.round(w[:, :1] * 8).clamp(-16, 16) / 8
    x, w = torch.zeros_like(x), torch.zeros_like(w)
    x[:, 0], w[:, :1] = 1.0, steps
    w[vocab // 2, 0] = 3.0 + gap
    t = torch.full_like(t, vocab // 2)
    dloss = torch.ones_like(dloss)
    got = run_ce(x, w, None, t, dloss)
    z = w[:, 0].double()
    logp = z - torch.logsumexp(z, 0)
    others = torch.arange(vocab, device=cuda) != vocab // 2
    rest = torch.logsumexp(z[others], 0) - torch.logsumexp(z, 0)  # log(1 - p), without the difference
    g = torch.where(others, logp.exp(), -rest.exp())
    rel = 2 * U * (logp.abs().max() + 10)
    loss = -torch.log1p(-rest.exp())
    # The sum of exponentials lies in [1, 2) and is a float64: each of its at most `vocab`
    # additions rounds by half a step, 2^-53, at most, and the logarithm of 1 + r is within r.
    # (A gap of 40 leaves 1 - p below the first step.)
    step = vocab * 2.0 ** -53 * 1.01
    within(got["loss"], loss.expand(n), (rel * loss + step).expand(n), "loss")
    within(got["db"], n * g, (rel + 2 * U * n) * n * g.abs() + n * step, "db")
    within(got["dw"][:, 0], n * g, (rel + 2 * U * n) * n * g.abs() + n * step, "dw")


@pytest.mark.parametrize("n, vocab, dim", [(300, 100, 512), (300, 128, 512), (600, 1000, 96), (60, 200, 4096), (17, 900, 400)])
@pytest.mark.parametrize("gap", [3.0, 11.5, 18.0])
def test_rows_sure_of_their_class_on_the_tensor_cores(cuda, n, vocab, dim, gap):
    """The same where the sums of exponentials are taken 128 classes at a time, logits split along
    the columns among them: the digits of what is left come from a sum that the largest logit's 1
    is not part of.

    The logits are exact, and so are their differences.  An exponential, 2^x by the hardware within
    2^-22 (4u) of an argument that two roundings put off by u |x| each, is within (2 |x| + 4) u; 36
    additions of positive terms are within 36u, the joining exponential within 4u: the sum of the
    others is within (2 |x| + 46) u of itself, its log1p and exponentials of it within 6u more.
    (From a sixteenth of the largest on, 16 of the others may share a sum with it: the 19 additions
    to its 1 + rest are 17 times as much of the rest.)
    The gradient's pairs hold 2^-22 of it and 2^-48 of the largest |dloss|."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 28)
    steps = torch.round(w[:, :1] * 8).clamp(-16, 16) / 8
    x, w = torch.zeros_like(x), torch.zeros_like(w)
    x[:, 0], w[:, :1] = 1.0, steps
    w[vocab // 2, 0] = 3.0 + gap
    t = torch.full_like(t, vocab // 2)
    dloss = torch.ones_like(dloss)
    got = run_ce(x, w, None, t, dloss)
    alone = run_ce(x, w, None, t, None)
    assert torch.equal(alone["loss"], got["loss"]) and torch.equal(alone["lse"], got["lse"])
    z = w[:, 0].double()
    logp = z - torch.logsumexp(z, 0)
    others = torch.arange(vocab, device=cuda) != vocab // 2
    rest = torch.logsumexp(z[others], 0) - torch.logsumexp(z, 0)
    g = torch.where(others, logp.exp(), -rest.exp())
    shared = 19 * 17 if rest.exp() / (1 - rest.exp()) > 0.06 else 0
    rel = U * (2 * logp.abs().max() + 52 + 4 * 4 + shared)
    loss = -torch.log1p(-rest.exp())
    within(got["loss"], loss.expand(n), (rel * loss).expand(n), "loss")
    within(got["db"], n * g, (rel + 2 * U * n) * n * g.abs(), "db")
    within(got["dw"][:, 0], n * g, (rel + 2 * U * (n + 16)) * n * g.abs() + n * 2.0 ** -48, "dw")


def own_bounds(x, w, b, t, dloss):
    """(dx, dw, db) in float64 and bounds by each row's and each class's own size: an entry of g is
    off by its rounding errors, relative to itself, and by its pair of 16-bit floats, 2^-22 of itself
    and 2^-48 of the largest entry of its row (dx) or class (dw)."""
    import torch

    live = (t != IGNORE).unsqueeze(1)
    xd, wd = torch.where(live, x.double(), 0.0), w.double()
    z = xd @ wd.t() + b.double()
    dz = product_bound(x.shape[1], xd.abs() @ wd.abs().t()) + 2 * U * (z.abs() + b.double().abs())
    lse = torch.logsumexp(z, 1, keepdim=True)
    at = torch.where(live, t.unsqueeze(1), 0)
    p = torch.exp(z - lse)
    dlse = (p * dz).sum(1, keepdim=True) * (1 + 1e-3) + (w.shape[0] / 256 + 32) * 2 * U + 4 * U * lse.abs()
    others = torch.ones_like(p).scatter_(1, at, 0.0)
    left = (p * others).sum(1, keepdim=True)  # 1 - p of the target, without the difference
    d = torch.where(live, dloss.double().unsqueeze(1), 0.0)
    g = d * (p * others - left * (1.0 - others))
    e = dz + dlse + 2 * U * (z.abs() + lse.abs())
    up = (torch.exp((z - lse + e).clamp(max=0.0)) - p) * others  # p at the end of its exponent's range
    up = up + up.sum(1, keepdim=True).clamp(max=1.0) * (1.0 - others)  # and what is left of the target's
    dg = d.abs() * up + 16 * U * g.abs()
    ag, ax, aw = g.abs(), xd.abs(), wd.abs()
    by_row, by_class = 2.0 ** -48 * ag.amax(1, keepdim=True), 2.0 ** -48 * ag.amax(0, keepdim=True)
    return {"dx": (g @ wd, (dg + by_row) @ aw + product_bound(w.shape[0], ag @ aw)),
            "dw": (g.t() @ xd, (dg + by_class * live).t() @ ax + product_bound(x.shape[0], ag.t() @ ax)),
            "db": (g.sum(0), dg.sum(0) + product_bound(x.shape[0], ag.sum(0)))}


def check_own(x, w, b, t, dloss):
    got = run_ce(x, w, b, t, dloss)
    abi.check_device_errors(0)
    want = {**ce_reference(x, w, b, t, None), **own_bounds(x, w, b, t, dloss)}
    for name, (value, tol) in want.items():
        within(got[name], value, tol + 1e-42, name)
    return got


GRADIENT_SHAPES = [(37, 53, 29), (530, 700, 120), (1031, 903, 65), (3000, 15, 120), (5, 5000, 180), (17, 900, 400)]


@pytest.mark.parametrize("n, vocab, dim", GRADIENT_SHAPES)
def test_gradients_of_classes_improbable_everywhere(cuda, n, vocab, dim):
    """Classes of probabilities down to 1e-35 in every row: their rows of dweight are held to their
    own size, not to that of the other classes'."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 33, ignored=0.1, spread=0.5)
    t = torch.where(t == IGNORE, t, t % (vocab - 8))
    b = b.clone()
    b[vocab - 8:] = -torch.arange(10.0, 81.0, 10.0, device=cuda)
    got = check_own(x, w, b, t, torch.ones(n, device=cuda))
    assert (got["dw"][vocab - 8:] != 0).any(1).all() and got["dw"][-1].abs().max() < 1e-25


@pytest.mark.parametrize("n, vocab, dim", GRADIENT_SHAPES)
def test_gradients_of_rows_with_a_small_share_of_the_loss(cuda, n, vocab, dim):
    """dloss over thirty decades, in no order: each row of dx is held to its own size."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 34, ignored=0.1)
    g = torch.Generator(device="cuda").manual_seed(1)
    share = 10.0 ** -torch.linspace(0, 30, n, device=cuda)[torch.randperm(n, device=cuda, generator=g)]
    got = check_own(x, w, b, t, dloss.sign() * share)
    assert (got["dx"][t != IGNORE] != 0).any(1).all()


@pytest.mark.parametrize("n, vocab, dim", [(530, 700, 120), (1031, 903, 65), (17, 900, 400), (60, 200, 4095)])
def test_gradients_of_rows_sure_of_their_class(cuda, n, vocab, dim):
    """Rows sure of their class to 1e-3 and to 1e-30, side by side, on the tensor cores."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 35, ignored=0.1, spread=0.25)
    at = torch.where(t == IGNORE, 0, t)
    w = torch.cat([w, torch.zeros(vocab, 1, device=cuda)], 1)
    w[:, -1] = torch.where(torch.arange(vocab, device=cuda) == vocab // 2, 1.0, 0.0)
    lift = torch.linspace(8, 70, n, device=cuda).unsqueeze(1)
    t = torch.where(t == IGNORE, t, vocab // 2)
    check_own(torch.cat([x, lift], 1), w, b * 0.1, t, torch.ones(n, device=cuda))


@pytest.mark.parametrize("n, vocab, dim", [(300, 100, 512), (300, 128, 512), (600, 1000, 96), (60, 200, 4096), (17, 900, 400),
                                           (1, 4, 450), (5, 200, 64), (1, 3000, 515), (3, 1000, 64), (16, 700, 128),
                                           (4000, 6, 1024), (9001, 16, 64), (300, 3, 64), (40, 90, 16)])
@pytest.mark.parametrize("gap", [40.0, 75.0])
def test_gradients_below_the_first_step_of_one(cuda, n, vocab, dim, gap):
    """What is left next to a probability that float64 too holds as 1, by the bounds of
    test_rows_sure_of_their_class_on_the_tensor_cores without the share of the largest |dloss|."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 28)
    steps = torch.round(w[:, :1] * 8).clamp(-16, 16) / 8
    x, w = torch.zeros_like(x), torch.zeros_like(w)
    x[:, 0], w[:, :1] = 1.0, steps
    w[vocab // 2, 0] = 3.0 + gap
    t = torch.full_like(t, vocab // 2)
    got = run_ce(x, w, None, t, torch.ones_like(dloss))
    z = w[:, 0].double()
    logp = z - torch.logsumexp(z, 0)
    others = torch.arange(vocab, device=cuda) != vocab // 2
    rest = torch.logsumexp(z[others], 0) - torch.logsumexp(z, 0)
    g = torch.where(others, logp.exp(), -rest.exp())
    rel = U * (2 * logp.abs().max() + 52 + 4 * 4)
    within(got["loss"], rest.exp().expand(n), (rel * rest.exp()).expand(n), "loss")
    within(got["db"], n * g, (rel + 2 * U * n) * n * g.abs(), "db")
    within(got["dw"][:, 0], n * g, (rel + 2 * U * (n + 16)) * n * g.abs(), "dw")
    # p of the other classes is the same in every row: dx is their logits' mean less the target's
    dx = (g * z).sum()
    within(got["dx"][:, 0], dx.expand(n), ((rel + 2 * U * (vocab + 16)) * (g * z).abs().sum()).expand(n), "dx")


# float32 path of few rows, one piece and several, logits split along the columns, a scale from a
# sample of the rows, and neither dimension a multiple of anything
UNLIKE_SHAPES = [(16, 700, 120), (300, 2000, 256), (520, 1300, 100), (60, 200, 4096), (3000, 2500, 80), (1301, 1999, 131)]


@pytest.mark.parametrize("n, vocab, dim", UNLIKE_SHAPES)
@pytest.mark.parametrize("size", [1e8, 1e12, 1e15, 1e25])
def test_a_large_row_leaves_the_others_their_digits(cuda, n, vocab, dim, size):
    """A row of x, or of the weight, far larger than the others: each other row's loss and dx, and
    each class's dweight, stay within what the sums of their own products allow."""
    x, w, b, t, dloss = ce_data(n, vocab, dim, 36, ignored=0.1)
    t[0] = t[7] = vocab // 2
    for at in (0, 7):
        big = x.clone()
        big[at] *= size
        check_own(big, w, b, t, dloss)
    for at in (3, vocab - 1):
        big = w.clone()
        big[at] *= size
        check_own(x, big, b, t, dloss)


@pytest.mark.parametrize("n, vocab, dim", UNLIKE_SHAPES)
def test_rows_and_columns_of_unlike_size(cuda, n, vocab, dim):
    """Rows of x over 25 decades, rows of the weight over 20, columns over 30 (of x and, the other
    way round, of the weight), and columns of either alone: features in units of their own."""
    import torch

    x, w, b, t, dloss = ce_data(n, vocab, dim, 37, ignored=0.1)
    g = torch.Generator(device="cuda").manual_seed(2)

    def decades(low, high, count):
        order = torch.randperm(count, device=cuda, generator=g)
        return 10.0 ** torch.linspace(low, high, count, device=cuda)[order]

    check_own(x * decades(-22, 3, n).unsqueeze(1), w, b, t, dloss)
    check_own(x, w * decades(-18, 2, vocab).unsqueeze(1), b, t, dloss)
    both = decades(-15, 15, dim)
    check_own(x * both, w / both, b, t, dloss)
    check_own(x * decades(-20, 0, dim), w, b, t, dloss)
    check_own(x, w * decades(-20, 0, dim), b, t, dloss)
    rare = x.clone()
    rare[:, 1] *= 1e-12
    check_own(rare, w, b, t, dloss)


def test_operands_of_unlike_size_through_views_of_any_layout(cuda):
    """As test_linear_cross_entropy_takes_views_of_any_layout, with rows and columns that the pairs
    do not hold; NaN in rows without a loss; each gradient alone."""
    import torch

    n, vocab, dim = 523, 1111, 139
    x, w, b, t, dloss = ce_data(n, vocab, dim, 38, ignored=0.2)
    x[5] *= 1e13
    w[:, 3] *= 1e-14
    t[5] = 4
    xt = x.t().contiguous().t()
    ws = torch.randn(vocab, dim + 3, device=cuda)
    ws[:, 1:1 + dim] = w
    bs = torch.stack([b, b + 1], 1)
    xn = xt.clone()
    xn[t == IGNORE] = float("nan")
    want = {**ce_reference(x, w, b, t, None), **own_bounds(x, w, b, t, dloss)}
    out = {"dx": torch.full((n, dim + 2), 55.0, device=cuda)[:, 1:1 + dim],
           "dw": torch.full((dim, vocab + 1), 55.0, device=cuda)[:, 1:].t(),
           "db": torch.full((vocab, 3), 55.0, device=cuda)[:, 1], "loss": torch.full((n,), 55.0, device=cuda)}
    names = {"dw": "dweight", "db": "dbias"}
    args = view(xn), view(ws[:, 1:1 + dim]), view(t), view(dloss)
    abi.linear_cross_entropy_grad(*args, bias=view(bs[:, 0]), ignore_target=IGNORE,
                                  **{names.get(k, k): view(v) for k, v in out.items()})
    abi.check_device_errors(0)
    for k, v in out.items():
        within(v, want[k][0], want[k][1] + 1e-42, k)
    for k, v in out.items():
        alone = torch.full(v.shape, 44.0, device=cuda)
        abi.linear_cross_entropy_grad(*args, bias=view(bs[:, 0]), ignore_target=IGNORE, **{names.get(k, k): view(alone)})
        assert torch.equal(alone, v), k


@pytest.mark.parametrize("n, vocab, dim", [(2 ** 21 - 1, 1, 1), (2 ** 21 - 1, 2, 0), (2 ** 20, 3, 0), (2 ** 20 - 1, 3, 0)])
def test_more_rows_than_a_grid_has_parts(cuda, n, vocab, dim):
    """Where 32 rows a CTA would be more than the 65535 parts of a launch's second axis."""
    check_ce(*ce_data(n, vocab, dim, 25, ignored=0.1))


def test_more_rows_than_a_piece_of_the_logits_holds(cuda):
    """4.7 GB of logits: the rows go in two pieces, and dweight and dbias add up over them.  The
    reference takes a thousand rows at a time; its bounds for dweight and dbias grow by the
    ratio of the lengths of the sums."""
    import torch

    n, vocab, dim, step = 9000, 131100, 40, 1000
    x, w, b, t, dloss = ce_data(n, vocab, dim, 27, ignored=0.1)
    t[4000:5000] = IGNORE
    got = run_ce(x, w, b, t, dloss)
    abi.check_device_errors(0)
    dw, dw_tol, db, db_tol = (torch.zeros(s, dtype=torch.float64, device=cuda) for s in (w.shape, w.shape, b.shape, b.shape))
    for i in range(0, n, step):
        rows = slice(i, i + step)
        want = ce_reference(x[rows], w, b, t[rows], dloss[rows])
        for name in ("loss", "lse", "dx"):
            within(got[name][rows], want[name][0], want[name][1] + 2.0 ** -40 * dloss.abs().max() * w.double().abs().sum(0) + 1e-42
                   if name == "dx" else want[name][1] + 1e-42, f"{name} of rows {i}")
        dw += want["dw"][0]
        db += want["db"][0]
        # (a gradient's smallest part goes by the largest |dloss| of all rows, not of these)
        dw_tol += want["dw"][1] + 2.0 ** -40 * dloss.abs().max() * x[rows].double().abs().sum(0)
        db_tol += want["db"][1] + 2.0 ** -40 * dloss.abs().max() * step
    longer = (n + 16) / (step + 16)
    within(got["dw"], dw, dw_tol * longer, "dw")
    within(got["db"], db, db_tol * longer, "db")


def test_pieces_of_rows_of_unlike_size(cuda):
    """The same in float32 products: a large row in the second piece.  Each chunk's bounds are its
    own, and those of dweight and dbias grow by the ratio of the lengths of the sums."""
    import torch

    n, vocab, dim, step = 9000, 131100, 24, 1000
    x, w, b, t, dloss = ce_data(n, vocab, dim, 40, ignored=0.1)
    t[4000:5000] = IGNORE
    x[6007] *= 1e13
    t[6007] = 77
    got = run_ce(x, w, b, t, dloss)
    abi.check_device_errors(0)
    dw, dw_tol, db, db_tol = (torch.zeros(s, dtype=torch.float64, device=cuda) for s in (w.shape, w.shape, b.shape, b.shape))
    for i in range(0, n, step):
        rows = slice(i, i + step)
        want = {**ce_reference(x[rows], w, b, t[rows], None), **own_bounds(x[rows], w, b, t[rows], dloss[rows])}
        for name in ("loss", "lse", "dx"):
            within(got[name][rows], want[name][0], want[name][1] + 1e-42, f"{name} of rows {i}")
        for total, tol, name in ((dw, dw_tol, "dw"), (db, db_tol, "db")):
            total += want[name][0]
            tol += want[name][1]
    longer = (n + 16) / (step + 16)
    within(got["dw"], dw, dw_tol * longer, "dw")
    within(got["db"], db, db_tol * longer, "db")
    del want
    torch.cuda.empty_cache()


def test_little_memory_makes_smaller_pieces(cuda):
    """Of a workspace of 1.7 GB, 1.2 can be had: the rows go in two pieces instead of one."""
    import torch

    lib = abi.lib()
    x, w, b, t, dloss = ce_data(1500, 131072, 24, 39, ignored=0.1)
    want = ce_reference(x, w, b, t, dloss)
    whole = run_ce(x, w, b, t, dloss)
    torch.cuda.synchronize()
    outs = run_ce(x, w, b, t, dloss)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    abi.check(lib.mtc_pool_trim(0), "trim")
    free = torch.cuda.mem_get_info()[0]
    hold = torch.empty(free - (1200 << 20), dtype=torch.uint8, device=cuda)
    for o in outs.values():
        o.fill_(7.0)
    try:
        abi.linear_cross_entropy_grad(view(x), view(w), view(t), view(dloss), dx=view(outs["dx"]), dweight=view(outs["dw"]),
                                      bias=view(b), dbias=view(outs["db"]), loss=view(outs["loss"]), lse=view(outs["lse"]),
                                      ignore_target=IGNORE)
        torch.cuda.synchronize()
        used, cached = ctypes.c_uint64(), ctypes.c_uint64()
        abi.check(lib.mtc_pool_stats(0, ctypes.byref(used), ctypes.byref(cached)), "pool stats")
        assert 0 < used.value < 1200 << 20  # it did run in less
    finally:
        del hold
        abi.check(lib.mtc_pool_trim(0), "trim")
    abi.check_device_errors(0)
    assert torch.equal(outs["loss"], whole["loss"]) and torch.equal(outs["lse"], whole["lse"])
    for name in ("dx", "dw", "db"):
        within(outs[name], want[name][0], want[name][1] + 1e-42, name)
    del want, whole, outs, x, w, b
    torch.cuda.empty_cache()  # the reference's, for what comes next


def test_linear_cross_entropy_beyond_32_bits(cuda):
    """A weight of 2.2e9 elements: the loss and sampled rows of its gradient against
    float64, on classes at the end of the vocabulary."""
    import torch

    n, vocab, dim = 260, 700000, 3200
    g = torch.Generator(device="cuda").manual_seed(70)
    w = torch.randn(vocab, dim, device=cuda, generator=g).mul_(0.02)
    x = torch.randn(n, dim, device=cuda, generator=g)
    t = torch.randint(vocab - 3000, vocab, (n,), device=cuda, generator=g)
    dloss = torch.full((n,), 1.0 / n, device=cuda)
    loss, dw = torch.empty(n, device=cuda), torch.empty_like(w)
    abi.linear_cross_entropy_grad(view(x), view(w), view(t), view(dloss), dweight=view(dw), loss=view(loss))
    abi.check_device_errors(0)
    z = torch.cat([x.double() @ w[i: i + 50000].double().t() for i in range(0, vocab, 50000)], 1)
    lse = torch.logsumexp(z, 1)
    want = lse - z.gather(1, t.unsqueeze(1)).squeeze(1)
    size = (x.double().abs() @ w[t].double().abs().t()).max() * 1.5  # sums of |x||w| vary little
    bound = 2 * product_bound(dim, size) + (vocab / 256 + 32) * 2 * U + 30 * U
    within(loss, want, torch.full_like(want, float(bound)), "loss")
    rows = torch.cat([t[:20], torch.tensor([0, vocab // 2, vocab - 1], device=cuda)])
    p = torch.exp(z[:, rows] - lse.unsqueeze(1)) - (t.unsqueeze(1) == rows).double()
    ref = (p * dloss.unsqueeze(1).double()).t() @ x.double()
    tol = ((p.abs() * (2 * float(bound) + 16 * U) + 2.0 ** -40) * dloss.unsqueeze(1).double()).t() @ x.double().abs()
    tol = tol + product_bound(n, (p.abs() * dloss.unsqueeze(1).double()).t() @ x.double().abs())
    within(dw[rows], ref, tol, "dw")


# ------------------------------------------------------------------ clipping --

def clip_reference(tensors, max_norm):
    norm = math.sqrt(sum(float(t.double().pow(2).sum()) for t in tensors))
    return norm, (float(np.float32(max_norm)) / norm if norm > float(np.float32(max_norm)) else 1.0)


def assert_clipped(tensors, outs, norm, max_norm):
    import torch

    want_norm, scale = clip_reference(tensors, max_norm)
    assert abs(norm.item() - want_norm) <= 1.01 * U * want_norm + 1e-45
    for t, o in zip(tensors, outs):
        if scale == 1.0:
            assert torch.equal(o, t)
        else:  # the factor's rounding and the product's
            within(o, t.double() * scale, 2.02 * U * (t.double() * scale).abs() + 1.5e-45, "clipped")


CLIP_SIZES = [[1], [3], [4547], [2, 64, 128, 4096, 3, 192], [8192, 8193, 8191, 1], [1] * 130, [0, 5, 0],
              [100003, 17, 65536], [37] * 1500, [3000001, 2500000]]


@pytest.mark.parametrize("sizes", CLIP_SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("over", [0.5, 3.0])
def test_clipping(cuda, sizes, over):
    import torch

    torch.manual_seed(len(sizes))
    store = torch.randn(sum(sizes) + 1, device=cuda)
    tensors = list(store[1:].split(sizes))  # offsets that break the 16-byte alignment
    max_norm = store[1:].double().norm().item() / over
    outs = [torch.full_like(t, 5.0) for t in tensors]
    norm = torch.empty((), device=cuda)
    abi.clip_global_norm([view(t) for t in tensors], max_norm, view(norm), [view(o) for o in outs])
    assert_clipped(tensors, outs, norm, max_norm)
    alone = torch.empty((), device=cuda)
    abi.global_norm([view(t) for t in tensors], view(alone))
    assert torch.equal(alone, norm)
    keep = store.clone()
    abi.clip_global_norm([view(t) for t in tensors], max_norm)  # in place, nothing beside the tensors
    for t, o in zip(tensors, outs):
        assert torch.equal(t, o)
    assert store[0] == keep[0]


def test_clipping_of_views_with_gaps(cuda):
    import torch

    torch.manual_seed(2)
    a = torch.randn(60, 70, device=cuda)
    b = torch.randn(33, 40, device=cuda)
    tensors = [a[:, 3:50], b.t(), a[:, 60], b.new_full((), 2.0)]
    ref = [t.clone() for t in tensors]
    rest = a[:, :3].clone()
    norm = torch.empty(1, device=cuda)
    abi.clip_global_norm([view(t) for t in tensors], 1.5, view(norm))
    assert_clipped(ref, tensors, norm, 1.5)
    assert torch.equal(a[:, :3], rest)
    outs = [torch.zeros(s, device=cuda).t() for s in ((47, 60), (33, 40))]
    abi.clip_global_norm([view(t) for t in ref[:2]], 1.5, view(norm), [view(o) for o in outs])
    assert_clipped(ref[:2], outs, norm, 1.5)


@pytest.mark.parametrize("views, rows", [(3, 700), (4, 700), (60, 700), (200, 3)])
def test_clipping_of_many_views_with_gaps(cuda, views, rows):
    """So many partial sums that they are added before the scaling, and as many as are not."""
    import torch

    torch.manual_seed(views)
    store = torch.randn(views, rows, 512, device=cuda)
    tensors = [s[:, 1:-1] for s in store] + [torch.randn(1000, device=cuda)]
    ref = [t.clone() for t in tensors]
    rest = store[:, :, 0].clone()
    norm, alone = torch.empty(1, device=cuda), torch.empty(1, device=cuda)
    abi.global_norm([view(t) for t in tensors], view(alone))
    for max_norm in (1e30, 2.0):
        abi.clip_global_norm([view(t) for t in tensors], max_norm, view(norm))
        assert torch.equal(alone, norm)
        assert_clipped(ref, tensors, norm, max_norm)
    assert torch.equal(store[:, :, 0], rest)


def test_norms_beyond_the_range_of_float32_squares(cuda):
    import torch

    for s in (1e30, 1e-30, 1e-42):
        t = torch.randn(5000, device=cuda) * s
        norm = torch.empty((), device=cuda)
        o = torch.empty_like(t)
        abi.clip_global_norm([view(t)], s, view(norm), [view(o)])
        assert_clipped([t], [o], norm, s)
    zero = torch.zeros(100, device=cuda)
    abi.clip_global_norm([view(zero)], 0.0, view(norm))
    assert norm == 0 and (zero == 0).all()
    t = torch.randn(100, device=cuda)
    abi.clip_global_norm([view(t)], 0.0, view(norm))
    assert (t == 0).all() and norm > 0
    abi.global_norm([], view(norm))
    assert norm == 0


def test_clipping_non_finite_gradients(cuda):
    import torch

    a, b = torch.ones(5000, device=cuda), torch.ones(70, device=cuda)
    norm = torch.empty((), device=cuda)
    b[3] = float("inf")
    oa, ob = torch.empty_like(a), torch.empty_like(b)
    abi.clip_global_norm([view(a), view(b)], 1.0, view(norm), [view(oa), view(ob)])
    assert norm.isinf() and (oa == 0).all() and ob[3].isnan() and (ob[:3] == 0).all()
    b[3] = float("nan")
    abi.clip_global_norm([view(a), view(b)], 1.0, view(norm), [view(oa), view(ob)])
    assert norm.isnan() and oa.isnan().all() and ob.isnan().all()


# ------------------------------------------------------------------ together --

def training_step(p, tokens, targets, scale, max_norm, stream=None):
    """One step's forward and backward of a tied-weight next-token model: embedding,
    a dense layer, the loss with its gradients, the embedding's gradient added to
    the output layer's, clipping, and plain descent.  Every call is the library's."""
    import torch

    n, (vocab, dim) = tokens.numel(), p["emb"].shape
    dev = p["emb"].device
    h = torch.empty(n, dim, device=dev)
    y, dy, dh = (torch.empty(n, dim, device=dev) for _ in range(3))
    loss = torch.empty(n, device=dev)
    d_emb, d_lin = torch.empty_like(p["emb"]), torch.empty_like(p["lin"])
    dloss = torch.full((1,), 1.0 / n, device=dev).expand(n)
    norm = torch.empty((), device=dev)
    abi.embedding(view(p["emb"]), view(tokens), view(h), scale=scale, stream=stream)
    abi.matmul(view(h), view(p["lin"].t()), view(y), abi.GEMM_SIMT_FFMA, stream=stream)
    abi.linear_cross_entropy_grad(view(y), view(p["emb"]), view(targets), view(dloss), dx=view(dy), dweight=view(d_emb),
                                  loss=view(loss), ignore_target=IGNORE, stream=stream)
    abi.matmul(view(dy.t()), view(h), view(d_lin), abi.GEMM_SIMT_FFMA, stream=stream)
    abi.matmul(view(dy), view(p["lin"]), view(dh), abi.GEMM_SIMT_FFMA, stream=stream)
    abi.embedding_grad(view(dh), view(tokens), view(d_emb), scale=scale, accumulate=True, stream=stream)
    abi.clip_global_norm([view(d_emb), view(d_lin)], max_norm, view(norm), stream=stream)
    return {"loss": loss, "norm": norm, "emb": d_emb, "lin": d_lin}, (h, y, dy, dh, dloss)


def step_data(n, vocab, dim, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    p = {"emb": torch.randn(vocab, dim, device="cuda", generator=g) * 0.3,
         "lin": torch.randn(dim, dim, device="cuda", generator=g) / math.sqrt(dim)}
    tokens = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    targets = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    targets[::5] = IGNORE
    return p, tokens, targets


@pytest.mark.parametrize("n, vocab, dim", [(50, 40, 16), (600, 1100, 64)])
def test_a_training_step_of_all_operators(cuda, n, vocab, dim):
    """The run of them together against autograd in float64."""
    import torch

    p, tokens, targets = step_data(n, vocab, dim, 31)
    got, _ = training_step(p, tokens, targets, 2.0, 0.05)
    abi.check_device_errors(0)
    emb, lin = (p[k].double().requires_grad_() for k in ("emb", "lin"))
    y = (emb[tokens] * 2.0) @ lin.t()
    loss = torch.nn.functional.cross_entropy(y @ emb.t(), targets, ignore_index=IGNORE, reduction="none")
    loss.sum().div(n).backward()
    norm, scale = clip_reference([emb.grad, lin.grad], 0.05)
    assert scale < 1.0
    # four float32 products in a row, each within (K + 16) 2u of its absolute sums; in the 2-norm those
    # sums exceed the result by at most sqrt(K), so 1e-4 covers K <= 1100 with room for the cancellation
    assert (got["loss"].double() - loss.detach()).abs().max() <= 1e-4 * loss.detach().abs().max()
    assert abs(got["norm"].item() - norm) <= 1e-4 * norm
    for k, grad in (("emb", emb.grad), ("lin", lin.grad)):
        assert (got[k].double() - grad * scale).norm() <= 1e-4 * (grad * scale).norm(), k


def test_recorded_steps_replay_with_the_same_bits(cuda):
    """Two recordings of the step with different data, replayed in turn and after
    eager calls that reuse the pool's blocks: each keeps its own workspaces."""
    import torch

    lib = abi.lib()
    stream = torch.cuda.Stream()
    torch.cuda.set_device(0)
    runs = []
    for seed, (n, vocab, dim) in ((41, (300, 900, 64)), (42, (500, 1100, 72))):
        p, tokens, targets = step_data(n, vocab, dim, seed)
        want, _ = training_step(p, tokens, targets, 1.5, 0.05)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            training_step(p, tokens, targets, 1.5, 0.05)
            torch.cuda.synchronize()
            bufs = None
            abi.check(lib.mtc_capture_begin(0, ctypes.c_void_p(stream.cuda_stream)), "capture")
            # dloss is filled by torch while recording on another stream would not be part of the
            # recording: training_step allocates and fills on the current stream, which is captured
            bufs = training_step(p, tokens, targets, 1.5, 0.05)
            g = ctypes.c_void_p()
            abi.check(lib.mtc_capture_end(1, ctypes.byref(g)), "capture end")
        runs.append((g, bufs, want, (p, tokens, targets)))
    for _ in range(3):
        for g, bufs, want, args in runs:
            for o in bufs[0].values():
                o.fill_(-9.0)
            torch.cuda.synchronize()
            abi.check(lib.mtc_graph_launch(g), "replay")
            training_step(*args, 1.5, 0.05)  # eager calls on another stream meanwhile
            torch.cuda.synchronize()
            for k in want:
                assert torch.equal(bufs[0][k], want[k]), k
    for g, *_ in runs:
        abi.check(lib.mtc_graph_destroy(g), "destroy")


def test_a_foreign_capture_is_refused(cuda):
    """On a stream that another framework records, a call that needs a workspace says
    so; the embedding lookup needs none and is recorded."""
    import torch

    x, w, b, t, dloss = ce_data(20, 30, 8, 50)
    loss = torch.empty(20, device=cuda)
    grad, out = torch.empty(30, 8, device=cuda), torch.empty(20, 8, device=cuda)
    norm = torch.empty((), device=cuda)
    run_ce(x, w, b, t, dloss)
    abi.embedding(view(w), view(t), view(out))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    views = [view(v) for v in (x, w, t, loss, grad, out, norm)]
    dl = view(dloss)
    many, repeated = view(x.repeat(20, 1)), view(t.repeat(20))  # few positions need no workspace
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, capture_error_mode="relaxed"):
        for call in (lambda: abi.linear_cross_entropy_grad(views[0], views[1], views[2], dl, dweight=views[4]),
                     lambda: abi.embedding_grad(many, repeated, views[4]),
                     lambda: abi.global_norm([views[1]], views[6]),
                     lambda: abi.clip_global_norm([views[1]], 1.0)):
            with pytest.raises(abi.MtcError, match="mtc_capture_begin"):
                call()
        abi.embedding(views[1], views[2], views[5], scale=3.0)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, w[t] * 3.0)


def test_two_streams_at_once(cuda):
    """Calls that overlap on two streams have workspaces of their own."""
    import torch

    data = [ce_data(700, 1500, 96, s, ignored=0.1) for s in (60, 61)]
    want = [run_ce(*d) for d in data]
    emb = [(torch.randn(9000, 64, device=cuda), make_tokens(9000, 500, s)) for s in (1, 2)]
    want_e = []
    for d, t in emb:
        g = torch.empty(500, 64, device=cuda)
        abi.embedding_grad(view(d), view(t), view(g))
        want_e.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got, got_e = [None, None], [None, None]
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = run_ce(*data[k])
                got_e[k] = torch.empty(500, 64, device=cuda)
                abi.embedding_grad(view(emb[k][0]), view(emb[k][1]), view(got_e[k]))
                abi.clip_global_norm([view(got[k]["dw"])], 1e30)
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(got_e[k], want_e[k])
            for name in want[k]:
                assert torch.equal(got[k][name], want[k][name]), name


def test_the_default_stream_and_another_at_once(cuda):
    """A call on the default stream and one on a stream that does not wait for it."""
    import torch

    data = [ce_data(900, 2100, 160, s, ignored=0.1) for s in (62, 63)]
    want = [run_ce(*d) for d in data]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for _ in range(8):
        got = [run_ce(*data[0])]
        with torch.cuda.stream(stream):
            got.append(run_ce(*data[1]))
        got.append(run_ce(*data[0]))
        torch.cuda.synchronize()
        for k, g in enumerate(got):
            for name in g:
                assert torch.equal(g[name], want[k % 2][name]), name


def test_a_recorded_call_follows_its_operands(cuda):
    """What the call finds out about its operands it finds out again at every replay: rows of like
    and of unlike size, a scale that the sample of the rows misses, rows without a loss."""
    import torch

    lib = abi.lib()
    n, vocab, dim = 1500, 2300, 96
    x, w, b, t, dloss = ce_data(n, vocab, dim, 64, ignored=0.1)
    variants = [(x, w, t)]
    big = x.clone()
    big[5] *= 1e13
    variants.append((big, w, t))
    missed = x * 1e-3
    missed[1] *= 2e5
    variants.append((missed, w * 0.5, t))
    thin = w.clone()
    thin[:, 7] *= 1e-15
    variants.append((x, thin, torch.where(torch.arange(n, device=cuda) % 3 == 0, t, IGNORE)))
    variants.append((x * 0.0, w, torch.full_like(t, IGNORE)))
    want = [run_ce(xx, ww, b, tt, dloss) for xx, ww, tt in variants]
    xs, ws, ts = x.clone(), w.clone(), t.clone()
    torch.cuda.set_device(0)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run_ce(xs, ws, b, ts, dloss)
        torch.cuda.synchronize()
        abi.check(lib.mtc_capture_begin(0, ctypes.c_void_p(stream.cuda_stream)), "capture")
        got = run_ce(xs, ws, b, ts, dloss)
        g = ctypes.c_void_p()
        abi.check(lib.mtc_capture_end(1, ctypes.byref(g)), "capture end")
    for k in (0, 1, 0, 2, 3, 1, 4, 0):
        for to, source in zip((xs, ws, ts), variants[k]):
            to.copy_(source)
        torch.cuda.synchronize()
        abi.check(lib.mtc_graph_launch(g), "replay")
        torch.cuda.synchronize()
        for name in got:
            assert torch.equal(got[name], want[k][name]), (k, name)
    abi.check_device_errors(0)
    abi.check(lib.mtc_graph_destroy(g), "destroy")
