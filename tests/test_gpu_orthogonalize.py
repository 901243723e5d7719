"""Newton-Schulz products on the GPU against their definition in float64.

U = 2^-24 is half a step of float32.  Two kinds of bounds:

One step, element by element, the worst that roundings can do.  A product of pairs of
16-bit floats is off by at most 2^-22 of each factor and 2^-22 for lo.lo, 12 U, and by its
additions: 48 MMAs a piece of 256 of K, each truncated to a step, two for good measure: 192 U;
pieces, up to 33 here, and the last roundings: 64 U.  Together 268 U of the product of the
magnitudes.  (Small matrices: float32 products, K + 8 <= 268 roundings of U where K <= 260,
K U beyond.)  Through the step: dS = f |X||X|^T, dB = |b| dS + |c| (2 |S| dS + f |S||S|) + 4 U |B|,
dX' = |a| 8 U |X| + dB |X| + f |B||X| + 8 U |X'|, with X itself off by 8 U |X| from its norm.

Several steps, in the Frobenius norm, roundings taken as independent: a product then is off
by 64 U of sqrt(sum a^2 b^2) (an element's 12 U and the truncations' 48 of half a step of the
partial sum at hand), which is at most 64 U |A|_F |B|_2.  The step is a function of X's
singular values alone, p(x) = a x + b x^3 + c x^5, odd, so errors grow by max |p'| over
[-s, s] at most (divided differences of p at x and +-y), s following max |p|.
"""
import ctypes
import math

import pytest
from test_gpu_lm_operators import U, view, within

from minitensor_cpp_b200 import abi

pytestmark = pytest.mark.gpu

EPS = 1e-7
QUINTIC = [abi.QUINTIC] * 5
CUBIC = [(1.5, -0.5, 0.0)] * 4


def f32(x):
    return ctypes.c_float(x).value


def floats(steps):
    return [tuple(f32(v) for v in s) for s in steps]


def matrix(seed, *shape, kind="noise"):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn(*shape, device="cuda", generator=g)
    if kind == "rank":  # a few strong directions over weak noise
        r = min(4, *shape[-2:])
        t = torch.randn(*shape[:-1], r, device="cuda", generator=g) @ torch.randn(*shape[:-2], r, shape[-1], device="cuda",
                                                                                  generator=g) + 1e-3 * t
    if kind == "decay":  # rows from 1 to 2^-20
        rows = torch.linspace(0, -20, shape[-2], device="cuda")
        t = t * torch.exp2(rows).unsqueeze(-1)
    return t * 1e-3


def normalised(t):
    x = t.double()
    norm = x.square().sum(dim=(-1, -2), keepdim=True).sqrt()
    return x / (norm + f32(EPS)).where(norm > 0, 1.0)


def reference(t, steps):
    import torch

    x = normalised(t)
    tall = t.shape[-2] > t.shape[-1]
    x = x.mT if tall else x
    for a, b, c in floats(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


def one_step_bound(t, step):
    x = normalised(t)
    tall = t.shape[-2] > t.shape[-1]
    x = x.mT if tall else x
    (a, b, c), = floats([step])
    f = max(268, x.shape[-1] + 8) * U
    xa = x.abs()
    s = x @ x.mT
    sa = s.abs()
    ds = (f + 16 * U) * (xa @ xa.mT)
    p = b * s + c * (s @ s)
    dp = abs(b) * ds + abs(c) * (2 * (sa @ ds) + f * (sa @ sa)) + 4 * U * p.abs()
    out = a * x + p @ x
    tol = abs(a) * 8 * U * xa + dp @ xa + (f + 8 * U) * (p.abs() @ xa) + 8 * U * out.abs() + 2.0 ** -49
    return (out.mT, tol.mT) if tall else (out, tol)


def norm_bound(t, steps):
    """Of the Frobenius norm of the error of each matrix."""
    import torch

    x = normalised(t)
    x = x.mT if t.shape[-2] > t.shape[-1] else x
    err = 8 * U * torch.ones(x.shape[:-2], dtype=torch.float64, device=x.device)
    s = 1.0
    size = lambda m: m.square().sum(dim=(-1, -2)).sqrt()
    for a, b, c in floats(steps):
        grid = torch.linspace(0, s, 20001, dtype=torch.float64)
        p = b * grid ** 2 + c * grid ** 4
        slope = (a + 3 * b * grid ** 2 + 5 * c * grid ** 4).abs().max().item()
        prod = x @ x.mT
        poly = b * prod + c * (prod @ prod)
        ds = 64 * U * s * size(x)
        dpoly = (abs(b) + 2 * abs(c) * s * s) * ds + 64 * U * (abs(c) * s * s * size(prod) + size(poly))
        new = a * x + poly @ x
        err = slope * err + s * dpoly + 64 * U * (size(poly) * s + abs(a) * size(x) + size(new))
        x, s = new, (grid * (a + p)).abs().max().item()
    return err


def run(ts, steps=QUINTIC, stream=None, eps=EPS):
    import torch

    outs = [torch.full_like(t, 99.0) for t in ts]
    abi.orthogonalize([view(t) for t in ts], [view(t) for t in outs], coefficients=steps, eps=eps, stream=stream)
    return outs


def check(ts, steps=QUINTIC):
    import torch

    got = run(ts, steps)
    abi.check_device_errors(0)
    for t, g in zip(ts, got):
        want = reference(t, steps)
        off = (g.double() - want).square().sum(dim=(-1, -2)).sqrt()
        tol = norm_bound(t, steps)
        assert (off <= tol).all(), f"{tuple(t.shape)}: off by {off.max().item():.3g}, {(off / tol).max().item():.3g} bounds"
    return got


# short and long sides around the four of a small kernel's tile, blocks of 64, tiles of 128 and
# 256, the change of the path, and K of one to several pieces
SHAPES = [(1, 1), (1, 2), (2, 1), (1, 300), (3, 3), (3, 64), (4, 4), (5, 7), (17, 33), (64, 2), (64, 64), (63, 65), (65, 65),
          (61, 200), (10, 2000), (2, 9000), (3, 30000), (100, 100), (96, 130), (127, 127), (128, 128), (129, 129), (128, 64),
          (120, 700), (33, 4097), (1, 60000), (257, 64), (130, 300), (192, 192), (255, 257), (256, 256), (257, 513), (300, 1000),
          (513, 385), (640, 640), (1000, 300), (771, 1031), (1025, 1025), (1500, 333), (2500, 2300), (140, 20000)]


@pytest.mark.parametrize("shape", SHAPES)
def test_one_step_against_float64(cuda, shape):
    for seed, kind in enumerate(("noise", "rank", "decay")):
        t = matrix(seed, *shape, kind=kind)
        got, = run([t], QUINTIC[:1])
        abi.check_device_errors(0)
        want, tol = one_step_bound(t, QUINTIC[0])
        within(got, want, tol, f"{shape}, {kind}")


@pytest.mark.parametrize("shape", SHAPES)
def test_five_steps_against_float64(cuda, shape):
    for seed, kind in enumerate(("noise", "rank", "decay")):
        check([matrix(seed + 10, *shape, kind=kind)])


@pytest.mark.parametrize("shape", [(40, 50), (300, 200), (130, 600)])
def test_other_coefficients(cuda, shape):
    t = matrix(3, *shape)
    for steps in (CUBIC, [(1.0, 0.0, 0.0)] * 3, [(0.5, 0.25, 0.0)], [(2.0, -1.5, 0.5), (1.875, -1.25, 0.375)] * 2,
                  [(3.0, 0.0, 1.0)] * 2, [(0.0, 1.0, 0.0)], [(0.0, 0.0, 1.0)], [(-1.0, 0.0, 0.0)], [(64.0, 0.0, 0.0)],
                  [(2.0 ** -10, 0.0, 2.0 ** -30)] * 4, [(0.0, 0.0, 0.0)], [(1.5, -0.5, 0.0)] * 32):
        check([t], steps)


def test_singular_values_come_close_to_one(cuda):
    """Those above 0.01 of the largest end in [0.65, 1.25], and the singular vectors stay."""
    import torch

    for shape in ((48, 64), (200, 333), (512, 300)):
        t = matrix(4, *shape).double()
        u, s, v = torch.linalg.svd(t, full_matrices=False)
        s = torch.logspace(0, -1, s.numel(), dtype=torch.float64, device=cuda)
        t = ((u * s) @ v).float()
        got = check([t])[0].double()
        inner = u.mT @ got @ v.mT
        values = inner.diagonal()
        assert values.min() > 0.65 and values.max() < 1.25
        assert (inner - values.diag()).abs().max() < 1e-3


def test_lists_of_many_sizes(cuda):
    """Small and large ones, batches, in one call: each as if alone within its bounds."""
    ts = [matrix(i, *s) for i, s in enumerate([(64, 2), (64, 64), (3, 64), (5, 300, 200), (2, 3, 40, 50), (1000, 77),
                                              (300, 300), (4, 100, 120), (1, 1), (7, 0), (0, 3, 3), (3, 129, 5), (600, 900)])]
    check(ts)


@pytest.mark.parametrize("shape, count", [((3, 5), 300), ((100, 90), 140), ((130, 150), 131)])
def test_more_matrices_than_a_launch_takes(cuda, shape, count):
    check([matrix(5, count, *shape)])
    check([t for t in matrix(6, count, *shape)])


def test_views(cuda):
    """Transposed, with gaps, reversed order of axes, broadcast, offsets without alignment; in and out."""
    import torch

    for r, c in ((40, 50), (50, 41), (129, 300), (300, 131), (64, 700)):
        t = matrix(7, r, c)
        want = run([t])[0]
        held = torch.zeros(2 * r + 1, 3 * c + 2, device=cuda)
        for part in (held[1:2 * r:2, 2:2 + 3 * c:3], held[:r, 1:1 + c], held.view(-1)[3:3 + r * c].view(c, r).t()):
            part.copy_(t)
            got = torch.zeros_like(t)
            abi.orthogonalize([view(part)], [view(got)])
            assert torch.equal(got, want)
            held.fill_(7.0)
            abi.orthogonalize([view(t)], [view(part)])
            assert torch.equal(part, want)
            part.fill_(7.0)
            assert (held == 7).all()
        one = matrix(8, 1, c).expand(r, c)  # one row for all: rank one
        check([one])
        b = matrix(9, c, 3, r)
        check([b.permute(1, 2, 0), b.permute(1, 0, 2)])


def test_in_place(cuda):
    import torch

    ts = [matrix(i, *s) for i, s in enumerate([(64, 64), (5, 30, 20), (300, 200), (2, 130, 140), (90, 4000)])]
    want = run(ts)
    abi.orthogonalize([view(t) for t in ts])
    for t, w in zip(ts, want):
        assert torch.equal(t, w)


@pytest.mark.parametrize("shape", [(5, 7), (60, 64), (200, 300), (100, 2000), (600, 520)])
def test_zeros_infinities_and_nan_stay_in_their_matrices(cuda, shape):
    import torch

    ts = matrix(10, 6, *shape)
    ts[1] = 0.0
    ts[2, 0, 1], ts[3, -1, -1], ts[4, 1, 0] = float("nan"), math.inf, -math.inf
    for eps in (0.0, EPS):
        got, = run([ts], eps=eps)
        abi.check_device_errors(0)
        assert (got[1] == 0).all() and got[2:5].isnan().all() and got[[0, 5]].isfinite().all()
    fine = ts[[0, 5]].contiguous()
    assert ((got[[0, 5]].double() - reference(fine, QUINTIC)).square().sum(dim=(1, 2)).sqrt() <= norm_bound(fine, QUINTIC)).all()


@pytest.mark.parametrize("shape", [(30, 40), (200, 300)])
def test_sizes_of_elements_do_not_matter(cuda, shape):
    """From the smallest float32 numbers to the largest; eps counts beside small norms."""
    import torch

    t = matrix(11, *shape)
    want = run([t], eps=0.0)[0]
    for e in (-40, -100, 100, 120):  # exact scaling
        got = run([t * 2.0 ** e], eps=0.0)[0]
        assert torch.equal(got, want), e
    tiny = (t / t.abs().max() * 1e-42)  # subnormal, of few digits: as they are
    exact = tiny.double() * 2.0 ** 200
    got = run([tiny], eps=0.0)[0].double()
    assert ((got - reference((exact / exact.abs().max()).float(), QUINTIC)).norm() <= 2 * norm_bound(exact, QUINTIC)).all()
    got = run([t], QUINTIC[:1], eps=1.0)[0].double()
    x = t.double() / (t.double().norm() + 1.0)
    a, b, c = floats(QUINTIC)[0]
    x = x if shape[0] <= shape[1] else x.mT
    want = a * x + (b * x @ x.mT + c * x @ x.mT @ x @ x.mT) @ x
    within(got, want, 300 * U * want.abs() + 1e-9, "eps")


def test_a_large_matrix(cuda):
    """Tiles of several bands, and positions behind 2^31 bytes."""
    import torch

    t = matrix(12, 9000, 9300)
    got, = run([t], CUBIC[:2])
    abi.check_device_errors(0)
    want = reference(t, CUBIC[:2])
    assert (got.double() - want).norm() <= norm_bound(t, CUBIC[:2])


def test_more_than_one_group(cuda):
    """Five matrices whose packed operands take more than is taken at a time; one input may come again."""
    import torch

    t = matrix(27, 8192, 8200)
    steps = CUBIC[:1]
    outs = [torch.full_like(t, 99.0) for _ in range(5)]
    abi.orthogonalize([view(t)] * 5, [view(o) for o in outs], coefficients=steps)
    abi.check_device_errors(0)
    want, tol = reference(t, steps), norm_bound(t, steps)
    assert all((o.double() - want).norm() <= tol for o in outs)


def test_paths_agree_where_they_meet(cuda):
    """The sizes on both sides of each change of the path, in one list and alone."""
    for shape in ((59, 61), (61, 61), (62, 62), (128, 128), (128, 129), (127, 300), (129, 129), (64, 300), (64, 330), (5, 5000)):
        t = matrix(28, *shape)
        check([t])
        check([t, matrix(29, 60, 60), matrix(30, 100, 90), matrix(31, 300, 280)])


def test_elements_behind_32_bits(cuda):
    """A batch whose last matrices lie behind 2^31 elements."""
    import torch

    ts = torch.zeros(2200, 1000, 1000, device=cuda)[:, :150, :170]
    ts[0], ts[2199] = matrix(13, 150, 170), matrix(14, 150, 170)
    abi.orthogonalize([view(ts)])
    assert torch.equal(ts[2199], run([matrix(14, 150, 170)])[0]) or \
        (ts[2199].double() - reference(matrix(14, 150, 170), QUINTIC)).norm() <= norm_bound(matrix(14, 150, 170), QUINTIC)
    assert not ts[1:2199].any()


def test_recorded_and_replayed_next_to_eager_calls(cuda):
    """Two graphs, with workspaces of their own, and eager calls on another stream at once."""
    import torch

    st = ctypes.c_void_p()
    abi.check(abi.lib().mtc_stream_create(0, ctypes.byref(st)))
    ts = [matrix(15, 300, 200), matrix(16, 40, 50), matrix(17, 90, 900)]
    outs = [[torch.zeros_like(t) for t in ts] for _ in range(2)]
    graphs = []
    run(ts)
    torch.cuda.synchronize()
    for out in outs:
        abi.check(abi.lib().mtc_capture_begin(0, st))
        abi.orthogonalize([view(t) for t in ts], [view(t) for t in out], stream=st.value)
        graph = ctypes.c_void_p()
        abi.check(abi.lib().mtc_capture_end(1, ctypes.byref(graph)))
        graphs.append(graph)
    for seed in (20, 30):
        for i, t in enumerate(ts):
            t.copy_(matrix(seed + i, *t.shape))
        for out in outs:
            for t in out:
                t.fill_(5.0)
        torch.cuda.synchronize()
        for graph in graphs:
            abi.check(abi.lib().mtc_graph_launch(graph))
        want = [run(ts) for _ in range(3)][-1]  # meanwhile
        abi.check(abi.lib().mtc_stream_synchronize(st))
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    for graph in graphs:
        abi.check(abi.lib().mtc_graph_destroy(graph))
    abi.check(abi.lib().mtc_stream_destroy(0, st))


def test_a_stream_that_torch_captures_is_refused(cuda):
    """The pool would hand the workspace on while the graph replays; a call of small matrices has none."""
    import torch

    t, small = matrix(18, 300, 200), matrix(19, 30, 20)
    out, want = torch.zeros_like(small), run([small])[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        abi.orthogonalize([view(small)], [view(out)])
        with pytest.raises(abi.MtcError, match="workspace"):
            abi.orthogonalize([view(t)])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_two_streams_at_once(cuda):
    import torch

    ts = [matrix(21, 700, 500), matrix(22, 260, 900)]
    want = [run([t])[0] for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    outs = [[torch.zeros_like(t) for _ in range(6)] for t in ts]
    torch.cuda.synchronize()
    for i in range(6):
        for t, s, o in zip(ts, streams, outs):
            abi.orthogonalize([view(t)], [view(o[i])], stream=s.cuda_stream)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(x, w) for x in o)


def test_the_same_inputs_give_the_same_bits(cuda):
    import torch

    ts = [matrix(23, 500, 1300), matrix(24, 60, 60), matrix(25, 3, 140, 150)]
    first = run(ts)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(run(ts), first))


def test_a_training_step(cuda):
    """Sampled answers scored, their loss's gradient, the update of the output layer: the operators in a row."""
    import torch

    n, vocab, dim, beta, lr = 400, 1500, 200, 0.01, 0.1
    g = torch.Generator(device="cuda").manual_seed(26)
    rnd = lambda *s: torch.randn(*s, device=cuda, generator=g)
    x, w, advantage = rnd(n, dim), rnd(vocab, dim) * 0.05, rnd(n)
    tokens = torch.randint(0, vocab, (n,), device=cuda, generator=g)
    tokens[::9] = -100
    live = tokens != -100
    count = int(live.sum())
    V = view
    z, logp, entropy = torch.empty(n, vocab, device=cuda), torch.empty(n, device=cuda), torch.empty(n, device=cuda)
    abi.matmul(V(x), V(w.t()), V(z))
    abi.token_log_probs(V(z), tokens=V(tokens), log_probs=V(logp), entropy=V(entropy), ignore_token=-100)
    dlp, dent = -advantage / count, torch.full((1,), -beta / count, device=cuda).expand(n)
    abi.token_log_probs_grad(V(z), V(z), tokens=V(tokens), dlog_probs=V(dlp), dentropy=V(dent), ignore_token=-100)
    dw, norm = torch.empty_like(w), torch.empty((), device=cuda)
    abi.matmul(V(z.t()), V(x), V(dw))
    abi.clip_global_norm([V(dw)], 1e-3, V(norm))
    update = torch.empty_like(w)
    abi.orthogonalize([V(dw)], [V(update)])
    new = w - lr * update
    abi.check_device_errors(0)

    wd = w.double().requires_grad_()
    at = torch.where(live, tokens, 0).unsqueeze(1)
    lp = torch.log_softmax(x.double() @ wd.t(), 1)
    h = -(lp.exp() * lp).sum(1)
    picked = lp.gather(1, at).squeeze(1)
    loss = -((advantage.double() * picked + beta * h) * live).sum() / count
    grad, = torch.autograd.grad(loss, wd)
    within(torch.where(live, logp, 0.0), (picked * live).detach(), 1e-5 * torch.ones(n, device=cuda), "log probabilities")
    within(entropy, (h * live).detach(), 1e-5 * torch.ones(n, device=cuda), "entropy")
    assert abs(norm.item() - grad.norm().item()) <= 1e-5 * grad.norm().item()
    clipped = grad * (1e-3 / grad.norm())
    assert (dw.double() - clipped).norm() <= 1e-5 * clipped.norm()
    want = w.double() - lr * reference(dw, QUINTIC)
    assert (new.double() - want).norm() <= lr * norm_bound(dw, QUINTIC) + 2 * U * want.norm()
    # the loss falls along the update at the rate that the gradient says
    step = reference(dw, QUINTIC)
    lp2 = torch.log_softmax(x.double() @ (w.double() - 1e-4 * step).t(), 1)
    h2 = -(lp2.exp() * lp2).sum(1)
    loss2 = -((advantage.double() * lp2.gather(1, at).squeeze(1) + beta * h2) * live).sum() / count
    assert (loss2 - loss).item() < 0


# of up to 64 rows: from one CTA's columns to a cluster's of eight, and beyond them; parts of the
# columns that are empty, of no whole four, and one column more than a part
FEW_ROWS = [(1, 129), (1, 13300), (1, 13301), (1, 106390), (1, 106500), (2, 50001), (4, 26600), (5, 8190), (7, 141), (8, 6003),
            (12, 8192), (16, 26007), (29, 4001), (32, 12161), (33, 3000), (48, 1031), (60, 2000), (61, 129), (64, 129), (64, 300),
            (64, 1027), (64, 4281), (64, 4400), (65, 1027)]


@pytest.mark.parametrize("shape", FEW_ROWS)
def test_few_rows(cuda, shape):
    """Alone, where CTAs are left over, and in batches; transposed and in place."""
    import torch

    for seed, kind in enumerate(("noise", "rank", "decay")):
        t = matrix(seed + 40, *shape, kind=kind)
        got, = run([t], QUINTIC[:1])
        abi.check_device_errors(0)
        want, tol = one_step_bound(t, QUINTIC[0])
        within(got, want, tol, f"{shape}, {kind}")
        check([t])
    ts = matrix(43, 40, *shape)
    got, = check([ts])
    check([ts.mT, matrix(44, 50, 60), matrix(45, 3, shape[0], 200)])
    abi.orthogonalize([view(ts)])
    assert torch.equal(ts, got)


def test_few_rows_that_hold_no_numbers(cuda):
    """In one CTA's part of the columns only: NaN all over that matrix, and there alone."""
    import torch

    ts = matrix(46, 5, 6, 30000)
    ts[1] = 0.0
    ts[2, 5, 29999], ts[3, 0, 15000] = float("nan"), -math.inf
    for eps in (0.0, EPS):
        got, = run([ts], eps=eps)
        abi.check_device_errors(0)
        assert (got[1] == 0).all() and got[2:4].isnan().all() and got[[0, 4]].isfinite().all()


def test_few_rows_recorded(cuda):
    """Clusters of several sizes in a graph of torch's (no workspace), replayed over new inputs beside eager calls."""
    import torch

    shapes = [(10, 3000), (3, 8192), (4, 33, 2000), (60, 1500), (20, 20)]
    ts, side = [matrix(50 + i, *s) for i, s in enumerate(shapes)], torch.cuda.Stream()
    outs = [torch.zeros_like(t) for t in ts]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        abi.orthogonalize([view(t) for t in ts], [view(o) for o in outs])
    for seed in (60, 70):
        for i, t in enumerate(ts):
            t.copy_(matrix(seed + i, *t.shape))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        want = [run(ts) for _ in range(3)][-1]  # meanwhile
        torch.cuda.synchronize()
        for t, o, w in zip(ts, outs, want):
            assert torch.equal(o, w)
        check(ts)


@pytest.mark.parametrize("shape", [(30, 40), (100, 100), (90, 128), (120, 700), (300, 200)])
def test_coefficients_at_their_limit(cuda, shape):
    """Singular values at 2^20 before a step, with polynomials of nothing, of little and of much: on each path."""
    t = matrix(80, *shape)
    for steps in ([(2.0 ** 20, 0.0, 0.0), (0.5, 0.0, 0.0)], [(2.0 ** 20, 0.0, 0.0), (0.0, 0.0, 0.0)],
                  [(2.0 ** 20, 0.0, 0.0), (1.0, -(2.0 ** -41), 0.0)], [(2.0 ** 20, 0.0, 0.0), (0.5, 0.0, 2.0 ** -82)],
                  [(0.0, 2.0 ** 20, 0.0), (2.0 ** -20, 0.0, 0.0)], [(2.0 ** 10, 0.0, 0.0), (2.0 ** 10, 0.0, 0.0), (-1.0, 0.0, 0.0)]):
        got, = check([t], steps)
        assert got.isfinite().all(), steps


@pytest.mark.parametrize("shape", [(30, 40), (100, 100), (90, 128), (120, 700), (300, 200)])
def test_coefficients_that_shrink_up_to_their_limit(cuda, shape):
    t = matrix(81, *shape)
    for steps in ([(2.0 ** -60, 0.0, 0.0)], [(2.0 ** -30, 0.0, 0.0), (1.0, 2.0 ** 60, 0.0)], [(2.0 ** -59, -(2.0 ** -60), 0.0)],
                  [(2.0 ** -30, 0.0, 0.0), (0.0, 2.0 ** 60, 2.0 ** 119)], [(2.0 ** -40, 0.0, 0.0), (2.0 ** 40, 0.0, 0.0)],
                  [(0.0, 0.0, 0.0), (1.0, 1.0, 1.0)]):
        check([t], steps)


def test_operands_behind_2_31_bytes(cuda):
    """A matrix whose packed operands take 2.7 GB, and one of odd sizes that has all of its own behind them."""
    big, odd = matrix(82, 13000, 13100), matrix(83, 601, 707)
    check([big, odd], CUBIC[:3])
    check([odd], CUBIC[:3])
