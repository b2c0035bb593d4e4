"""The output layer with its loss (linear_softmax_cross_entropy), the orthogonalised update (newton_schulz, muon_step_multi)
and the host layer's forms of them, against their definitions in 64 bits.

Bars. A float32-accurate product's element is held to 1e-5 * |a_row| * |b_col|, the bar of every product in this library.
Logits off by ez change a probability p by at most p * (exp(2 ez) - 1), plus 2^-20 p for exponential, sum and quotient; the
gradients' bars follow from that bound through their own products. The gradients' products take softmax - one-hot, times 2^15, as
two float16 numbers, whose smallest spacing is 2^-24: an element is off by 2^-22 of itself or by half a spacing, 2^-25 / 2^15 =
2^-40, whichever is more. Newton-Schulz: one step changes X by products whose
operands (22 bits kept of each) and sums err by 3 * 2^-22 relative to the Frobenius norms of its terms, (|a| + |b| + |c|) of
them; five steps pass an error on by at most 3.4445 a step; X is kept times 2^13, so an element is off by 2^-25 / 2^13 = 2^-38 at least."""
import ctypes
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
IGNORE = -100


@pytest.fixture(scope="module")
def capi():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from origindl_amd import capi
    return capi


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(N, K, V, out_in, bias, ignored, i64, seed, spread=1.5):
    g = gen(seed)
    x = torch.randn(N, K, device="cuda", generator=g)
    w = torch.randn((V, K) if out_in else (K, V), device="cuda", generator=g) * (spread / math.sqrt(K))
    b = torch.randn(V, device="cuda", generator=g) if bias else None
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    t[torch.rand(N, device="cuda", generator=g) < ignored] = IGNORE
    return x, w, b, t if i64 else t.int()


def definition(x, w, b, t, out_in, gy=1.0, ignore=IGNORE):
    """loss, gx, gw, gb and the bars of the last three and of the loss, in float64."""
    keep = (t.long() != ignore).nonzero()[:, 0]
    W = (w if out_in else w.t()).double()                       # [V, K]
    X, label = x[keep].double(), t.long()[keep]
    C = max(1, len(keep))
    z = torch.mm(X, W.t())
    if b is not None:
        z = z + b.double()
    lse = torch.logsumexp(z, dim=1) if len(keep) else z.new_zeros(0)
    loss = (lse - z.gather(1, label[:, None])[:, 0]).sum() / C
    p = torch.exp(z - lse[:, None])
    d = p.clone()
    d[torch.arange(len(keep), device=x.device), label] -= 1
    xn, wn = X.norm(dim=1), W.norm(dim=1)
    ez = 1e-5 * xn * wn.max()                                    # [n]
    dd = p * (torch.expm1(2 * ez) + 2.0 ** -20)[:, None] + 2.0 ** -23 * d.abs()
    f = abs(gy) / C
    gx, gw, gb = torch.zeros_like(x, dtype=torch.float64), torch.mm(d.t(), X) * (gy / C), d.sum(0) * (gy / C)
    gx[keep] = torch.mm(d, W) * (gy / C)
    tx = torch.full_like(gx, 1e-30)
    tx[keep] += f * (torch.mm(dd + 2.0 ** -40, W.abs()) + 1e-5 * d.norm(dim=1)[:, None] * W.norm(dim=0)[None, :])
    dd = dd + 2.0 ** -40
    tw = f * (torch.mm(dd.t(), X.abs()) + 1e-5 * d.norm(dim=0)[:, None] * X.norm(dim=0)[None, :]) + 1e-30
    tb = f * (dd.sum(0) + 2.0 ** -22 * d.abs().sum(0)) + 1e-30
    if not out_in:
        gw, tw = gw.t(), tw.t()
    tl = float((2 * ez).max() if len(keep) else 0) + 2.0 ** -20 * (1 + float(lse.abs().max() if len(keep) else 0))
    return (loss, gx, gw, gb), (tl, tx, tw, tb)


def run(capi, x, w, b, t, out_in, gy=None, **kw):
    loss, saved = capi.linear_softmax_cross_entropy(x, w, b, t, w_out_in=out_in, **kw)
    grads = capi.linear_softmax_cross_entropy_backward(gy, x, w, b, t, saved, w_out_in=out_in, **kw)
    return (loss,) + grads, saved


def check(got, want, bars):
    assert abs(float(got[0]) - float(want[0])) <= bars[0], (float(got[0]), float(want[0]), bars[0])
    for name, a, e, tol in zip(("gx", "gw", "gb"), got[1:], want[1:], bars[1:]):
        if a is not None:
            off = (a.double() - e).abs()
            assert bool((off <= tol).all()), (name, float((off / tol).max()))


# one token to many, one feature, one class, sizes around every tile (64, 128, 256) and its half, and several pieces
CE_SHAPES = [(1, 1, 1), (1, 64, 1000), (2, 3, 5), (3, 17, 64), (5, 33, 65), (16, 100, 130), (31, 257, 511), (64, 128, 256), (65, 96, 97),
             (96, 769, 300), (128, 64, 1025), (200, 768, 2000), (257, 130, 769), (770, 100, 3001), (1025, 300, 1100), (33, 40, 129), (1, 4097, 3), (8, 5, 6000),
             # few rows over large weights stream them: ends of the vocabulary and of K off every step, 32 rows to 256
             (1, 64, 100000), (7, 129, 50003), (32, 2050, 3001), (33, 2047, 3002), (64, 100, 60004), (5, 1000003, 6), (64, 2000, 4001), (65, 300, 30001), (128, 1031, 6002),
             (129, 64, 100003), (200, 2000, 3500), (256, 515, 12007), (3, 2, 3000001), (70, 1, 6000001)]


@pytest.mark.parametrize("shape", CE_SHAPES)
@pytest.mark.parametrize("out_in", [False, True])
def test_loss_and_gradients(capi, shape, out_in):
    N, K, V = shape
    for bias, ignored, i64 in ((True, 0.0, True), (False, 0.3, False)):
        x, w, b, t = make(N, K, V, out_in, bias, ignored, i64, seed=N + K + V)
        gy = torch.tensor(-0.75, device="cuda")
        got, saved = run(capi, x, w, b, t, out_in, gy)
        want, bars = definition(x, w, b, t, out_in, -0.75)
        check(got, want, bars)
        assert float(saved[0][2]) == float((t != IGNORE).sum())
        assert not capi.linear_softmax_cross_entropy_bad_label(saved)


@pytest.mark.parametrize("shape", [(300, 1025, 70000), (2050, 64, 40000)])
def test_a_vocabulary_in_several_pieces(capi, shape):
    """Pieces of the vocabulary: the last one is shorter, gx is added up over them, gw and gb are written piece by piece."""
    N, K, V = shape
    for out_in in (False, True):
        x, w, b, t = make(N, K, V, out_in, True, 0.1, True, seed=7)
        got, _ = run(capi, x, w, b, t, out_in)
        check(got, *definition(x, w, b, t, out_in))


def test_rows_that_do_not_count_may_hold_anything(capi):
    for N, K, V in ((7, 40, 90), (130, 200, 700), (9, 200, 31000)):
        x, w, b, t = make(N, K, V, False, True, 0.4, True, seed=3)
        t[2], t[5] = IGNORE, IGNORE
        want, bars = definition(x, w, b, t, False)
        bad = x.clone()
        out = (t == IGNORE).nonzero()[:, 0]
        assert len(out) >= 2
        bad[out] = float("nan")
        bad[out[0]] = float("inf")
        bad[out[1]] = 3e38
        got, _ = run(capi, bad, w, b, t, False)
        check(got, want, bars)
        assert bool((got[1][out] == 0).all())


def test_no_row_counts_and_no_rows(capi):
    x, w, b, t = make(9, 20, 50, False, True, 0.0, True, seed=4)
    t[:] = IGNORE
    x[3] = float("nan")
    got, saved = run(capi, x, w, b, t, False)
    assert float(got[0]) == 0 and all(bool((g == 0).all()) for g in got[1:]) and float(saved[0][2]) == 0
    got, saved = run(capi, x[:0].contiguous(), w, b, t[:0].contiguous(), False)
    assert float(got[0]) == 0 and got[1].shape == (0, 20) and bool((got[2] == 0).all()) and bool((got[3] == 0).all())
    assert not capi.linear_softmax_cross_entropy_bad_label(saved)


@pytest.mark.parametrize("K", [30, 110000])
def test_another_ignore_index_and_labels_out_of_range(capi, K):
    x, w, b, t = make(40, K, 60, True, True, 0.0, True, seed=5)
    t[::3] = 7
    got, saved = run(capi, x, w, b, t, True, ignore_index=7)
    check(got, *definition(x, w, b, t, True, ignore=7))
    assert not capi.linear_softmax_cross_entropy_bad_label(saved)
    # a label out of range is flagged, and its row is left out as an ignored one is
    for label in (60, -1, 1 << 40):
        t2 = t.clone()
        t2[1] = label
        got, saved = run(capi, x, w, b, t2, True, ignore_index=7)
        assert capi.linear_softmax_cross_entropy_bad_label(saved)
        t3 = t.clone()
        t3[1] = 7
        check(got, *definition(x, w, b, t3, True, ignore=7))


@pytest.mark.parametrize("K", [48, 10000])
def test_entries_masked_by_the_bias(capi, K):
    """-inf and the type's lowest value in the bias: probability 0, no gradient; a whole tile of them; a label among them."""
    N, V = 33, 700
    x, w, b, t = make(N, K, V, False, True, 0.0, True, seed=6)
    t = t % 100
    b[100:640] = -float("inf")
    b[650:660] = torch.finfo(torch.float32).min
    got, _ = run(capi, x, w, b, t, False)
    want, bars = definition(x, w, torch.where(b < -1e30, torch.full_like(b, -1e30), b), t, False)
    check(got, want, bars)
    masked = b < -1e30
    assert bool((got[3][masked] == 0).all()) and bool((got[2][:, masked] == 0).all())
    t[5] = 120
    loss, _ = capi.linear_softmax_cross_entropy(x, w, b, t)
    assert float(loss) == float("inf")


@pytest.mark.parametrize("K", [64, 11000])
def test_nan_in_a_counted_row_or_weight_reaches_the_loss(capi, K):
    x, w, b, t = make(20, K, 600, True, False, 0.0, True, seed=8)
    bad = x.clone()
    bad[4, 3] = float("nan")
    assert math.isnan(float(capi.linear_softmax_cross_entropy(bad, w, b, t, w_out_in=True)[0]))
    bad = w.clone()
    bad[128:400] = float("nan")
    t = t % 100
    assert math.isnan(float(capi.linear_softmax_cross_entropy(x, bad, b, t, w_out_in=True)[0]))


@pytest.mark.parametrize("sx,sw", [(1e20, 1e-20), (1e-18, 1e18), (1e-38, 1.0), (1e-30, 1e-30), (0.0, 1.0), (1.0, 0.0)])
def test_magnitudes_far_from_one(capi, sx, sw):
    """Operands are scaled by powers of two of their own: nothing over- or underflows on the way to a logit of ordinary size."""
    for K in (70, 31000):
        x, w, b, t = make(50, K, 200, False, True, 0.0, True, seed=9)
        x, w = x * sx, w * sw
        got, _ = run(capi, x, w, b, t, False)
        check(got, *definition(x, w, b, t, False))


def test_confident_logits(capi):
    """Logits of a trained model: probabilities next to 1, others far under the smallest float16."""
    x, w, b, t = make(100, 256, 1000, False, False, 0.0, True, seed=10, spread=12.0)
    t = (x @ w).argmax(dim=1)
    got, _ = run(capi, x, w, b, t, False)
    check(got, *definition(x, w, b, t, False))


@pytest.mark.parametrize("K", [130, 7000])
def test_any_subset_of_the_gradients_has_the_same_bits(capi, K):
    x, w, b, t = make(150, K, 900, False, True, 0.2, True, seed=11)
    _, saved = capi.linear_softmax_cross_entropy(x, w, b, t)
    whole = capi.linear_softmax_cross_entropy_backward(None, x, w, b, t, saved)
    for mask in range(8):
        need = [bool(mask & (1 << i)) for i in range(3)]
        part = capi.linear_softmax_cross_entropy_backward(None, x, w, b, t, saved, need_gx=need[0], need_gw=need[1], need_gb=need[2])
        for want, g, p in zip(need, whole, part):
            assert (p is None) == (not want) and (p is None or torch.equal(p, g))


def test_gradient_against_differences_of_the_loss(capi):
    """(L(x + h u) - L(x - h u)) / 2h against <gx, u>: a loss rounds by 2^-23 L and carries the products' error in its logits
    (1e-5 |x||w| at most, both calls), the third derivative of log-sum-exp along u is at most 2 max|dz|^3."""
    x, w, b, t = make(24, 40, 80, False, True, 0.2, True, seed=12)
    loss, saved = capi.linear_softmax_cross_entropy(x, w, b, t)
    gx, gw, gb = capi.linear_softmax_cross_entropy_backward(None, x, w, b, t, saved)
    g = gen(13)
    h = 2.0 ** -5
    ez = 1e-5 * float(x.norm(dim=1).max() * w.norm(dim=0).max()) * 1.2
    for which, grad in (("x", gx), ("w", gw), ("b", gb)):
        u = torch.randn(grad.shape, device="cuda", generator=g)
        u /= u.norm()
        args = {"x": x, "w": w, "b": b}
        ends = []
        for s in (h, -h):
            moved = dict(args)
            moved[which] = args[which] + s * u
            ends.append(float(capi.linear_softmax_cross_entropy(moved["x"], moved["w"], moved["b"], t)[0]))
        dz = (u.double() @ w.double() if which == "x" else x.double() @ u.double() if which == "w" else u).abs().max()
        tol = (2.0 ** -22 * float(loss) + 4 * ez) / (2 * h) + h * h / 6 * 2 * float(dz) ** 3 + 1e-5
        assert abs((ends[0] - ends[1]) / (2 * h) - float((grad.double() * u.double()).sum())) <= tol


@pytest.mark.parametrize("N,K", [(300, 200), (90, 4000)])
def test_two_calls_give_the_same_bits_and_other_streams_work(capi, N, K):
    x, w, b, t = make(N, K, 2000, True, True, 0.1, True, seed=14)
    first, _ = run(capi, x, w, b, t, True)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for s in (s1, s2):  # two calls under way at once, each with its own workspace
        with torch.cuda.stream(s):
            outs.append(run(capi, x, w, b, t, True)[0])
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, e) for a, e in zip(o, first))


@pytest.mark.parametrize("K,rows,cols", [(96, 96, 200), (5000, 100, 90), (96, 260, 1100)])
def test_recorded_calls_replay(capi, K, rows, cols):
    x, w, b, t = make(200, K, 1500, False, True, 0.1, True, seed=15)
    run(capi, x, w, b, t, False)
    m = torch.randn(rows, cols, device="cuda", generator=gen(16))
    buf = torch.zeros_like(m)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, saved = run(capi, x, w, b, t, False)
        o = capi.newton_schulz(m)
        (p,) = capi.muon_step_multi([m], [o], [buf], lr=0.1)
    ref_buf = torch.zeros_like(m)
    for i in range(3):
        x.copy_(torch.randn(x.shape, device="cuda", generator=gen(17 + i)))
        m.copy_(torch.randn(m.shape, device="cuda", generator=gen(27 + i)))
        graph.replay()
        torch.cuda.synchronize()
        want, _ = run(capi, x, w, b, t, False)
        wo = capi.newton_schulz(m)
        (wp,) = capi.muon_step_multi([m], [wo], [ref_buf], lr=0.1)
        assert all(torch.equal(a, e) for a, e in zip(got, want)), i
        assert torch.equal(o, wo) and torch.equal(p, wp) and torch.equal(buf, ref_buf), i


def test_weights_and_matrices_off_their_alignment(capi):
    """Dense tensors that start in the middle of a buffer, on 4 bytes."""
    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        return buf[1:].view(t.shape).copy_(t)

    for N, K, V in ((70, 100, 300), (60, 3001, 2001)):
        for out_in in (False, True):
            x, w, b, t = make(N, K, V, out_in, True, 0.1, True, seed=19)
            got, _ = run(capi, off(x), off(w), off(b), t, out_in)
            check(got, *definition(x, w, b, t, out_in))
    for rows, cols in ((100, 70), (140, 300)):
        g, p, buf = (torch.randn(rows, cols, device="cuda", generator=gen(i)) for i in (1, 2, 3))
        want_buf = buf.clone()
        want = capi.muon_step_multi([p], [g], [want_buf], lr=0.1)[0]
        buf = off(buf)
        got = capi.muon_step_multi([off(p)], [off(g)], [buf], lr=0.1)[0]
        # the norm's partial sums are taken in another order: its error, 2^-50, is not seen in float32 but where a rounding tips
        assert float((got - want).norm()) <= 2.0 ** -20 * float(want.norm()) and torch.equal(buf, want_buf)


def test_output_layer_refuses_what_does_not_fit(capi):
    x, w, b, t = make(8, 16, 32, False, True, 0.0, True, seed=18)
    _, saved = capi.linear_softmax_cross_entropy(x, w, b, t)
    f, bwd = capi.linear_softmax_cross_entropy, capi.linear_softmax_cross_entropy_backward
    for args in ((x.t(), w, b, t), (x.double(), w, b, t), (x, w.half(), b, t), (x, w, b[:31].contiguous(), t), (x, w, b, t[:7].contiguous()),
                 (x, w, b, t.float()), (x[:, :15].contiguous(), w, b, t), (x, w, b, t[:, None]), (x[None], w, b, t), (x.cpu(), w, b, t)):
        with pytest.raises(capi.OdlInvalidArgument):
            f(*args)
        with pytest.raises(capi.OdlInvalidArgument):
            bwd(None, *args, saved)
    with pytest.raises(capi.OdlInvalidArgument):
        bwd(torch.ones(2, device="cuda"), x, w, b, t, saved)
    with pytest.raises(capi.OdlInvalidArgument):
        bwd(None, x, w, b, t, (saved[0], saved[1][:7].contiguous()))


# ------------------------------------------------------------------------------------------- orthogonalised updates
def schulz64(u, steps=5, coef=COEF, eps=1e-7):
    a, b, c = coef
    x = u.double()
    x = x / (x.norm() + eps)
    for _ in range(steps):
        if x.shape[0] <= x.shape[1]:
            m = x @ x.t()
            x = a * x + (b * m + c * (m @ m)) @ x
        else:
            m = x.t() @ x
            x = a * x + x @ (b * m + c * (m @ m))
    return x


def schulz_bar(steps, coef=COEF):
    """Relative to the larger of the Frobenius norms of X0 and of the result."""
    lift = abs(coef[0])
    return sum(abs(v) for v in coef) * 3 * 2.0 ** -22 * sum(lift ** i for i in range(steps))


MATRICES = [(1, 1), (1, 7), (7, 1), (2, 3), (31, 33), (64, 64), (65, 100), (100, 65), (97, 97), (128, 300), (300, 128), (257, 769), (769, 257),
            (770, 800), (1030, 1030), (33, 4099), (2100, 2100), (64, 4096), (4096, 128), (128, 513), (513, 60), (120, 1000), (129, 4000)]


@pytest.mark.parametrize("shape", MATRICES)
def test_newton_schulz(capi, shape):
    g = torch.randn(*shape, device="cuda", generator=gen(shape[0] + shape[1])) * 3e-4
    for steps, coef in ((1, COEF), (5, COEF), (3, (1.5, -0.5, 0.0)), (4, (1.875, -1.25, 0.375))):
        got, want = capi.newton_schulz(g, steps=steps, coefficients=coef).double(), schulz64(g, steps, coef)
        off = float((got - want).norm()) / max(1.0, float(want.norm()))
        assert off <= schulz_bar(steps, coef), (steps, off)


def test_newton_schulz_brings_singular_values_near_one(capi):
    g = gen(3)
    u, _ = torch.linalg.qr(torch.randn(200, 120, device="cuda", generator=g).double())
    v, _ = torch.linalg.qr(torch.randn(120, 120, device="cuda", generator=g).double())
    s = torch.logspace(0, -1.2, 120, device="cuda", dtype=torch.float64)
    o = capi.newton_schulz(((u * s) @ v.t()).float().contiguous(), steps=8).double()
    core = u.t() @ o @ v
    values = torch.linalg.svdvals(core)
    assert float(values.min()) > 0.6 and float(values.max()) < 1.3
    assert float((core - torch.diag(core.diagonal())).norm()) < 1e-2 and float((o - u @ core @ v.t()).norm()) < 1e-2


@pytest.mark.parametrize("batch,rows,cols", [(2, 40, 50), (3, 130, 70), (33, 65, 64), (5, 1, 9), (3, 140, 600), (34, 150, 131)])
def test_a_batch_gives_what_its_matrices_give(capi, batch, rows, cols):
    g = torch.randn(batch, rows, cols, device="cuda", generator=gen(batch))
    got = capi.newton_schulz(g)
    for i in range(batch):
        off = float((got[i].double() - schulz64(g[i])).norm()) / max(1.0, float(schulz64(g[i]).norm()))
        assert off <= schulz_bar(5)


def test_newton_schulz_at_the_edges(capi):
    assert bool((capi.newton_schulz(torch.zeros(70, 90, device="cuda")) == 0).all())
    for bad in (float("nan"), float("inf")):
        g = torch.randn(70, 90, device="cuda", generator=gen(1))
        g[3, 4] = bad
        assert bool(capi.newton_schulz(g).isnan().all())
    assert capi.newton_schulz(torch.empty(0, 5, device="cuda")).shape == (0, 5)
    assert capi.newton_schulz(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    one = torch.zeros(100, 130, device="cuda")
    one[7, 9] = -1e-3  # one element carries the whole norm
    got, want = capi.newton_schulz(one), schulz64(one)
    assert float((got.double() - want).norm()) <= schulz_bar(5)
    for scale in (1e30, 1e-4, 1e-20):  # squares past float32's range, and a norm that eps hides
        g = torch.randn(60, 80, device="cuda", generator=gen(2)) * scale
        got, want = capi.newton_schulz(g).double(), schulz64(g)
        floor = 2.0 ** -38 * math.sqrt(60 * 80) * sum(3.4445 ** i for i in range(6))
        assert float((got - want).norm()) <= schulz_bar(5) * max(1.0 if scale > 1e-10 else 0.0, float(want.norm())) + floor
    for t in (torch.randn(4, 4, device="cuda").t()[::2], torch.randn(4, 4, device="cuda").double(), torch.randn(4, device="cuda"),
              torch.randn(4, 4)):
        with pytest.raises(capi.OdlInvalidArgument):
            capi.newton_schulz(t)


def muon64(p, g, buf, lr, momentum, nesterov, decay):
    buf = momentum * buf.double() + g.double()
    o = schulz64(g.double() + momentum * buf if nesterov else buf)
    scale = lr * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
    return p.double() * (1 - lr * decay) - scale * o, buf, scale * max(1.0, float(o.norm()))


@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (False, 0.1)])
def test_muon_steps_over_a_list_of_shapes(capi, nesterov, decay):
    """Shapes that repeat out of order, one of them more often than a launch takes, an empty and a one-row one among them."""
    shapes = [(64, 100), (300, 40), (64, 100), (1, 50), (0, 3), (300, 40), (129, 129)] + [(20, 30)] * 35
    g = gen(21)
    ps = [torch.randn(*s, device="cuda", generator=g) for s in shapes]
    bufs = [torch.zeros(*s, device="cuda") for s in shapes]
    for step in range(3):
        gs = [torch.randn(*s, device="cuda", generator=g) * 1e-2 for s in shapes]
        want = [muon64(p, q, b, 0.05, 0.9, nesterov, decay) for p, q, b in zip(ps, gs, bufs)]
        before = [b.clone() for b in bufs]
        new = capi.muon_step_multi(ps, gs, bufs, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=decay)
        for p, q, b, old, n, (wp, wb, unit) in zip(ps, gs, bufs, before, new, want):
            if p.numel() == 0:
                continue
            # 0.9 as a float32, its product with the old value and the sum are each off by at most 2^-24 of their size:
            # |old| * 0.9 carries all three, |g| the last
            assert bool(((b.double() - wb).abs() <= 2.0 ** -24 * (3 * 0.9 * old.abs() + q.abs()).double() * 1.01).all())
            assert float((n.double() - wp).norm()) <= schulz_bar(5) * unit + 2.0 ** -22 * float(p.norm())
        ps = new


def test_muon_step_in_place_through_the_library(capi):
    """p_out may be p: what the host layer's recorded steps do."""
    from origindl_amd._lib import lib
    p, g, buf = (torch.randn(90, 70, device="cuda", generator=gen(i)) for i in range(3))
    want = capi.muon_step_multi([p.clone()], [g], [buf.clone()], lr=0.1)[0]
    rows, cols = (ctypes.c_int64 * 1)(90), (ctypes.c_int64 * 1)(70)
    nb = lib().query("odl_hip_muon_step_multi_workspace_bytes", 1, rows, cols)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    ptr = lambda t: (ctypes.c_void_p * 1)(t.data_ptr())
    lib().call("odl_hip_muon_step_multi", 1, ptr(p), ptr(g), ptr(buf), rows, cols, 0.1, 0.95, 1, 0.0, 5, *COEF, 1e-7, ptr(p), ws.data_ptr(), nb,
               capi._stream())
    assert torch.equal(p, want)


def test_muon_step_refuses_what_does_not_fit(capi):
    a, b = torch.randn(8, 9, device="cuda"), torch.randn(9, 8, device="cuda")
    step = capi.muon_step_multi
    for args in (([a], [b], [a.clone()]), ([a], [a, a], [a]), ([a, b], [a, b], [a, a]), ([a.double()], [a], [a.clone()]), ([a[0]], [a[0]], [a[1]]),
                 ([a, a.clone()], [a, a], [b.reshape(8, 9), b.reshape(8, 9)])):
        with pytest.raises(capi.OdlInvalidArgument):
            step(*args, lr=0.1)
    assert step([], [], [], lr=0.1) == []


# ------------------------------------------------------------------------------------------------ the host layer
@pytest.fixture(scope="module")
def h():
    import oraclelib as ol
    return ol.host_driver()


@pytest.mark.parametrize("out_in", [0, 1])
@pytest.mark.parametrize("bias", [False, True])
def test_host_operator_and_its_gradients(capi, h, out_in, bias):
    x, w, b, t = make(37, 50, 210, bool(out_in), bias, 0.2, True, seed=31)
    for factor in (1.0, -2.5):
        loss, gx, gw, gb = np.zeros(1, np.float32), np.empty((37, 50), np.float32), np.empty(tuple(w.shape), np.float32), np.empty(210, np.float32)
        assert h.odl_host_linear_softmax_ce(x.cpu().numpy(), w.cpu().numpy(), out_in, b.cpu().numpy() if bias else None, t.cpu().numpy(), 1,
                                            IGNORE, 37, 50, 210, factor, loss, gx, gw, gb) == 0
        want, bars = definition(x, w, b, t, bool(out_in), factor)
        dev = lambda a: torch.from_numpy(a).cuda()
        check((torch.from_numpy(loss)[0], dev(gx), dev(gw), dev(gb) if bias else None), want, bars)


def test_host_operator_reports_labels_out_of_range(capi, h):
    x, w, b, t = make(10, 20, 30, False, False, 0.0, True, seed=32)
    loss = np.zeros(1, np.float32)
    call = lambda labels, V=30: h.odl_host_linear_softmax_ce(x.cpu().numpy(), w.cpu().numpy(), 0, None, labels, 1, IGNORE, 10, 20, V, 1.0, loss, None,
                                                             None, None)
    good = t.cpu().numpy()
    assert call(good) == 0
    ignored = good.copy()
    ignored[2] = IGNORE
    assert call(ignored) == 0
    for bad in (30, -1):
        labels = good.copy()
        labels[3] = bad
        assert call(labels) == -1
        labels[2] = IGNORE
        assert call(labels) == -1


def test_host_newton_schulz(capi, h):
    for batch, rows, cols in ((0, 50, 80), (3, 70, 40)):
        g = torch.randn(*((batch,) if batch else ()), rows, cols, generator=torch.Generator().manual_seed(5))
        o = np.empty(tuple(g.shape), np.float32)
        assert h.odl_host_newton_schulz(g.numpy(), batch, rows, cols, 5, o) == 0
        assert torch.equal(torch.from_numpy(o), capi.newton_schulz(g.cuda()).cpu())
    assert h.odl_host_newton_schulz(g.numpy(), 3, 70, 40, 0, o) == -1


def train64(x, t, params, steps, lr, decay, adam_lr):
    """Linear + ReLU + Linear + loss, Muon for the weights, Adam for the biases, in float64."""
    w1, b1, w2, b2 = (p.double() for p in params)
    m1, m2 = torch.zeros_like(w1), torch.zeros_like(w2)
    am, av = [torch.zeros_like(b1), torch.zeros_like(b2)], [torch.zeros_like(b1), torch.zeros_like(b2)]
    losses = []
    for step in range(1, steps + 1):
        pre = x.double() @ w1 + b1
        a = pre.clamp(min=0)
        (loss, ga, gw2, gb2), _ = definition(a, w2, b2, t, False)
        gp = ga * (pre > 0)
        grads_b = [gp.sum(0, keepdim=True), gb2.reshape(b2.shape)]
        w1, m1, _ = muon64(w1, x.double().t() @ gp, m1, lr, 0.95, True, decay)
        w2, m2, _ = muon64(w2, gw2, m2, lr, 0.95, True, decay)
        for i, (bias, g) in enumerate(zip((b1, b2), grads_b)):
            am[i] = 0.9 * am[i] + 0.1 * g
            av[i] = 0.999 * av[i] + 0.001 * g * g
            new = bias - adam_lr * (am[i] / (1 - 0.9 ** step)) / ((av[i] / (1 - 0.999 ** step)).sqrt() + 1e-8)
            b1, b2 = (new, b2) if i == 0 else (b1, new)
        losses.append(float(loss))
    return [w1, b1, w2, b2], losses


def test_host_training_steps_with_muon(capi, h):
    """A run of the operators as a training program uses them: both layers' weights by Muon, the biases by Adam. Two steps
    from float32 gradients: an orthogonalised update's elements err by its bar, its inputs' error (relative 1e-5) passes
    through the steps with at most 3.4445^5; the second step's gradients see the first one's parameters. The recorded step
    and the one after moving the optimizer's state into a fresh one give the bits of plain steps."""
    N, D, H, V, lr, decay, adam_lr = 48, 40, 72, 300, 0.02, 0.01, 1e-3
    g = torch.Generator().manual_seed(41)
    x, t = torch.randn(N, D, generator=g), torch.randint(0, V, (N,), generator=g)
    start = [torch.randn(D, H, generator=g) / D ** 0.5, 0.1 * torch.randn(1, H, generator=g), torch.randn(H, V, generator=g) / H ** 0.5,
             0.1 * torch.randn(1, V, generator=g)]
    flat = torch.cat([p.reshape(-1) for p in start]).numpy()
    results = {}
    for mode in (0, 1, 2):
        params, losses = flat.copy(), np.zeros(3, np.float32)
        assert h.odl_host_muon_train(x.numpy(), t.numpy(), N, D, H, V, 3, mode, lr, decay, adam_lr, params, losses) == 0
        results[mode] = (params, losses)
    assert np.array_equal(results[0][0], results[2][0]) and np.array_equal(results[0][1], results[2][1])
    assert np.array_equal(results[0][0], results[1][0]) and np.array_equal(results[0][1], results[1][1])
    params, losses = flat.copy(), np.zeros(1, np.float32)
    assert h.odl_host_muon_train(x.numpy(), t.numpy(), N, D, H, V, 1, 0, lr, decay, adam_lr, params, losses) == 0
    want, want_losses = train64(x.cuda(), t.cuda(), [p.cuda() for p in start], 1, lr, decay, adam_lr)
    assert abs(losses[0] - want_losses[0]) <= 1e-4 * want_losses[0]
    at = 0
    for i, (p, w) in enumerate(zip(start, want)):
        got = torch.from_numpy(params[at:at + p.numel()]).reshape(p.shape).cuda().double()
        at += p.numel()
        if i % 2 == 0:
            scale = lr * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * min(p.shape) ** 0.5 * 1.21
            assert float((got - w).norm()) <= scale * (schulz_bar(5) + 1e-5 * 3.4445 ** 5) + 2.0 ** -22 * float(p.norm())
        else:  # Adam's first step is adam_lr times the gradient's sign, smoothed by eps against the gradient's size
            assert bool(((got - w).abs() <= 0.02 * adam_lr).float().mean() > 0.97) and bool(((got - p.cuda().double()).abs() <= 1.01 * adam_lr).all())


def test_host_muon_steps_a_shared_parameter_once_and_keeps_its_state(capi, h):
    """A parameter registered under two names gives the bits of the same one registered once; the momentum in a state taken
    after the first step is that step's, the gradient itself, whatever either optimizer has done since."""
    rows, cols = 40, 56
    g = torch.Generator().manual_seed(77)
    p, q = torch.randn(rows, cols, generator=g), torch.randn(rows, cols, generator=g)
    results = []
    for names in (1, 2):
        o, kept = np.empty((rows, cols), np.float32), np.empty((rows, cols), np.float32)
        assert h.odl_host_muon_shared(p.numpy(), q.numpy(), rows, cols, names, 3, 0.05, o, kept) == 0
        assert np.array_equal(kept, q.numpy())
        results.append(o)
    assert np.array_equal(results[0], results[1])
    want, buf = p, torch.zeros_like(p)
    for _ in range(3):
        want, buf, _ = muon64(want, q, buf, 0.05, 0.95, True, 0.0)
    off = float((torch.from_numpy(results[0]).double() - want).norm())
    assert off <= 3 * (0.05 * 1.21 * rows ** 0.5 * schulz_bar(5) + 2.0 ** -22 * float(p.norm()))
