"""The output layer with its loss and the orthogonalised updates where their sizes, magnitudes and masks end, against their
definitions in 64 bits; the bars are those of test_gpu_lm_training."""
import ctypes
import math

import numpy as np
import pytest
import torch

from test_gpu_lm_training import COEF, check, definition, gen, make, run, schulz64, schulz_bar

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from origindl_amd import capi
    return capi


@pytest.mark.parametrize("count,rows,cols", [(63, 384, 1920), (63, 320, 1920), (35, 2000, 130), (33, 90, 5000)])
def test_a_batch_stays_inside_the_workspace_it_asks_for(capi, count, rows, cols):
    """What lies right behind the workspace keeps its bytes, whatever the last group's products are cut into."""
    from origindl_amd._lib import lib
    g = torch.randn(count, rows, cols, device="cuda", generator=gen(rows)) * 1e-2
    out = torch.empty_like(g)
    nb, guard = lib().query("odl_hip_newton_schulz_workspace_bytes", count, rows, cols), 64 << 20
    ws = torch.full((nb + guard,), 0x5A, dtype=torch.uint8, device="cuda")
    lib().call("odl_hip_newton_schulz", g.data_ptr(), count, rows, cols, 5, *COEF, 1e-7, out.data_ptr(), ws.data_ptr(), nb, capi._stream())
    assert bool((ws[nb:] == 0x5A).all())
    for i in (0, 31, 32, count - 1):
        want = schulz64(g[i])
        assert float((out[i].double() - want).norm()) <= schulz_bar(5) * max(1.0, float(want.norm())), i


# ---------------------------------------------------------------------------------- the factor of an update: outputs and inputs
def factor(inputs, outputs):
    """What an orthogonalised update of a layer is multiplied by: more where it has more outputs than inputs."""
    return math.sqrt(max(1.0, outputs / inputs))


@pytest.fixture(scope="module")
def h():
    import oraclelib as ol
    return ol.host_driver()


def muon_of(p, g, buf, lr, scale, decay=0.0, momentum=0.95):
    buf = momentum * buf + g
    o = schulz64(g + momentum * buf)
    return p * (1 - lr * decay) - lr * scale * o, buf, lr * scale * float(o.norm())


def test_updates_of_matrices_kept_either_way_round(capi):
    """[outputs, inputs], [inputs, outputs] and both of one shape in the same launches."""
    shapes = [(96, 40), (96, 40), (40, 96), (40, 96), (300, 130), (300, 130), (200, 4100), (4100, 200), (70, 70)]
    in_out = [False, True, False, True, True, False, True, True, True]
    g = gen(51)
    ps, gs, bufs = ([torch.randn(*s, device="cuda", generator=g) for s in shapes] for _ in range(3))
    want = [muon_of(p.double(), q.double(), b.double(), 0.05, factor(*(s if f else s[::-1])), 0.1)
            for p, q, b, s, f in zip(ps, gs, bufs, shapes, in_out)]
    new = capi.muon_step_multi(ps, gs, [b.clone() for b in bufs], lr=0.05, weight_decay=0.1, in_out=in_out)
    for p, n, (w, _, unit) in zip(ps, new, want):
        assert float((n.double() - w).norm()) <= schulz_bar(5) * unit + 2.0 ** -22 * float(p.norm())
    # without the list all are [outputs, inputs]
    plain = capi.muon_step_multi(ps, gs, [b.clone() for b in bufs], lr=0.05, weight_decay=0.1)
    none = capi.muon_step_multi(ps, gs, [b.clone() for b in bufs], lr=0.05, weight_decay=0.1, in_out=[False] * len(ps))
    assert all(torch.equal(a, b) for a, b in zip(plain, none))
    assert all(torch.equal(a, b) for a, b, f in zip(plain, new, in_out) if not f)
    with pytest.raises(capi.OdlInvalidArgument):
        capi.muon_step_multi(ps, gs, bufs, lr=0.05, in_out=[True])


@pytest.mark.parametrize("rows,cols", [(40, 96), (96, 40)])
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
def test_host_optimizer_knows_which_side_counts_the_outputs(h, rows, cols, kind):
    g = torch.Generator().manual_seed(52)
    p, q = torch.randn(rows, cols, generator=g), torch.randn(rows, cols, generator=g)
    o = np.empty((rows, cols), np.float32)
    assert h.odl_host_muon_place(p.numpy(), q.numpy(), rows, cols, kind, 0.05, o) == 0
    scale = factor(rows, cols) if kind in (1, 2) else factor(cols, rows)
    want, _, unit = muon_of(p.double(), q.double(), torch.zeros(rows, cols, dtype=torch.float64), 0.05, scale)
    assert float((torch.from_numpy(o).double() - want).norm()) <= schulz_bar(5) * unit + 2.0 ** -22 * float(p.norm())


def test_training_steps_with_muon(h):
    """Linear, ReLU, Linear and the loss, the weights by Muon and the biases by Adam: three steps, of them the last recorded or with
    the state moved into a fresh optimizer, give the bits of plain ones; the first one is held to 64 bits. An orthogonalised
    update's elements err by its bar, its inputs' error (relative 1e-5) passes through five steps with at most 3.4445 each."""
    N, D, H, V, lr, decay, adam_lr = 48, 40, 72, 300, 0.02, 0.01, 1e-3
    g = torch.Generator().manual_seed(41)
    x, t = torch.randn(N, D, generator=g), torch.randint(0, V, (N,), generator=g)
    start = [torch.randn(D, H, generator=g) / D ** 0.5, 0.1 * torch.randn(1, H, generator=g), torch.randn(H, V, generator=g) / H ** 0.5,
             0.1 * torch.randn(1, V, generator=g)]
    flat = torch.cat([p.reshape(-1) for p in start]).numpy()
    results = []
    for mode in (0, 1, 2):
        params, losses = flat.copy(), np.zeros(3, np.float32)
        assert h.odl_host_muon_train(x.numpy(), t.numpy(), N, D, H, V, 3, mode, lr, decay, adam_lr, params, losses) == 0
        results.append((params, losses))
    for params, losses in results[1:]:
        assert np.array_equal(params, results[0][0]) and np.array_equal(losses, results[0][1])
    params, losses = flat.copy(), np.zeros(1, np.float32)
    assert h.odl_host_muon_train(x.numpy(), t.numpy(), N, D, H, V, 1, 0, lr, decay, adam_lr, params, losses) == 0
    w1, b1, w2, b2 = (p.double().cuda() for p in start)
    pre = x.double().cuda() @ w1 + b1
    (loss, ga, gw2, gb2), _ = definition(pre.clamp(min=0), w2, b2, t.cuda(), False)
    gp = ga * (pre > 0)
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    assert abs(float(losses[0]) - float(loss)) <= 1e-4 * float(loss)
    at = 0
    for p, w, grad in ((start[0], w1, x.double().cuda().t() @ gp), (start[1], b1, gp.sum(0)), (start[2], w2, gw2), (start[3], b2, gb2)):
        got = torch.from_numpy(params[at:at + p.numel()]).reshape(p.shape).cuda().double()
        at += p.numel()
        if p.shape[0] > 1:
            want, _, unit = muon_of(w, grad, zero, lr, factor(*p.shape), decay)
            assert float((got - want).norm()) <= unit * (schulz_bar(5) + 1e-5 * 3.4445 ** 5) + 2.0 ** -22 * float(p.norm())
        else:
            # Adam's first step is adam_lr * g / (|g| + 1e-8): the sign, where the gradient is known well enough
            sure = grad.reshape(p.shape).abs() > 1e-4 * grad.abs().max()
            want = w - adam_lr * grad.reshape(p.shape) / (grad.reshape(p.shape).abs() + 1e-8)
            assert bool(((got - want).abs()[sure] <= 0.01 * adam_lr).all()) and bool(((got - w).abs() <= 1.01 * adam_lr).all())


# ----------------------------------------------------------------------------------------------------- large vocabularies
@pytest.mark.parametrize("shape", [(256, 33, 400001), (90, 40, 500000), (40, 130, 1600003), (3, 150, 1500001), (200, 1024, 200001)])
@pytest.mark.parametrize("out_in", [False, True])
def test_few_rows_over_a_vocabulary_in_several_pieces(capi, shape, out_in):
    """Pieces that end inside a tile, with and without logits kept from the forward pass: gx adds up over them, gw and gb are written
    piece by piece, a label may lie in any of them."""
    N, K, V = shape
    x, w, b, t = make(N, K, V, out_in, True, 0.1, True, seed=61)
    t[0], t[N // 2], t[N - 1] = 0, V // 2, V - 1
    got, saved = run(capi, x, w, b, t, out_in)
    check(got, *definition(x, w, b, t, out_in))
    part = capi.linear_softmax_cross_entropy_backward(None, x, w, b, t, saved, w_out_in=out_in, need_gw=False, need_gb=False)
    assert torch.equal(part[0], got[1])


@pytest.mark.parametrize("N,V,out_in", [(1, 1 << 30, False), (200, (1 << 28) + 3, True)])
def test_vocabularies_past_what_one_launch_counts(capi, N, V, out_in):
    """The largest vocabulary, one feature: the logits of more tiles than a launch has threads for. With one feature z = x w is one
    product, off by 2^-22 of it at most, and a probability by that times 2 |z| and 2^-20 besides (exponential, sum, quotient)."""
    x, w, _, t = make(N, 1, V, out_in, False, 0.0, True, seed=62)
    t[0] = V - 1
    (loss, gx, gw, gb), saved = run(capi, x, w, None, t, out_in)
    assert not capi.linear_softmax_cross_entropy_bad_label(saved)
    X, flat, step = x.double(), w.view(-1), 1 << (22 if N > 1 else 26)
    lse = torch.full((N,), -math.inf, device="cuda", dtype=torch.float64)
    for v in range(0, V, step):
        lse = torch.logaddexp(lse, torch.logsumexp(X * flat[v:v + step].double(), dim=1))
    want = float((lse - X[:, 0] * flat[t].double()).mean())
    top = float(X.abs().max()) * float(flat.abs().max())
    assert abs(float(loss) - want) <= 2.0 ** -21 * top + 2.0 ** -20 * (1 + float(lse.abs().max()))
    want_gx = torch.zeros(N, device="cuda", dtype=torch.float64)
    grad = gw.view(-1)
    for v in range(0, V, step):
        part = flat[v:v + step].double()
        d = torch.exp(X * part - lse[:, None])
        bar = d * (2 * 2.0 ** -22 * top + 2.0 ** -20)
        inside = (t >= v) & (t < v + step)
        d[inside.nonzero()[:, 0], t[inside] - v] -= 1
        want_gx += torch.mv(d, part)
        for got, scale in ((grad, X), (gb, torch.ones_like(X))):
            off = (got[v:v + step].double() - (d * scale).sum(0) / N).abs()
            tol = (bar * scale.abs()).sum(0) / N + 2.0 ** -20 * (d * scale).abs().sum(0) / N + 2.0 ** -100
            assert bool((off <= tol).all()), (v, float((off / tol).max()))
    # sum_v d w: a sum of V terms p w, whose error relative to the sum of their magnitudes (at most max |w|) is that of p and of the sum
    tol = float(flat.abs().max()) / N * (2 * 2.0 ** -22 * top + 2.0 ** -18)
    assert bool(((gx[:, 0].double() - want_gx / N).abs() <= tol).all())


# --------------------------------------------------------------------------------------------------- masks and magnitudes
LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("N,K,V", [(5, 40, 130), (300, 70, 1000), (9, 300, 21000), (130, 600, 10500)])
def test_a_mask_of_the_lowest_value_that_leaves_nothing(capi, N, K, V):
    """Every entry masked with the type's lowest value: x w is lost in it (|z| < 2^-25 of it), all entries are equal, the loss is the
    logarithm of their number and the gradient 1 / their number. Entries at -inf beside them are no entries."""
    x, w, b, t = make(N, K, V, False, True, 0.0, True, seed=71)
    for gone in (0, V // 3):
        b[:] = LOWEST
        b[V - gone:] = -float("inf")
        t %= V - gone
        (loss, gx, gw, gb), _ = run(capi, x, w, b, t, False)
        left = V - gone
        assert abs(float(loss) - math.log(left)) <= 2.0 ** -20 * (1 + math.log(left))
        d = torch.full((N, left), 1.0 / left, device="cuda", dtype=torch.float64)
        d[torch.arange(N, device="cuda"), t] -= 1
        d /= N
        zeros = torch.zeros(N, V - left, device="cuda", dtype=torch.float64)
        d, size = torch.cat([d, zeros], 1), torch.cat([d.abs(), zeros], 1)
        # a probability is off by 2^-20 of itself, as an operand by 2^-40 besides; products are held to 1e-5 of their rows
        e = size * 2.0 ** -20 + 2.0 ** -40 / N
        for got, want, tol in ((gb, d.sum(0), e.sum(0)),
                               (gx, d @ w.t().double(), e @ w.t().double().abs() + 1e-5 * d.norm(dim=1)[:, None] * w.double().norm(dim=1)),
                               (gw, x.t().double() @ d, x.t().double().abs() @ e + 1e-5 * x.double().norm(dim=0)[:, None] * d.norm(dim=0))):
            assert bool(((got.double() - want).abs() <= tol).all())
        assert bool((gb[left:] == 0).all()) and bool((gw[:, left:] == 0).all())


@pytest.mark.parametrize("N,K,V", [(6, 30, 200), (300, 64, 900), (6, 300, 21000)])
def test_masks_that_leave_an_entry_and_logits_near_the_ends_of_the_range(capi, N, K, V):
    x, w, b, t = make(N, K, V, True, True, 0.0, True, seed=72)
    # all but one entry at the lowest value: it has the whole probability
    b[:] = LOWEST
    b[7] = 0.25
    t[:] = 7
    (loss, gx, gw, gb), _ = run(capi, x, w, b, t, True)
    assert float(loss) == 0 and all(bool((g == 0).all()) for g in (gx, gw, gb))
    # logits of 3e38 and of -3e38 side by side: their distance overflows, the probabilities are 1 and 0
    b[:] = -3e38
    b[3] = 3e38
    t[:] = 3
    (loss, gx, gw, gb), _ = run(capi, x, w, b, t, True)
    assert float(loss) == 0 and all(bool((g == 0).all()) for g in (gx, gw, gb))
    t[0] = 5
    loss, _ = capi.linear_softmax_cross_entropy(x, w, b, t, w_out_in=True)
    # (the entries are float32's neighbours of 3e38; the mean of one such distance and N - 1 zeros, rounded once)
    assert float(loss) == float(np.float32((float(b[3]) - float(b[5])) / N))


@pytest.mark.parametrize("rows,cols", [(50, 60), (300, 90), (200, 5000), (1, 1)])
def test_a_zero_matrix_gives_zeros_without_eps_too(capi, rows, cols):
    zero = torch.zeros(rows, cols, device="cuda")
    for eps in (0.0, 1e-7):
        assert bool((capi.newton_schulz(zero, eps=eps) == 0).all())
        p, buf = torch.randn(rows, cols, device="cuda", generator=gen(81)), zero.clone()
        (new,) = capi.muon_step_multi([p], [zero], [buf], lr=0.1, eps=eps)
        assert torch.equal(new, p) and bool((buf == 0).all())
    # without eps the magnitude does not matter, down to float32's smallest numbers
    g = torch.randn(rows, cols, device="cuda", generator=gen(82))
    small = (g.double() * 2.0 ** -140).float()
    got, want = capi.newton_schulz(small, eps=0.0), schulz64(small, eps=0.0)
    assert float((got.double() - want).norm()) <= schulz_bar(5) * max(1.0, float(want.norm()))


@pytest.mark.parametrize("N,K,V", [(50, 70, 200), (300, 70, 200), (50, 31000, 200)])
@pytest.mark.parametrize("sx,sw", [(1e35, 1e-32), (1e-32, 1e35), (3e36, 1e-36)])
def test_operands_of_opposite_magnitudes(capi, N, K, V, sx, sw):
    """Logits up to thousands from operands near the ends of float32's range. Few rows over large weights: an operand's three bfloat16
    parts end at bfloat16's smallest number, 2^-133, so an element is off by that at most and a logit by 2^-133 (|x|_1 + |w|_1): of
    weights about 1e-38 that is their seventh bit, and the bars are widened by it."""
    x, w, b, t = make(N, K, V, False, True, 0.0, True, seed=91)
    x, w = x * sx, w * sw
    got, _ = run(capi, x, w, b, t, False)
    want, bars = definition(x, w, b, t, False)
    if N * K >= 50 * 31000:
        e = 2.0 ** -133 * float(x.double().abs().sum(1).max() + w.double().abs().sum(0).max())
        lift = math.expm1(2 * e)  # of a probability, in each gradient: softmax - one-hot is off by lift * p, |p| <= 1
        W, X = w.t().double(), x.double()
        bars = (bars[0] + 2 * e, bars[1] + lift * W.abs().max(dim=0).values / N, bars[2] + lift * X.abs().sum(0)[:, None] / N, bars[3] + lift)
    check(got, want, bars)
    assert all(bool(g.isfinite().all()) for g in got)


@pytest.mark.parametrize("N,K,V", [(300, 8, 2), (250, 8, 750001), (70, 2000, 3001)])
def test_a_mean_gradient_whose_sum_is_out_of_range(capi, N, K, V):
    """Rows of 1e37 to 2e37 under one label: the sum over the rows overflows, the mean does not."""
    g = gen(92)
    x = (1 + torch.rand(N, K, device="cuda", generator=g)) * 1e37
    w, b = torch.zeros(V, K, device="cuda"), torch.zeros(V, device="cuda")
    t = torch.zeros(N, dtype=torch.long, device="cuda")
    got, _ = run(capi, x, w, b, t, True)
    want, bars = definition(x, w, b, t, True)
    check(got, want, bars)
    assert bool(got[2].isfinite().all())


@pytest.mark.parametrize("N,K,V", [(300, 256, 700), (64, 3000, 2100)])
def test_rows_and_entries_of_unequal_size(capi, N, K, V):
    """Rows of x, and entries of w, from 1 down to 2^-24 of the largest: each row's logits keep the bar of a float32 product of its own
    row (an element is off by 2^-39 of the largest, 2^-15 of an element 2^-24 as large, and those errors add up as a sum's)."""
    x, w, b, t = make(N, K, V, True, True, 0.1, True, seed=95)
    x = x * torch.logspace(0, -24, N, base=2, device="cuda")[torch.randperm(N, device="cuda", generator=gen(96))][:, None]
    w = w * torch.logspace(0, -24, V, base=2, device="cuda")[torch.randperm(V, device="cuda", generator=gen(97))][:, None]
    got, _ = run(capi, x, w, b, t, True)
    check(got, *definition(x, w, b, t, True))


def test_a_bias_without_dimensions_is_refused(capi):
    x, w, _, t = make(4, 8, 1, False, False, 0.0, True, seed=98)
    with pytest.raises(capi.OdlInvalidArgument):
        capi.linear_softmax_cross_entropy(x, w, torch.zeros((), device="cuda"), t)
    loss, _ = capi.linear_softmax_cross_entropy(x, w, torch.zeros(1, device="cuda"), t)
    assert float(loss) == 0  # one class: its probability is 1
