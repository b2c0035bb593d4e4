"""Workloads of the framework's language-model training operators: the output layer with its loss and gradients
(linear_softmax_cross_entropy) and the orthogonalised optimiser update (newton_schulz, muon_step_multi).

Each case is a dict of plain values; `prepare` makes its inputs, `run` makes one pass — in plain torch operations, or through
the framework's entry points where `own` is set — and `exact` computes the same outputs in 64 bits."""
import math

import torch

own = False

IGNORE = -100
MUON = {"lr": 0.02, "momentum": 0.95}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7


def listed():
    return [
        # scoring one position of a sequence: latency, the weights are read once
        {"name": "loss_one_row", "op": "ce", "N": 1, "K": 2048, "V": 32000, "train": False, "bias": True, "out_in": False,
         "ignored": 0.0, "i64": True},
        # a small classifier's training step: launches count
        {"name": "train_small", "op": "ce", "N": 64, "K": 256, "V": 1000, "train": True, "bias": True, "out_in": False,
         "ignored": 0.0, "i64": False},
        # a padded batch of ragged sequences, weights shared with an embedding ([V, K]), nothing a multiple of a tile
        {"name": "train_padded_odd", "op": "ce", "N": 1337, "K": 771, "V": 50001, "train": True, "bias": False, "out_in": True,
         "ignored": 0.25, "i64": True},
        # an ordinary training step
        {"name": "train_tokens", "op": "ce", "N": 4096, "K": 1024, "V": 32000, "train": True, "bias": True, "out_in": False,
         "ignored": 0.0, "i64": True},
        # the largest: a wide model over a large vocabulary
        {"name": "train_large", "op": "ce", "N": 8192, "K": 2048, "V": 128000, "train": True, "bias": False, "out_in": True,
         "ignored": 0.0, "i64": True},
        # validation loss of a long document
        {"name": "loss_long", "op": "ce", "N": 16384, "K": 1024, "V": 32000, "train": False, "bias": True, "out_in": False,
         "ignored": 0.05, "i64": True},
        # the update of a small projection: latency
        {"name": "orth_small", "op": "ns", "count": 1, "rows": 128, "cols": 128},
        # the framework's MLP's hidden layer
        {"name": "orth_hidden", "op": "ns", "count": 1, "rows": 1000, "cols": 1000},
        # tall and odd
        {"name": "orth_tall_odd", "op": "ns", "count": 1, "rows": 2001, "cols": 333},
        # the largest square layer
        {"name": "orth_large", "op": "ns", "count": 1, "rows": 4096, "cols": 4096},
        # an optimiser step over the equal projections of a stack of layers
        {"name": "muon_layers", "op": "muon", "count": 8, "rows": 512, "cols": 512, "nesterov": True, "decay": 0.0},
        # an optimiser step of one wide feed-forward matrix, with weight decay
        {"name": "muon_wide", "op": "muon", "count": 1, "rows": 1024, "cols": 4096, "nesterov": True, "decay": 0.01},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over their logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("ce", "ce", "ns", "muon"))
    if kind == "ce":
        most = 3 * 8192 * 2048 * 128000
        while True:
            case = {"op": "ce", "N": _spread(rng, 1, 16384), "K": _spread(rng, 64, 2048), "V": _spread(rng, 1000, 128000),
                    "train": rng.random() < 0.7, "bias": rng.random() < 0.5, "out_in": rng.random() < 0.5,
                    "ignored": rng.choice((0.0, 0.1, 0.5)), "i64": rng.random() < 0.7}
            if (3 if case["train"] else 1) * case["N"] * case["K"] * case["V"] <= most and case["N"] * case["V"] <= 8192 * 128000:
                return case
    while True:
        case = {"op": kind, "count": 1 if kind == "ns" else rng.randint(1, 12), "rows": _spread(rng, 64, 4096), "cols": _spread(rng, 64, 4096)}
        if kind == "muon":
            case["nesterov"] = rng.random() < 0.7
            case["decay"] = rng.choice((0.0, 0.01))
        short, long = sorted((case["rows"], case["cols"]))
        if case["count"] * short * short * long <= 4096 ** 3:
            return case


def _gradient(case, gen):
    """Matrices with the falling spectrum of a layer's gradient: a part of low rank under noise."""
    count, rows, cols = case["count"], case["rows"], case["cols"]
    rank = max(1, min(rows, cols) // 8)
    out = []
    for _ in range(count):
        left = torch.randn(rows, rank, device="cuda", generator=gen) * torch.logspace(0, -2, rank, device="cuda")
        low = left @ torch.randn(rank, cols, device="cuda", generator=gen)
        out.append((low + 0.3 * torch.randn(rows, cols, device="cuda", generator=gen)) * 1e-3)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "ce":
        N, K, V = case["N"], case["K"], case["V"]
        state["x"] = torch.randn(N, K, device="cuda", generator=gen)
        state["w"] = torch.randn((V, K) if case["out_in"] else (K, V), device="cuda", generator=gen) * (1.5 / math.sqrt(K))
        state["b"] = torch.randn(V, device="cuda", generator=gen) * 0.5 if case["bias"] else None
        # frequent classes come first, as in a vocabulary sorted by frequency
        u = torch.rand(N, device="cuda", generator=gen, dtype=torch.float64)
        t = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)
        t[torch.rand(N, device="cuda", generator=gen) < case["ignored"]] = IGNORE
        state["t"] = t if case["i64"] else t.int()
        state["gy"] = torch.rand((), device="cuda", generator=gen) + 0.5
        return state
    state["g"] = _gradient(case, gen)
    if case["op"] == "muon":
        state["p"] = [torch.randn(case["rows"], case["cols"], device="cuda", generator=gen) / math.sqrt(case["cols"]) for _ in state["g"]]
        state["buf"] = [(a + b) * 5.0 for a, b in zip(_gradient(case, gen), state["g"])]
    return state


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_ce(s, train):
    x, w, b, t = s["x"], s["w"], s["b"], s["t"].long()
    counted = t != IGNORE
    count = counted.sum().clamp(min=1)
    at = torch.where(counted, t, torch.zeros_like(t))[:, None]
    w_kv = w.t() if s["case"]["out_in"] else w
    z = x @ w_kv
    if b is not None:
        z = z + b
    z = z - z.max(dim=1, keepdim=True).values
    picked = z.gather(1, at)[:, 0]
    p = z.exp_()
    total = p.sum(dim=1)
    rows = torch.where(counted, (total.log() - picked).double(), torch.zeros((), dtype=torch.float64, device=x.device))
    loss = (rows.sum() / count).float()
    if not train:
        return loss
    p = p.div_(total[:, None])
    p.scatter_(1, at, p.gather(1, at) - 1)
    p = p.mul_((s["gy"] / count * counted)[:, None])
    gx = p @ w_kv.t()
    gw = p.t() @ x if s["case"]["out_in"] else x.t() @ p
    return (loss, gx, gw) if b is None else (loss, gx, gw, p.sum(dim=0))


def _plain_ns(g):
    """g: [count, rows, cols]."""
    a, b, c = COEFFICIENTS
    tall = g.shape[1] > g.shape[2]
    x = g.transpose(1, 2).contiguous() if tall else g
    norm = x.double().square().sum(dim=(1, 2), keepdim=True).sqrt()
    x = x / (norm + EPS).float()
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2).contiguous()
        poly = b * gram + c * (gram @ gram)
        # each step passes on what its product rounds, up to 1.6 times: long sums are added up in quarters
        if poly.shape[2] <= 1024:
            x = a * x + poly @ x
        else:
            x = a * x + sum(p @ q for p, q in zip(poly.chunk(4, dim=2), x.chunk(4, dim=1)))
    return x.transpose(1, 2).contiguous() if tall else x


def _plain_muon(s):
    case, mu = s["case"], MUON["momentum"]
    g, p, buf = torch.stack(s["g"]), torch.stack(s["p"]), torch.stack(s["buf"])
    buf = buf * mu + g
    for kept, new in zip(s["buf"], buf):
        kept.copy_(new)
    o = _plain_ns(g + buf * mu if case["nesterov"] else buf)
    scale = MUON["lr"] * math.sqrt(max(1.0, case["rows"] / case["cols"]))
    p = p * (1 - MUON["lr"] * case["decay"]) - o * scale
    return list(p.unbind(0)) + s["buf"]


# ------------------------------------------------------------------------------------------------------------ run
def run(state):
    case = state["case"]
    if own:
        from origindl_amd import capi
        if case["op"] == "ce":
            x, w, b, t = state["x"], state["w"], state["b"], state["t"]
            loss, saved = capi.linear_softmax_cross_entropy(x, w, b, t, ignore_index=IGNORE, w_out_in=case["out_in"])
            if not case["train"]:
                return loss
            gx, gw, gb = capi.linear_softmax_cross_entropy_backward(state["gy"], x, w, b, t, saved, ignore_index=IGNORE,
                                                                    w_out_in=case["out_in"], need_gb=b is not None)
            return (loss, gx, gw) if b is None else (loss, gx, gw, gb)
        if case["op"] == "ns":
            return capi.newton_schulz(state["g"][0], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        p = capi.muon_step_multi(state["p"], state["g"], state["buf"], nesterov=case["nesterov"], weight_decay=case["decay"],
                                 steps=STEPS, coefficients=COEFFICIENTS, eps=EPS, **MUON)
        return p + state["buf"]
    if case["op"] == "ce":
        return _plain_ce(state, case["train"])
    if case["op"] == "ns":
        return _plain_ns(state["g"][0][None])[0]
    return _plain_muon(state)


# ---------------------------------------------------------------------------------------------------------- exact
def _exact_ce(s):
    x, w, b, t = s["x"].double(), s["w"], s["b"], s["t"].tolist()
    if not s["case"]["out_in"]:
        w = w.t()
    keep = [n for n, label in enumerate(t) if label != IGNORE]
    count = max(1, len(keep))
    keep = torch.tensor(keep, device=x.device, dtype=torch.long)
    label = s["t"].long()[keep]
    V, step, train = w.shape[0], 16384, s["case"]["train"]
    xk = x[keep]

    def logits(v0):
        z = torch.mm(xk, w[v0:v0 + step].double().t())
        return z if b is None else z + b[v0:v0 + step].double()

    lse = torch.full((len(keep),), -math.inf, device=x.device, dtype=torch.float64)
    hit = torch.zeros(len(keep), device=x.device, dtype=torch.float64)
    rows = torch.arange(len(keep), device=x.device)
    for v0 in range(0, V, step):
        z = logits(v0)
        lse = torch.logaddexp(lse, torch.logsumexp(z, dim=1))
        inside = (label >= v0) & (label < v0 + step)
        hit[inside] = z[rows[inside], label[inside] - v0]
    loss = (lse - hit).sum() / count
    if not train:
        return loss
    gx = torch.zeros_like(x)
    gw = torch.empty(w.shape, device=x.device, dtype=torch.float64)
    gb = torch.empty(V, device=x.device, dtype=torch.float64)
    gxk = torch.zeros_like(xk)
    factor = s["gy"].double() / count
    for v0 in range(0, V, step):
        d = torch.exp(logits(v0) - lse[:, None])
        inside = (label >= v0) & (label < v0 + step)
        d[rows[inside], label[inside] - v0] -= 1
        d *= factor
        gxk += torch.mm(d, w[v0:v0 + step].double())
        gw[v0:v0 + step] = torch.mm(d.t(), xk)
        gb[v0:v0 + step] = d.sum(dim=0)
    gx[keep] = gxk
    if not s["case"]["out_in"]:
        gw = gw.t().contiguous()
    return (loss, gx, gw) if b is None else (loss, gx, gw, gb)


def _exact_ns(u):
    """u: [rows, cols] in 64 bits; the polynomial is applied from the side of the shorter dimension."""
    a, b, c = COEFFICIENTS
    x = u / (torch.linalg.vector_norm(u) + EPS)
    eye = torch.eye(min(u.shape), device=u.device, dtype=torch.float64)
    for _ in range(STEPS):
        if u.shape[0] <= u.shape[1]:
            m = torch.mm(x, x.t())
            x = torch.mm(a * eye + torch.mm(m, b * eye + c * m), x)
        else:
            m = torch.mm(x.t(), x)
            x = torch.mm(x, a * eye + torch.mm(m, b * eye + c * m))
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ce":
        return _exact_ce(s)
    if case["op"] == "ns":
        return _exact_ns(s["g"][0].double())
    mu, scale = MUON["momentum"], MUON["lr"] * max(1.0, case["rows"] / case["cols"]) ** 0.5
    params, bufs = [], []
    for g, p, buf in zip(s["g"], s["p"], s["buf"]):
        g = g.double()
        buf = mu * buf.double() + g
        o = _exact_ns(g + mu * buf if case["nesterov"] else buf)
        params.append((1 - MUON["lr"] * case["decay"]) * p.double() - scale * o)
        bufs.append(buf)
    return params + bufs


# ----------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "ce":
        N, K, V = case["N"], case["K"], case["V"]
        inputs = 4 * (N * K + K * V + (V if case["bias"] else 0)) + N * (8 if case["i64"] else 4)
        if not case["train"]:
            return {"bytes": inputs + 4, "flops": 2 * N * K * V}
        return {"bytes": inputs + 4 + 4 * (N * K + K * V + (V if case["bias"] else 0)), "flops": 6 * N * K * V}
    m, n = sorted((case["rows"], case["cols"]))
    flops = case["count"] * STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)
    elements = case["count"] * m * n
    return {"bytes": 4 * elements * (2 if case["op"] == "ns" else 5), "flops": flops}
