"""Operators next to routed training, as a user of this framework times them.

Three kinds of case:

``balance``  ``ops.expert_balance``: the balance loss of the routing to experts, the z-loss of its
             logits and every expert's load; with ``train`` the gradient at the logits.
``ortho``    ``ops.orthogonalize``: the Newton-Schulz products that bring the singular values of a stack
             of matrices near 1.
``muon``     ``ops.muon_step``: one step of the Muon optimizer over the matrices of a model: momentum,
             orthogonalised update, decayed weights.

``own`` chooses between the framework's operators and their plain form in elementary torch.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _balance(tokens, experts, top_k, score="softmax", sequences=1, dtype="bf16", masked=0.0, train=True):
    """``tokens`` of all ``sequences`` together."""
    return dict(kind="balance", tokens=tokens, experts=experts, top_k=top_k, score=score, sequences=sequences, dtype=dtype,
                masked=masked, train=train)


def _ortho(count, rows, cols, dtype="bf16", rank=8):
    return dict(kind="ortho", count=count, rows=rows, cols=cols, dtype=dtype, rank=rank)


def _muon(dim, blocks, ratio=4.0, experts=0, dtype="bf16", master=False, nesterov=True, adjust="match_rms_adamw", decay=0.1):
    """The matrices of ``blocks`` transformer blocks ``dim`` wide; with ``experts`` their MLP is a stack of that many."""
    return dict(kind="muon", dim=dim, blocks=blocks, ratio=ratio, experts=experts, dtype=dtype, master=master, nesterov=nesterov,
                adjust=adjust, decay=decay)


def listed():
    return [
        # the load of a rollout tile of odd sides while a model is watched: no gradient, some experts masked
        dict(_balance(10125, 24, 3, masked=0.05, train=False), name="balance_watch"),
        # a small ragged batch: launches and the host
        dict(_balance(1350, 24, 3, masked=0.1), name="balance_small"),
        # a training batch of eight samples, each balanced by itself: sigmoid scores of 64 experts
        dict(_balance(65536, 64, 8, score="sigmoid", sequences=8, dtype="fp32"), name="balance_train"),
        # many tokens, few experts, the whole batch balanced together
        dict(_balance(262144, 8, 2), name="balance_tokens"),
        # one small projection: bound by launches
        dict(_ortho(1, 128, 128), name="ortho_one"),
        # a block's largest weight
        dict(_ortho(1, 3840, 960), name="ortho_fc"),
        # a stack of experts' weights of odd width in fp32
        dict(_ortho(24, 776, 384, dtype="fp32"), name="ortho_stack"),
        # the step of a narrow pixel-stage model in fp32: few, small matrices
        dict(_muon(128, 2, dtype="fp32"), name="muon_small"),
        # blocks whose MLPs are eight experts each
        dict(_muon(512, 4, ratio=2.0, experts=8, adjust="original"), name="muon_experts"),
        # bf16 weights rounded from fp32 masters
        dict(_muon(640, 6, master=True), name="muon_master"),
        # twelve blocks in bf16
        dict(_muon(960, 12), name="muon_bf16"),
        # fp32 weights of a mid-sized model
        dict(_muon(384, 6, dtype="fp32", nesterov=False), name="muon_fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["balance", "ortho", "muon"])
    if kind == "balance":
        experts = _log(rng, 2, 512)
        sequences = rng.choice([1, 1, 2, 3, 8, 16])
        per = _log(rng, 1, min(262144, 4194304 // experts) // sequences)
        return _balance(per * sequences, experts, rng.randint(1, min(8, experts)), rng.choice(["softmax", "sigmoid"]), sequences,
                        rng.choice(["bf16", "fp32"]), rng.choice([0.0, 0.05, 0.5]), rng.random() < 0.7)
    dtype = rng.choice(["bf16", "fp32"])
    if kind == "ortho":
        rows, cols = _log(rng, 1, 2400), _log(rng, 1, 2400)
        small = min(rows, cols)
        most = 4e11 / (15 * small * rows * cols + 5 * small**3)
        return _ortho(_log(rng, 1, max(1, min(32, most))), rows, cols, dtype, rng.randint(0, 12))
    dim = 8 * _log(rng, 2, 120)
    blocks = rng.randint(1, max(1, min(12, int(1.4e12 / (176 * dim**3)))))
    experts = rng.choice([0, 0, 4, 7]) if dim <= 480 else 0
    return _muon(dim, blocks, rng.choice([1.5, 2.0, 4.0]), experts, dtype, dtype == "bf16" and rng.random() < 0.5, rng.random() < 0.7,
                 rng.choice(["original", "match_rms_adamw"]), rng.choice([0.0, 0.1]))


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_balance(c, g):
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    logits = _randn(g, t, e) * 1.5 + _randn(g, e) * 0.7  # some experts are liked by all
    if c["masked"]:  # experts that a token may not take; every 50th token is padding and may take none
        off = torch.rand(t, e, generator=g, device="cuda") < c["masked"]
        off |= (torch.arange(t, device="cuda") % 50 == 49)[:, None]
        logits = logits.masked_fill(off, -math.inf)
    s = dict(logits=logits.to(_DTYPES[c["dtype"]]))
    top, index = s["logits"].float().sort(dim=1, descending=True, stable=True)
    s["index"] = index[:, :k].int().masked_fill(top[:, :k] == -math.inf, -1).contiguous()
    if c["train"]:  # what the two losses are weighed by
        s["logits"].requires_grad_()
        s["weights"] = [torch.tensor(w, device="cuda") for w in (1e-2, 1e-3)]
    return s


def _gradients(g, count, rows, cols, rank):
    """A gradient's rough look: some strong directions above noise, rows of different magnitudes."""
    x = _randn(g, count, rows, cols) * torch.exp(0.5 * _randn(g, count, rows, 1))
    if rank:
        x += _randn(g, count, rows, rank) @ _randn(g, count, rank, cols)
    return x * (torch.exp(_randn(g, count, 1, 1)) * 1e-3)


def _prepare_ortho(c, g):
    return dict(x=_gradients(g, c["count"], c["rows"], c["cols"], c["rank"]).to(_DTYPES[c["dtype"]]))


def _shapes(c):
    """(tensors, matrices in each, rows, columns) of the step's weights, by kind; single matrices have no stack."""
    d, h, e, n = c["dim"], int(c["dim"] * c["ratio"]), c["experts"], c["blocks"]
    return [(n, 0, 3 * d, d), (n, 0, d, d)] + ([(n, 0, e, d), (n, e, h, d), (n, e, d, h)] if e else [(n, 0, h, d), (n, 0, d, h)])


def _prepare_muon(c, g):
    """Weights of one kind are views of one buffer."""
    dt, groups = _DTYPES[c["dtype"]], []
    for n, e, rows, cols in _shapes(c):
        count = n * max(e, 1)
        p = _randn(g, count, rows, cols) * 0.02
        groups.append(dict(p=p.to(dt), g=_gradients(g, count, rows, cols, 8).to(dt), m=_gradients(g, count, rows, cols, 8) * 0.5,
                           master=p if c["master"] else None))
    s = dict(groups=groups)
    for k in ("p", "g", "m", "master"):
        s[k] = None if groups[0][k] is None else [
            v for q, (n, e, rows, cols) in zip(groups, _shapes(c)) for v in q[k].view(n, *([e] if e else []), rows, cols)]
    return s


def prepare(case, seed):
    s = {"balance": _prepare_balance, "ortho": _prepare_ortho, "muon": _prepare_muon}[case["kind"]](case, _gen(seed))
    s["case"] = case
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    c = state["case"]
    return {"balance": _run_balance, "ortho": _run_ortho, "muon": _run_muon}[c["kind"]](state, c)


def _run_balance(s, c):
    if own:
        from strata_amd import ops

        balance, z, load = ops.expert_balance(s["logits"], s["index"], c["score"], c["sequences"])
    else:
        balance, z, load = _plain_balance(s["logits"], s["index"], c)
    if not c["train"]:
        return balance, z, load
    return balance.detach(), z.detach(), load, torch.autograd.grad((balance, z), s["logits"], s["weights"])[0]


def _run_ortho(s, c):
    if own:
        from strata_amd import ops

        return ops.orthogonalize(s["x"])
    return _plain_ortho(s["x"]).to(s["x"].dtype)


_LR, _MOMENTUM, _EPS, _COEFFICIENTS = 3e-4, 0.95, 1e-7, (3.4445, -4.7750, 2.0315)


def _run_muon(s, c):
    if own:
        from strata_amd import ops

        ops.muon_step(s["p"], s["g"], s["m"], lr=_LR, momentum=_MOMENTUM, nesterov=c["nesterov"], weight_decay=c["decay"],
                      adjust=c["adjust"], masters=s["master"])
    else:
        [_plain_muon(q, c) for q in s["groups"]]
    return [{k: q[k] for k in ("p", "m", "master")} for q in s["groups"]]


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_balance(logits, index, c):
    """For each sequence, of n tokens that have an expert left: sum over experts of E load / (k n) * mean over its tokens of
    the score, normalised over the token's experts; the mean over sequences.  z: the mean over all tokens of the squared
    log-sum-exp of their logits."""
    t, e = logits.shape
    b, k = c["sequences"], c["top_k"]
    ok = torch.isfinite(logits.detach())
    some = ok.any(dim=1)
    low = logits.float().masked_fill(~ok, -1e30)
    top = low.detach().amax(dim=1, keepdim=True)
    lse = (torch.exp(low - top).sum(dim=1, keepdim=True).log() + top)[:, 0]
    if c["score"] == "sigmoid":  # normalised by way of its logarithm, which does not underflow
        low = torch.minimum(low, torch.zeros_like(low)) - torch.log1p(torch.exp(-low.abs()))
        low = low.masked_fill(~ok, -1e30)
        top = low.detach().amax(dim=1, keepdim=True)
    ex = torch.exp(low - top) * ok
    score = ex / ex.sum(dim=1, keepdim=True).clamp_min(1e-30)
    n = some.view(b, -1).sum(dim=1)
    row = torch.arange(b, device=logits.device).repeat_interleave(t // b)[:, None]
    load = torch.bincount(torch.where(index >= 0, row * e + index, b * e).reshape(-1), minlength=b * e + 1)[:-1].view(b, e)
    n1 = n.clamp_min(1).float()[:, None]
    mean = score.view(b, t // b, e).sum(dim=1) / n1
    each = (load * (e / k) / n1 * mean).sum(dim=1)
    balance = each.sum() / (n > 0).sum().clamp_min(1)
    z = (lse.masked_fill(~some, 0.0) ** 2).sum() / n.sum().clamp_min(1)
    return balance, z, load.sum(dim=0).int()


def _plain_ortho(x):
    """x / |x|, then five times a x + (b g + c g g) x with g = x x^T, of the matrix or, where it is taller than wide, of its
    transpose."""
    a, b, c = _COEFFICIENTS
    tall = x.shape[-2] > x.shape[-1]
    x = x.float().mT.contiguous() if tall else x.float()
    x = x / x.square().sum(dim=(-2, -1), keepdim=True).sqrt().clamp_min(_EPS)
    for _ in range(5):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT.contiguous() if tall else x


def _plain_muon(q, c):
    g, m = q["g"].float(), q["m"]
    m.copy_(_MOMENTUM * m + (1 - _MOMENTUM) * g)
    o = _plain_ortho(_MOMENTUM * m + (1 - _MOMENTUM) * g if c["nesterov"] else m)
    w = (q["p"] if q["master"] is None else q["master"]).float()
    w = w * (1 - _LR * c["decay"]) - _LR * _factor(c, *q["p"].shape[1:]) * o
    q["p"].copy_(w)
    if q["master"] is not None:
        q["master"].copy_(w)


def _factor(c, rows, cols):
    return 0.2 * math.sqrt(max(rows, cols)) if c["adjust"] == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _products(count, rows, cols):
    """Operations of five steps: two symmetric products, half of which follows from the other, and a full one."""
    m, n = min(rows, cols), max(rows, cols)
    return 5 * count * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    c = case
    if c["kind"] == "balance":
        t, e, k, b = c["tokens"], c["experts"], c["top_k"], 2 if c["dtype"] == "bf16" else 4
        # an exponential counts as one operation
        return {"bytes": t * (e * b * (2 if c["train"] else 1) + k * 4) + 4 * e + 8, "flops": t * e * (10 if c["train"] else 5)}
    w = 2 if c["dtype"] == "bf16" else 4
    if c["kind"] == "ortho":
        n = c["count"] * c["rows"] * c["cols"]
        return {"bytes": 2 * n * w, "flops": _products(c["count"], c["rows"], c["cols"])}
    groups = [(n * max(e, 1), rows, cols) for n, e, rows, cols in _shapes(c)]
    each = w + 8 + (w + 8 if c["master"] else 2 * w)  # the gradient, the momentum, the weights
    return {"bytes": each * sum(n * rows * cols for n, rows, cols in groups), "flops": sum(_products(*q) for q in groups)}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"balance": _exact_balance, "ortho": _exact_ortho, "muon": _exact_muon}[case["kind"]](s, case)


def _exact_balance(s, c):
    l, idx = s["logits"].detach().double(), s["index"].long()
    t, e = l.shape
    b, k, per = c["sequences"], c["top_k"], t // c["sequences"]
    ok = l > -math.inf
    live = ok.any(dim=1)
    lse = torch.where(live, torch.logsumexp(l, dim=1), 0.0)
    key = l if c["score"] == "softmax" else torch.where(ok, torch.nn.functional.logsigmoid(torch.where(ok, l, 0.0)), -math.inf)
    p = torch.softmax(key, dim=1).nan_to_num(0.0)
    full = [q for q in range(b) if live[q * per:(q + 1) * per].any()]
    load = torch.zeros(e, dtype=torch.int64, device="cuda")
    balance, dl = torch.zeros((), dtype=torch.float64, device="cuda"), torch.zeros_like(l)
    for q in full:
        at = slice(q * per, (q + 1) * per)
        n = int(live[at].sum())
        seen = idx[at][idx[at] >= 0].bincount(minlength=e)
        load += seen
        f = seen.double() * e / (k * n)
        balance += (f * p[at].sum(dim=0) / n).sum() / len(full)
        if c["train"]:
            d = p[at] * (f - p[at] @ f[:, None]) / (n * len(full))
            dl[at] = float(s["weights"][0].double()) * (d if c["score"] == "softmax" else d * torch.sigmoid(-l[at]).masked_fill(~ok[at], 0.0))
    many = max(int(live.sum()), 1)
    z = lse.square().sum() / many
    if not c["train"]:
        return balance, z, load.int()
    dl += float(s["weights"][1].double()) * 2 / many * lse[:, None] * torch.softmax(l, dim=1).nan_to_num(0.0)
    return balance, z, load.int(), dl


def _exact_matrix(x):
    """One matrix, in its own orientation: the products on the shorter side."""
    x = x / max(float(torch.linalg.norm(x)), _EPS)
    a, b, c = _COEFFICIENTS
    for _ in range(5):
        if x.shape[0] <= x.shape[1]:
            g = x @ x.T
            x = a * x + b * (g @ x) + c * (g @ (g @ x))
        else:
            g = x.T @ x
            x = a * x + b * (x @ g) + c * ((x @ g) @ g)
    return x


def _exact_ortho(s, c):
    return torch.stack([_exact_matrix(x.double()) for x in s["x"]])


def _exact_muon(s, c):
    out = []
    for q in s["groups"]:
        g = q["g"].double()
        m = 0.95 * q["m"].double() + 0.05 * g
        u = 0.95 * m + 0.05 * g if c["nesterov"] else m
        w = (q["p"] if q["master"] is None else q["master"]).double()
        f = _LR * _factor(c, *w.shape[1:])
        w = torch.stack([(1 - _LR * c["decay"]) * a - f * _exact_matrix(b) for a, b in zip(w, u)])
        out.append(dict(p=w, m=m, master=None if q["master"] is None else w))
    return out
