"""Operators of routed training, as a user of this framework times them.

Three kinds of case:

``route``    ``ops.expert_route``: scores of the experts, the choice of ``top_k`` for each token and
             their weights; with ``train`` the gradient at the logits.
``experts``  ``ops.expert_mlp``: the chosen experts' MLPs over all tokens and the weighted sum
             with the block's residual; with ``train`` every gradient.
``adamw``    ``ops.adamw_step``: one AdamW step over many tensors, states in 32 or in 8 bits, with
             the clipping of the gradients by their global norm.

``own`` chooses between the framework's operators and their plain form in elementary torch.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BLOCK = 256  # elements that share a scale of an 8-bit state


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _route(tokens, experts, top_k, score="softmax", bias=False, groups=1, top_groups=1, renormalize=True, scale=1.0,
           dtype="bf16", masked=0.0, train=False):
    return dict(kind="route", tokens=tokens, experts=experts, top_k=top_k, score=score, bias=bias, groups=groups,
                top_groups=top_groups, renormalize=renormalize, scale=scale, dtype=dtype, masked=masked, train=train)


def _experts(tokens, experts, top_k, dim, hidden, skew=0.5, dropped=0.0, biases=True, residual=True, train=False):
    return dict(kind="experts", tokens=tokens, experts=experts, top_k=top_k, dim=dim, hidden=hidden, skew=skew,
                dropped=dropped, biases=biases, residual=residual, train=train)


def _adamw(dim, blocks, ratio=4.0, extra=0, dtype="bf16", bits=32, master=False, clip=1.0, decay=0.1):
    """The tensors of ``blocks`` transformer blocks ``dim`` wide, and ``extra`` single tensors of odd sizes."""
    return dict(kind="adamw", dim=dim, blocks=blocks, ratio=ratio, extra=extra, dtype=dtype, bits=bits, master=master,
                clip=clip, decay=decay)


def listed():
    return [
        # the router of one column's token while a model is served: latency alone
        dict(_route(1, 8, 2), name="route_token"),
        # the router of a rollout tile of odd sides, weights as the softmax gives them, some experts masked
        dict(_route(10125, 24, 3, renormalize=False, masked=0.05), name="route_tile"),
        # the router of a training batch: 64 experts in 8 groups, balance bias, its gradient
        dict(_route(65536, 64, 8, score="sigmoid", bias=True, groups=8, top_groups=4, scale=2.5, dtype="fp32", train=True),
             name="route_train"),
        # one token through its experts: bound by reading their weights
        dict(_experts(1, 8, 2, 1024, 4096), name="experts_token"),
        # a small ragged batch over many narrow experts, padding tokens among it
        dict(_experts(1350, 24, 3, 384, 776, dropped=0.1), name="experts_ragged"),
        # the block's MLP of a rollout step on one face
        dict(_experts(32768, 8, 2, 1024, 2048), name="experts_rollout"),
        # training: a small batch with an uneven load
        dict(_experts(2000, 16, 2, 768, 1536, skew=1.0, train=True), name="experts_train_small"),
        # training: a full batch
        dict(_experts(16384, 8, 2, 1024, 4096, train=True), name="experts_train"),
        # the step of a narrow pixel-stage model in fp32: few, small tensors
        dict(_adamw(128, 2, extra=3, dtype="fp32"), name="adamw_small"),
        # the step of twelve blocks in bf16 with fp32 master weights
        dict(_adamw(960, 12, master=True), name="adamw_master"),
        # the same with states in 8 bits and no master weights, no clipping
        dict(_adamw(640, 12, extra=20, bits=8, clip=0.0), name="adamw_8bit"),
        # fp32 weights, 8-bit states, clipped
        dict(_adamw(384, 6, extra=9, dtype="fp32", bits=8), name="adamw_8bit_clip"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "experts", "experts", "adamw"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = rng.randint(2, 24)
        top_groups = rng.randint(1, groups)
        return _route(_log(rng, 1, min(65536, 4194304 // (groups * per))), groups * per, rng.randint(1, min(8, top_groups * per)),
                      rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, top_groups, rng.random() < 0.6,
                      rng.choice([1.0, 2.5]), rng.choice(["bf16", "fp32"]), rng.choice([0.0, 0.05, 0.5]), rng.random() < 0.5)
    if kind == "experts":
        experts = rng.randint(2, 40)
        top_k = rng.randint(1, min(4, experts))
        dim, hidden = 8 * _log(rng, 8, 128), 8 * _log(rng, 16, 512)
        train = rng.random() < 0.5
        most = 3.2e11 / ((3 if train else 1) * 4 * top_k * dim * hidden)
        return _experts(_log(rng, 1, max(2, min(32768, most))), experts, top_k, dim, hidden, round(rng.uniform(0, 1.5), 2),
                        rng.choice([0.0, 0.0, 0.1]), rng.random() < 0.8, rng.random() < 0.8, train)
    dim = 8 * _log(rng, 2, 128)
    blocks = rng.randint(1, max(1, min(12, int(1.2e8 / (12 * dim * dim)))))
    dtype = rng.choice(["bf16", "fp32"])
    return _adamw(dim, blocks, rng.choice([2.0, 4.0]), rng.randint(0, 60), dtype, rng.choice([32, 8]),
                  dtype == "bf16" and rng.random() < 0.5, rng.choice([0.0, 1.0]), rng.choice([0.0, 0.1]))


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_route(c, g):
    t, e = c["tokens"], c["experts"]
    logits = torch.randn(t, e, generator=g, device="cuda") * 1.5
    if c["masked"]:  # experts that a token may not take; every 50th token is padding and may take none
        off = torch.rand(t, e, generator=g, device="cuda") < c["masked"]
        off |= (torch.arange(t, device="cuda") % 50 == 49)[:, None]
        logits = logits.masked_fill(off, -math.inf)
    s = dict(logits=logits.to(_DTYPES[c["dtype"]]))
    s["bias"] = torch.randn(e, generator=g, device="cuda") * 0.05 if c["bias"] else None
    if c["train"]:
        s["dweights"] = torch.randn(t, c["top_k"], generator=g, device="cuda").to(s["logits"].dtype)
    return s


def _prepare_experts(c, g):
    t, e, k, d, h = (c[n] for n in ("tokens", "experts", "top_k", "dim", "hidden"))

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).bfloat16()

    s = dict(x=rnd(t, d), w1=rnd(e, h, d, std=d**-0.5), w2=rnd(e, d, h, std=h**-0.5))
    s["b1"], s["b2"] = (rnd(e, h, std=0.1), rnd(e, d, std=0.1)) if c["biases"] else (None, None)
    s["residual"] = rnd(t, d) if c["residual"] else None
    logits = torch.randn(t, e, generator=g, device="cuda") + c["skew"] * torch.randn(e, generator=g, device="cuda")
    top, index = logits.sort(dim=1, descending=True)
    s["weights"] = torch.softmax(top[:, :k], dim=1).bfloat16()
    drop = torch.rand(t, 1, generator=g, device="cuda") < c["dropped"]  # padding tokens take no expert
    s["index"] = index[:, :k].int().masked_fill(drop, -1).contiguous()
    if c["train"]:
        s["dout"] = rnd(t, d)
    return s


def _sizes(c):
    d, h = c["dim"], int(c["dim"] * c["ratio"])
    return [n for _ in range(c["blocks"]) for n in (3 * d * d, 3 * d, d * d, d, h * d, h, d * h, d)] + \
        [(k * k * 13 + 7 * k) % 40000 + 1 for k in range(c["extra"])]


def _prepare_adamw(c, g):
    """Every tensor is a view of one buffer of its kind, from a whole block of it on."""
    sizes, dt = _sizes(c), _DTYPES[c["dtype"]]
    starts, n = [], 0
    for k in sizes:
        starts.append(n)
        n += -(-k // _BLOCK) * _BLOCK
    first = torch.tensor(starts, device="cuda")
    at = torch.zeros(n, dtype=torch.int32, device="cuda")
    at[first] = 1
    of = at.cumsum(0).long() - 1  # which tensor an element belongs to
    valid = torch.arange(n, device="cuda") - first[of] < torch.tensor(sizes, device="cuda")[of]

    def views(flat, per=1):
        return [flat[a // per: a // per + -(-k // per)] for a, k in zip(starts, sizes)]

    def rnd(std):
        return torch.randn(n, generator=g, device="cuda").mul_(std).mul_(valid)

    p, grad = rnd(0.02), rnd(1.0)
    grad *= torch.exp(torch.randn(len(sizes), generator=g, device="cuda"))[of] * 0.01  # each tensor's own magnitude
    s = dict(p=p.to(dt), g=grad.to(dt), valid=valid, step=torch.full((1,), 20, dtype=torch.int64, device="cuda"))
    s["master"] = p if c["master"] else None
    m, v = rnd(0.004), rnd(0.01).square_()
    if c["bits"] == 8:
        s["m"], s["m_scale"] = _pack(m.double(), valid, 1)
        s["v"], s["v_scale"] = _pack(v.double(), valid, 0)
        s["m_scales"], s["v_scales"] = views(s["m_scale"], _BLOCK), views(s["v_scale"], _BLOCK)
    else:
        s["m"], s["v"] = m, v
        s["m_scales"] = s["v_scales"] = None
    s["params"], s["grads"], s["ms"], s["vs"] = (views(s[k]) for k in ("p", "g", "m", "v"))
    s["masters"] = views(s["master"]) if c["master"] else None
    return s


def prepare(case, seed):
    s = {"route": _prepare_route, "experts": _prepare_experts, "adamw": _prepare_adamw}[case["kind"]](case, _gen(seed))
    s["case"] = case
    if case.get("train"):
        for k in ("logits", "x", "weights", "w1", "b1", "w2", "b2", "residual"):
            if s.get(k) is not None:
                s[k].requires_grad_()
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    c = state["case"]
    return {"route": _run_route, "experts": _run_experts, "adamw": _run_adamw}[c["kind"]](state, c)


def _grads(out, s, names, dout):
    names = [n for n in names if s[n] is not None]
    return dict(zip(names, torch.autograd.grad(out, [s[n] for n in names], dout)))


def _run_route(s, c):
    if own:
        from strata_amd import ops

        weights, index = ops.expert_route(s["logits"], c["top_k"], c["score"], s["bias"], c["groups"], c["top_groups"],
                                          c["renormalize"], c["scale"])
    else:
        weights, index = _plain_route(s["logits"], s["bias"], c)
    if not c["train"]:
        return weights, index
    return weights.detach(), index, _grads(weights, s, ("logits",), s["dweights"])


def _run_experts(s, c):
    if own:
        from strata_amd import ops

        out = ops.expert_mlp(s["x"], s["weights"], s["index"], s["w1"], s["b1"], s["w2"], s["b2"], s["residual"])
    else:
        out = _plain_experts(s["x"], s["weights"], s["index"], s["w1"], s["b1"], s["w2"], s["b2"], s["residual"])
    if not c["train"]:
        return out
    return out.detach(), _grads(out, s, ("x", "weights", "w1", "b1", "w2", "b2", "residual"), s["dout"])


_LR, _BETAS, _EPS = 3e-4, (0.9, 0.95), 1e-8


def _run_adamw(s, c):
    if own:
        from strata_amd import ops

        norm = ops.adamw_step(s["params"], s["grads"], s["ms"], s["vs"], s["step"], lr=_LR, betas=_BETAS, eps=_EPS,
                              weight_decay=c["decay"], max_norm=c["clip"] or None, masters=s["masters"],
                              exp_avg_scales=s["m_scales"], exp_avg_sq_scales=s["v_scales"])
        m, v = s["m"], s["v"]
        if c["bits"] == 8:
            m, v = ops.adamw_state_values(m, s["m_scale"]), ops.adamw_state_values(v, s["v_scale"])
    else:
        norm, m, v = _plain_adamw(s, c)
    return dict(p=s["p"], m=m, v=v, master=s["master"], norm=norm, step=s["step"])


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_route(logits, bias, c):
    """Scores s (softmax over the experts that are not masked, or sigmoid); the key of an expert is s + bias (the logit
    where there is neither a bias nor a group), kept in 64 bits; the groups with the largest sums of their two best keys
    stay; the top_k largest keys of those (the lower index of two equal ones), -1 where too few are left."""
    t, e = logits.shape
    k, g = c["top_k"], c["groups"]
    l64 = logits.double()
    ok = torch.isfinite(l64)
    low = l64.masked_fill(~ok, -math.inf)
    if c["score"] == "softmax":
        top = low.amax(dim=1, keepdim=True)
        ex = torch.exp(low - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
        s = ex / ex.sum(dim=1, keepdim=True).clamp_min(1e-300)
    else:
        s = ok / (1 + torch.exp(-l64.masked_fill(~ok, 0.0)))
    with torch.no_grad():
        key = low if bias is None and g == 1 else (s + (0 if bias is None else bias.double())).masked_fill(~ok, -math.inf)
        if g > 1:
            best = key.view(t, g, -1).topk(2, dim=2).values
            rank = best[..., 0] + best[..., 1].masked_fill(best[..., 1] == -math.inf, 0.0)
            stay = torch.zeros_like(rank, dtype=torch.bool)
            stay.scatter_(1, rank.sort(dim=1, descending=True, stable=True).indices[:, : c["top_groups"]], True)
            key = key.masked_fill(~stay.repeat_interleave(e // g, dim=1), -math.inf)
        top, index = key.sort(dim=1, descending=True, stable=True)
        top, index = top[:, :k], index[:, :k]
        have = top > -math.inf
    w = s.gather(1, index) * have
    if c["renormalize"]:
        total = w.sum(dim=1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    return (w * c["scale"]).to(logits.dtype), torch.where(have, index, torch.full_like(index, -1)).int()


def _plain_experts(x, weights, index, w1, b1, w2, b2, residual):
    """out[t] = residual[t] + sum over s of weights[t, s] * (gelu(x[t] w1[e]^T + b1[e]) w2[e]^T + b2[e]), e = index[t, s];
    slots with index -1 add nothing.  Each expert's rows are gathered to one length for a batched product."""
    t, k = index.shape
    e = w1.shape[0]
    flat = index.reshape(-1).long()
    order = flat.sort(stable=True).indices
    count = torch.bincount(flat + 1, minlength=e + 1)
    cap = max(1, int(count[1:].max()))
    start = count.cumsum(0)[:-1]
    row = start[:, None] + torch.arange(cap, device=x.device)  # [E, cap]: an expert's slots, in order
    have = torch.arange(cap, device=x.device) < count[1:, None]
    slot = order[row.clamp_max(t * k - 1)]
    xe = x.float()[slot // k]
    z = torch.bmm(xe, w1.float().transpose(1, 2))
    if b1 is not None:
        z = z + b1.float()[:, None]
    h = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    y = torch.bmm(h, w2.float().transpose(1, 2))
    if b2 is not None:
        y = y + b2.float()[:, None]
    y = y * weights.float().reshape(-1)[slot][..., None] * have[..., None]
    out = torch.zeros(t, y.shape[2], device=x.device).index_add(0, (slot // k).reshape(-1), y.reshape(e * cap, -1))
    return (out if residual is None else out + residual.float()).bfloat16()


def _unpack(code, scale, signed):
    """What an 8-bit state stands for, in 64 bits: scale * (c/127)^2 with the code's sign, or scale * ((c+1)/256)^2."""
    c = code.view(-1, _BLOCK).double()
    r = c.abs() / 127 if signed else (c + 1) / 256
    return (torch.sign(c) * r * r if signed else r * r).mul_(scale.double()[:, None]).view(-1)


def _pack(x, valid, signed):
    """Codes and scales of a state: the largest magnitude of each block, rounded to 32 bits, is its scale; the code is
    the nearest one in the square root's domain."""
    b = x.view(-1, _BLOCK)
    scale = b.abs().amax(dim=1).float()
    r = torch.sqrt(b.abs() / torch.where(scale > 0, scale, torch.ones_like(scale)).double()[:, None])
    if signed:
        code = (torch.round(r * 127).clamp_(max=127) * torch.sign(b)).to(torch.int8)
    else:
        code = (torch.round(r * 256) - 1).clamp_(0, 255).to(torch.uint8)
    return code.view(-1) * valid, scale


def _plain_adamw(s, c):
    """m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2, p = p (1 - lr decay) - lr mh / (sqrt(vh) + eps); g times
    clip / (norm + 1e-6) where the norm of all gradients is over clip.  8-bit states in 64 bits, for the codes' borders."""
    wide = torch.float64 if c["bits"] == 8 else torch.float32
    s["step"] += 1
    t = s["step"].double()
    norm, coef = None, 1.0
    if c["clip"]:
        norm = s["g"].double().square().sum().sqrt().reshape(1)
        coef = (c["clip"] / (norm + 1e-6)).clamp(max=1.0).to(wide)
    g = s["g"].to(wide) * coef
    m, v = s["m"], s["v"]
    if c["bits"] == 8:
        m, v = _unpack(m, s["m_scale"], True), _unpack(v, s["v_scale"], False)
    m = m * _BETAS[0] + (1 - _BETAS[0]) * g
    v = (v * _BETAS[1] + (1 - _BETAS[1]) * g * g) * s["valid"]
    rate = (_LR / (1 - _BETAS[0]**t)).to(wide)
    denom = torch.sqrt(v) / torch.sqrt(1 - _BETAS[1]**t).to(wide) + _EPS
    p = (s["p"] if s["master"] is None else s["master"]).to(wide)
    p = p * (1 - _LR * c["decay"]) - rate * m / denom
    s["p"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    if c["bits"] == 8:
        for x, k, signed in ((m, "m", True), (v, "v", False)):
            code, scale = _pack(x, s["valid"], signed)
            s[k].copy_(code)
            s[k + "_scale"].copy_(scale)
        m, v = _unpack(s["m"], s["m_scale"], True).float(), _unpack(s["v"], s["v_scale"], False).float()
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
        m, v = s["m"], s["v"]
    return norm, m, v


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "route":
        t, e, k, b = c["tokens"], c["experts"], c["top_k"], 2 if c["dtype"] == "bf16" else 4
        # an exponential counts as one operation; one comparison an expert and chosen slot
        return {"bytes": t * (e * b * (2 if c["train"] else 1) + k * (b + 4) + (k * b if c["train"] else 0)) + 4 * e * c["bias"],
                "flops": t * e * (4 + k + (4 if c["train"] else 0))}
    if c["kind"] == "experts":
        t, e, k, d, h = (c[n] for n in ("tokens", "experts", "top_k", "dim", "hidden"))
        rows = max(1.0, t * k * (1 - c["dropped"]))
        params = min(e, rows) * (2 * h * d + (h + d) * c["biases"])
        act = t * (d * (2 + c["residual"]) + k) * 2 + t * k * 4
        if not c["train"]:
            return {"bytes": 2 * params + act, "flops": 4 * rows * d * h}
        grads = 2 * (e * (2 * h * d + (h + d) * c["biases"]) + t * (d * (2 + c["residual"]) + k))
        return {"bytes": 2 * params + act + grads, "flops": 12 * rows * d * h}
    n = sum(_sizes(c))
    w = 2 if c["dtype"] == "bf16" else 4
    state = 2 * (4 * 4 if c["bits"] == 32 else 2 * (1 + 4 / _BLOCK) + 4)  # read and written; in 8 bits also the values
    each = w + (w + 8 if c["master"] else 2 * w) + (16 if c["bits"] == 32 else 4 * (1 + 4 / _BLOCK) + 8)
    return {"bytes": n * each, "flops": n * 16}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "experts": _exact_experts, "adamw": _exact_adamw}[case["kind"]](s, case)


def _exact_route(s, c):
    l = s["logits"].detach().double()
    t, e = l.shape
    ok = l > -math.inf
    if c["score"] == "softmax":
        score = torch.softmax(torch.where(ok, l, -math.inf), dim=1).nan_to_num(0.0)
    else:
        score = torch.sigmoid(l) * ok
    bias = torch.zeros(e, dtype=torch.float64, device="cuda") if s["bias"] is None else s["bias"].double()
    key = torch.where(ok, l if s["bias"] is None and c["groups"] == 1 else score + bias, -math.inf)
    left = torch.ones(t, e, dtype=torch.bool, device="cuda")
    if c["groups"] > 1:  # one group after the other: the first of the largest
        by = key.reshape(t, c["groups"], -1).sort(dim=2, descending=True).values
        two = by[:, :, 0] + torch.where(by[:, :, 1] > -math.inf, by[:, :, 1], 0.0)
        left = torch.zeros(t, c["groups"], dtype=torch.bool, device="cuda")
        for _ in range(c["top_groups"]):
            at = _first_max(two.masked_fill(left, -math.inf), ~left)
            left[torch.arange(t, device="cuda"), at] = True
        left = left[:, :, None].expand(t, c["groups"], e // c["groups"]).reshape(t, e)
    left = left & ok
    chosen = []
    for _ in range(c["top_k"]):
        at = _first_max(torch.where(left, key, -math.inf), left)
        some = left.any(dim=1)
        chosen.append(torch.where(some, at, -1))
        left[torch.arange(t, device="cuda"), at] = False
    index = torch.stack(chosen, dim=1)
    have = index >= 0
    sel = score.gather(1, index.clamp_min(0)) * have
    total = sel.sum(dim=1, keepdim=True) if c["renormalize"] else torch.ones(t, 1, dtype=torch.float64, device="cuda")
    total = torch.where(total > 0, total, 1.0)
    w = c["scale"] * sel / total
    if not c["train"]:
        return w, index.int()
    dw = s["dweights"].double() * have
    ds = c["scale"] / total * (dw - (dw * sel).sum(dim=1, keepdim=True) / total if c["renormalize"] else dw) * have
    full = torch.zeros_like(score).scatter_add_(1, index.clamp_min(0), ds)
    if c["score"] == "softmax":
        dl = score * (full - (score * full).sum(dim=1, keepdim=True))
    else:
        dl = full * score * (1 - score)
    return w, index.int(), dict(logits=dl)


def _first_max(key, allowed):
    """The lowest index of the largest allowed key of each row."""
    top = key.masked_fill(~allowed, -math.inf).amax(dim=1, keepdim=True)
    return ((key == top) & allowed).int().argmax(dim=1)


def _exact_experts(s, c):
    x, w, idx, w1, w2 = s["x"].double(), s["weights"].double(), s["index"], s["w1"], s["w2"]
    train, t, k = c["train"], c["tokens"], c["top_k"]
    out = torch.zeros_like(x) if s["residual"] is None else s["residual"].double().clone()
    if train:
        do = s["dout"].double()
        gr = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("x", "weights", "w1", "b1", "w2", "b2")
              if s[n] is not None}
        if s["residual"] is not None:
            gr["residual"] = do.clone()
    u0 = math.sqrt(2 / math.pi)
    for e in range(c["experts"]):
        tok, slot = (idx == e).nonzero(as_tuple=True)
        if not tok.numel():
            continue
        a, b = w1[e].double(), w2[e].double()
        z = x[tok] @ a.T + (s["b1"][e].double() if s["b1"] is not None else 0)
        th = torch.tanh(u0 * (z + 0.044715 * z**3))
        h = 0.5 * z * (1 + th)
        y = h @ b.T + (s["b2"][e].double() if s["b2"] is not None else 0)
        we = w[tok, slot][:, None]
        out.index_add_(0, tok, we * y)
        if train:
            dy = do[tok]
            gr["weights"][tok, slot] = (dy * y).sum(dim=1)
            dy = we * dy
            gr["w2"][e] = dy.T @ h
            dz = (dy @ b) * (0.5 * (1 + th) + 0.5 * z * (1 - th * th) * u0 * (1 + 3 * 0.044715 * z * z))
            gr["w1"][e] = dz.T @ x[tok]
            gr["x"].index_add_(0, tok, dz @ a)
            if s["b1"] is not None:
                gr["b1"][e], gr["b2"][e] = dz.sum(dim=0), dy.sum(dim=0)
    return (out, gr) if train else out


def _exact_adamw(s, c):
    g, t = s["g"].double(), 21
    norm = math.sqrt(float((g * g).sum()))
    if c["clip"] and norm > c["clip"] - 1e-6:
        g = g * (c["clip"] / (norm + 1e-6))
    if c["bits"] == 8:
        lm, lv = s["m"].double() / 127, (s["v"].double() + 1) / 256
        m0 = lm * lm.abs() * s["m_scale"].double().repeat_interleave(_BLOCK)
        v0 = lv * lv * s["v_scale"].double().repeat_interleave(_BLOCK)
    else:
        m0, v0 = s["m"].double(), s["v"].double()
    m, v = 0.9 * m0 + (1 - 0.9) * g, torch.where(s["valid"], 0.95 * v0 + (1 - 0.95) * g * g, 0.0)
    p = s["p"].double() if s["master"] is None else s["master"].double()
    step = (m / (1 - 0.9**t)) / ((v / (1 - 0.95**t)).sqrt() + _EPS)
    p = p - _LR * c["decay"] * p - _LR * step
    if c["bits"] == 8:  # the nearest of all values that a code can stand for, in the root's domain
        roots = torch.arange(0, 128, device="cuda", dtype=torch.float64) / 127
        m = _nearest(m.abs(), roots, s["valid"]) * m.sign()
        v = _nearest(v, torch.arange(1, 257, device="cuda", dtype=torch.float64) / 256, s["valid"])
    return dict(p=p, m=m, v=v, master=None if s["master"] is None else p,
                norm=torch.tensor([norm], dtype=torch.float64) if c["clip"] else None, step=s["step"] + 1)


def _nearest(x, roots, valid):
    scale = x.view(-1, _BLOCK).amax(dim=1).float().double().repeat_interleave(_BLOCK)
    r = (x / scale.clamp_min(1e-300)).sqrt()
    at = torch.bucketize(r, (roots[1:] + roots[:-1]) / 2)
    return torch.where(valid, roots[at], roots[0]).square() * scale
