"""Routing to experts (``ops.expert_route``) and the plan of the chosen pairs against the float64 oracle.

The index has to be equal.  Weights (u = 2^-24): a score's exponent x - top is rounded once (|x| u
relative in the score), exp and the reciprocal are within 4 u, the sum of a lane's scores and of its
neighbours' has at most 64 + 6 roundings, the sum of the chosen ones top_k, and quotient, scale and
product 4: u (span + 80 + top_k) relative, span the largest |logit - top| chosen; then the rounding to
the logits' type.
"""

import math

import pytest
import torch

from oracle import experts as O
from strata_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0**-24


def _logits(T, E, dtype, seed, masked=0.0, ties=False):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(T, E, generator=g) * 2
    if ties:
        l = torch.round(l)
    if masked:
        l[torch.rand(T, E, generator=g) < masked] = -math.inf
        l[::7] = -math.inf  # rows with nothing left
        l[1::11, :1] = math.nan
        l[2::13, -1:] = math.inf
        l[3::17] = torch.finfo(dtype).min  # the type's lowest value is a logit like others
    return l.to(dtype)


def _check(l, kw, got, gpu_weights_dtype):
    w, i = got
    ww, wi = O.route(l, **kw)
    assert i.dtype == torch.int32 and w.dtype == gpu_weights_dtype
    assert torch.equal(i.cpu().view(wi.shape), wi)
    ok = torch.isfinite(l.double())
    lo = torch.where(ok, l.double(), 0.0)
    span = (lo.gather(1, wi.clamp_min(0).long()) - torch.where(ok, l.double(), -math.inf).amax(1, keepdim=True).nan_to_num(0, 0, 0)).abs()
    span = torch.minimum(span.amax(1, keepdim=True), torch.tensor(120.0, dtype=torch.float64))  # beyond, the score is 0
    half = 2.0**-8 if w.dtype == torch.bfloat16 else U
    tol = ww * (U * (span + 80 + kw["top_k"]) + half) + 1e-37
    assert ((w.cpu().double().view(ww.shape) - ww).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 5, 5), (63, 8, 1), (65, 9, 4), (257, 16, 2), (130, 24, 3),
                                   (31, 33, 7), (200, 64, 8), (33, 65, 6), (17, 128, 8), (40, 200, 5), (9, 300, 64),
                                   (5, 512, 10)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(gpu, T, E, k, score, dtype):
    print(f"route {T} {E} {k} {score} {dtype}", flush=True)
    for seed, masked, ties, renorm in ((0, 0.0, False, True), (1, 0.3, False, False), (2, 0.0, True, False), (3, 0.5, True, True)):
        l = _logits(T, E, dtype, seed, masked, ties)
        kw = dict(top_k=k, score=score, renormalize=renorm, scale=1.5)
        _check(l, kw, ops.expert_route(l.to(gpu), **kw), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,groups,top", [(70, 8, 2, 4, 2), (33, 24, 3, 2, 1), (129, 64, 8, 8, 4), (11, 60, 6, 20, 3),
                                              (40, 96, 4, 4, 4), (7, 192, 8, 8, 3), (5, 512, 16, 64, 8), (3, 6, 1, 6, 1)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_bias_and_groups(gpu, T, E, k, groups, top, with_bias, dtype):
    print(f"route {T} {E} {k} groups {groups}/{top} bias {with_bias} {dtype}", flush=True)
    g = torch.Generator().manual_seed(9)
    bias = torch.randn(E, generator=g) * 0.3 if with_bias else None
    if with_bias:
        bias[E // 2] = math.nan  # masks its expert
        bias[0] = -5.0
    for score, masked, ties in (("sigmoid", 0.0, False), ("softmax", 0.3, False), ("sigmoid", 0.2, True)):
        l = _logits(T, E, dtype, 4, masked, ties)
        kw = dict(top_k=k, score=score, bias=bias, groups=groups, top_groups=top, renormalize=True, scale=2.5)
        lm = l.clone()
        if with_bias:
            lm[:, E // 2] = -math.inf
        got = ops.expert_route(l.to(gpu), k, score, bias.to(gpu) if with_bias else None, groups, top, True, 2.5)
        _check(lm, kw, got, dtype)


@pytest.mark.parametrize("T,E,k,groups,top", [(70, 512, 16, 64, 8), (37, 512, 64, 512, 100), (75, 256, 8, 8, 4), (66, 320, 6, 160, 9)])
def test_route_many_experts_in_groups(gpu, T, E, k, groups, top):
    """Every token of a workgroup whose scratch is at its largest."""
    print(f"route {T} {E} {k} groups {groups}/{top}", flush=True)
    l = _logits(T, E, torch.float32, 8)
    kw = dict(top_k=k, score="sigmoid", bias=torch.randn(E, generator=torch.Generator().manual_seed(3)), groups=groups, top_groups=top)
    _check(l, kw, ops.expert_route(l.to(gpu), **dict(kw, bias=kw["bias"].to(gpu))), torch.float32)


def test_route_near_ties_are_told_apart(gpu):
    """Keys s + bias whose difference a 32-bit sum loses: 64 bits choose, in either order."""
    l = torch.zeros(2, 8)
    l[:, 1] = 1e-8
    l[1] = l[1].flip(0)
    b = torch.zeros(8)
    for bias in (b, b + 3.0):
        _, i = ops.expert_route(l.to(gpu), 1, "sigmoid", bias.to(gpu))
        assert i.flatten().tolist() == [1, 6]


def test_route_layouts_and_leading_dims(gpu):
    """Rows inside a wider tensor, an odd first element, a transposed view, leading dimensions, no tokens."""
    big = _logits(40, 50, torch.float32, 5)
    l = big[:, 3:27].clone()
    want = O.route(l, 4)
    views = [big.to(gpu)[:, 3:27], l.t().contiguous().to(gpu).t(), l.view(4, 2, 5, 24).to(gpu)]
    for v in views:
        w, i = ops.expert_route(v, 4)
        assert tuple(w.shape) == (*v.shape[:-1], 4)
        assert torch.equal(i.cpu().view(-1, 4), want[1])
        assert (w.cpu().double().view(-1, 4) - want[0]).abs().max() <= 100 * U
    row = l[:1].to(gpu).expand(5, 24)
    w, i = ops.expert_route(row, 4)
    assert torch.equal(i.cpu(), want[1][:1].expand(5, 4))
    w, i = ops.expert_route(l[0].to(gpu), 4)
    assert i.cpu().tolist() == want[1][0].tolist()
    w, i = ops.expert_route(torch.zeros(0, 3, 8, device=gpu), 2)
    assert tuple(w.shape) == tuple(i.shape) == (0, 3, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (65, 24, 3), (50, 64, 8), (21, 100, 4), (6, 300, 9)])
def test_route_gradient(gpu, T, E, k, score, renorm, dtype):
    """Against the differentiated oracle.  ds has roundings of the scores (as the weights), of a / S
    and of their difference, whose terms may cancel: u (span + 100 + 2 top_k) of c (|dw| + |a| / S), times s
    (and 1 - s); the softmax's sum of s ds likewise."""
    print(f"route gradient {T} {E} {k} {score} {renorm} {dtype}", flush=True)
    l = _logits(T, E, dtype, 6, 0.2)
    l[3::17] = 1.0  # the oracle's softmax takes exp of the logits themselves
    g = torch.Generator().manual_seed(7)
    dw = torch.randn(T, k, generator=g).to(dtype)
    x = l.to(gpu).requires_grad_()
    w, i = ops.expert_route(x, k, score, renormalize=renorm, scale=1.5)
    (dl,) = torch.autograd.grad(w, x, dw.to(gpu))
    l64 = torch.where(torch.isfinite(l.double()), l.double(), math.nan).requires_grad_()
    (want,) = torch.autograd.grad(O.route_weights(l64, i.cpu(), score, renorm, 1.5), l64, dw.double())
    want = want.nan_to_num(0.0)
    s, ok = O.scores(l, score)
    have = i.cpu() >= 0
    sel = s.gather(1, i.cpu().clamp_min(0).long()) * have
    S = sel.sum(1, keepdim=True) if renorm else torch.ones(T, 1, dtype=torch.float64)
    S = torch.where(S > 0, S, 1.0)
    a = (dw.double().abs() * sel).sum(1, keepdim=True)
    mag = 1.5 / S * (torch.zeros(T, E, dtype=torch.float64).scatter_add_(1, i.cpu().clamp_min(0).long(), dw.double().abs() * have)
                     + a / S)
    mag = s * (mag + (1.5 / S * 2 * a if score == "softmax" else 0))
    half = 2.0**-8 if dtype == torch.bfloat16 else U
    tol = U * (30 + 100 + 2 * k) * mag + half * want.abs() + 1e-37
    assert ((dl.cpu().double() - want).abs() <= tol).all()
    assert (dl.cpu()[~ok] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_gradient_of_nothing(gpu, score, dtype):
    """Renormalised weights of one chosen expert are constant, and equal gradients move nothing: zeros, not
    the roundings of the gradients."""
    l = _logits(70, 24, dtype, 9, 0.3).to(gpu)
    dw = torch.randn(70, 1, generator=torch.Generator().manual_seed(1)).to(dtype).to(gpu)
    for k in (1, 4):
        x = l.clone().requires_grad_()
        w, _ = ops.expert_route(x, k, score, renormalize=True, scale=2.5)
        assert not torch.autograd.grad(w, x, dw.expand(70, k))[0].any()


def test_route_repeats_and_replays(gpu):
    l = _logits(1000, 64, torch.float32, 8).to(gpu)
    b = (torch.randn(64, generator=torch.Generator().manual_seed(1)) * 0.1).to(gpu)
    call = lambda: ops.expert_route(l, 8, "sigmoid", b, 8, 4)  # noqa: E731
    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        again = call()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(want, got, again))


@pytest.mark.parametrize("tile", [16, 64, 256])
@pytest.mark.parametrize("n,E", [(0, 3), (1, 1), (2, 8), (63, 5), (64, 64), (65, 2), (1000, 100), (1024, 512), (1025, 8), (1026, 512), (2048, 24), (2049, 200), (4050, 24), (4096, 100), (4097, 100),
                                 (5000, 1), (4097, 300), (70000, 24), (40000, 512), (70000, 512)])
def test_plan(gpu, n, E, tile):
    """Rows sorted by expert, stable; offsets and tiles; indices that name no expert left out."""
    print(f"plan {n} {E} {tile}", flush=True)
    g = torch.Generator().manual_seed(n)
    k = next(d for d in (3, 2, 1) if n % d == 0)
    idx = (torch.rand(n, generator=g) ** 2 * E).int()
    idx[torch.rand(n, generator=g) < 0.1] = -1
    if n > 4:
        idx[3], idx[4] = E, 2**31 - 1
    w = torch.randn(n, generator=g).bfloat16()
    plan = ops._expert_plan(idx.view(-1, k).to(gpu), w.view(-1, k).to(gpu), E, tile).cpu()
    token, weight, slot_row, off = plan[:n], plan[n:2 * n].view(torch.float32), plan[2 * n:3 * n], plan[3 * n:3 * n + E + 1]
    tiles = plan[3 * n + E + 1:ops._plan_size(n, E, tile)]
    ok = (idx >= 0) & (idx < E)
    order = torch.where(ok, idx, E).sort(stable=True).indices[: int(ok.sum())]
    R = order.numel()
    assert torch.equal(token[:R].long(), order // k) and torch.equal(weight[:R], w[order].float())
    want = torch.full((n,), -1, dtype=torch.int32)
    want[order] = torch.arange(R, dtype=torch.int32)
    assert torch.equal(slot_row, want)
    count = torch.bincount(idx[ok].long(), minlength=E)
    assert torch.equal(off.long(), torch.cat([torch.zeros(1, dtype=torch.int64), count.cumsum(0)]))
    wt = [(e, int(off[e]) + r) for e in range(E) for r in range(0, int(count[e]), tile)]
    assert int(tiles[0]) == len(wt)
    assert tiles[1:1 + 2 * len(wt)].view(-1, 2).tolist() == [list(t) for t in wt]


def _far(base, E, dtype, seed):
    """Tokens whose logits lie near ``base``, every third one an ordinary one."""
    g = torch.Generator().manual_seed(seed)
    l = base + torch.randn(13, E, generator=g)
    l[::3] -= base
    return l.to(dtype)


FAR = [-18.0, -21.0, -25.0, -60.0, -86.0, -87.5, -88.2, -89.0, -92.0, -95.0, -100.0, -104.0, -110.0, -200.0, -700.0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("form", ["plain", "bias", "groups"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_tiny_scores(gpu, score, form, dtype):
    """Renormalised weights and their gradient where the chosen scores are small, denormal or 0 in 32 bits: the weights
    are exp(l - m) / sum, m the largest chosen logit, up to 1 + e^m in a sigmoid.  Roundings: as in test_route (80 + top_k) u
    and u of the exponent: |l - m|, or at most 25 where the scores' sum is above 2^-30 and they are taken as they are.
    The gradient w (dw - mean): 25 for the exponent, 70 each for the sums of w and of w dw, 2 top_k, and some ten
    of single operations, with |l - m| of at most 8: (240 + 2 top_k) u of w (|dw| + |dw of slot 0| + sum of w |dw|).
    The reference's own: a softmax's s (ds - sum of s ds) leaves 2^-53 of each |dw| where the sum cancels to 0.
    A softmax's chosen scores are small where its bias keeps it from the largest ones (here of two experts)."""
    for base in FAR:
        for E, k in ((8, 1), (8, 2), (24, 5), (64, 8), (132, 7)):
            l = _far(base, E, dtype, E)
            bias, groups, top = None, 1, 1
            if form == "groups":
                groups, top = E // 4, 2 + k // 4
            if form != "plain" or score == "softmax":
                bias = torch.zeros(E)
            if score == "softmax":
                l[:, E // 2: E // 2 + 2] = 0.0
                bias[E // 2: E // 2 + 2] = -5.0
            kw = dict(score=score, groups=groups, top_groups=top, renormalize=True, scale=2.5)
            ww, wi = O.route(l, k, bias=bias, **kw)
            x = l.to(gpu).requires_grad_()
            w, i = ops.expert_route(x, k, bias=bias.to(gpu) if bias is not None else None, **kw)
            what = (score, form, base, E, k)
            assert torch.equal(i.cpu(), wi), what
            lc = l.double().gather(1, wi.clamp_min(0).long())
            half = 2.0**-8 if dtype == torch.bfloat16 else U
            rel = U * ((lc - lc.amax(1, keepdim=True)).abs() + 25 + 80 + k) + half
            assert torch.isfinite(w).all(), what
            assert ((w.detach().cpu().double() - ww).abs() <= rel * ww + 1e-37).all(), what
            dw = torch.randn(13, k, generator=torch.Generator().manual_seed(k)).to(dtype)
            (dl,) = torch.autograd.grad(w, x, dw.to(gpu))
            l64 = l.double().requires_grad_()
            (want,) = torch.autograd.grad(O.route_weights(l64, wi, score, True, 2.5), l64, dw.double())
            d = dw.double().abs()
            mag = torch.zeros(13, E, dtype=torch.float64).scatter_add_(1, wi.long(), ww * (d + d[:, :1] + (ww * d).sum(1, keepdim=True) / 2.5))
            tol = U * (240 + 2 * k) * mag + half * want.abs() + 2.5 * 2.0**-50 * d.sum(1, keepdim=True) + 1e-37
            assert torch.isfinite(dl).all(), what
            assert ((dl.cpu().double() - want).abs() <= tol).all(), what


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_scores_that_are_zero_in_64_bits(gpu, score):
    """Logits so low that the scores are 0 in 64 bits too: an index, weights and gradients of 0."""
    for low in (-1e3, -1e4, -1e30, torch.finfo(torch.float32).min):
        l = torch.full((5, 8), low)
        bias = torch.zeros(8)
        if score == "softmax":
            l[:, 3], bias[3] = 0.0, -5.0
        x = l.to(gpu).requires_grad_()
        w, i = ops.expert_route(x, 2, score, bias.to(gpu), renormalize=True)
        assert i.tolist() == [[0, 1]] * 5 and not w.any(), low
        (dl,) = torch.autograd.grad(w, x, torch.ones_like(w) + torch.arange(2, device=gpu))
        assert not dl.any(), low


@pytest.mark.parametrize("E", [64, 132, 300, 512])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_near_ties_of_many_experts(gpu, score, E):
    """A bias that lifts every score to within a rounding of 1: all keys s + bias lie within 1.2e-7 of each
    other, and 64 bits choose."""
    for seed in range(12):
        l = _logits(1, E, torch.float32, seed)
        s, _ = O.scores(l, score)
        bias = (1.0 - s[0]).float()
        for groups, top in ((1, 1), (E // 4, 5)):
            _, want = O.route(l, 9, score, bias, groups, top)
            _, got = ops.expert_route(l.to(gpu), 9, score, bias.to(gpu), groups, top)
            assert torch.equal(got.cpu(), want), (seed, groups)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_route_bias_that_is_not_finite(gpu, bad):
    """It masks its expert as a logit would: never chosen, not in the softmax's sum, a gradient of 0."""
    l = _logits(40, 24, torch.float32, 10)
    bias = torch.zeros(24)
    bias[[5, 17]] = bad
    gone = l.clone()
    gone[:, [5, 17]] = -math.inf
    x, y = l.to(gpu).requires_grad_(), gone.to(gpu).requires_grad_()
    got = ops.expert_route(x, 4, "softmax", bias.to(gpu), renormalize=False)
    want = ops.expert_route(y, 4, "softmax", torch.zeros(24, device=gpu), renormalize=False)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not ((got[1] == 5) | (got[1] == 17)).any()
    d = torch.randn(40, 4, generator=torch.Generator().manual_seed(2)).to(gpu)
    gx, gy = torch.autograd.grad(got[0], x, d)[0], torch.autograd.grad(want[0], y, d)[0]
    assert torch.equal(gx, gy) and not gx[:, [5, 17]].any()
