"""The experts' MLPs (``ops.expert_mlp``) against the float64 oracle, every output inside the bound that the
oracle derives from its operands (oracle/experts.py: bf16 operands, fp32 sums)."""

import math

import pytest
import torch

from oracle import experts as O
from strata_amd import ops

from .conftest import rel_l2

pytestmark = pytest.mark.gpu
NAMES = ("x", "weights", "w1", "b1", "w2", "b2", "residual")


def _case(T, E, k, C, H, N, seed, biases=True, residual=True, dropped=0.1, skew=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).bfloat16()  # noqa: E731
    c = dict(x=r(T, C), w1=r(E, H, C, std=C**-0.5), w2=r(E, N, H, std=H**-0.5), b1=r(E, H, std=0.2) if biases else None,
             b2=r(E, N, std=0.2) if biases else None, residual=r(T, N) if residual else None, dout=r(T, N))
    c["weights"] = torch.rand(T, k, generator=g).bfloat16()
    logits = torch.randn(T, E, generator=g) + skew * torch.randn(E, generator=g)
    idx = torch.stack([logits.argsort(1, descending=True)[:, s % E] for s in range(k)], 1).int()
    idx[torch.rand(T, k, generator=g) < dropped] = -1
    c["index"] = idx
    return c


def _to(c, gpu, train):
    out = {n: t.to(gpu) if t is not None else None for n, t in c.items()}
    if train:
        for n in NAMES:
            if out[n] is not None:
                out[n].requires_grad_()
    return out


def _call(d):
    return ops.expert_mlp(d["x"], d["weights"], d["index"], d["w1"], d["b1"], d["w2"], d["b2"], d["residual"])


def _inside(got, want, what):
    value, bound = want
    diff = (got.detach().cpu().double().view(value.shape) - value).abs()
    assert torch.isfinite(got).all(), what
    assert (diff <= bound).all(), (what, float((diff / bound).max()))
    # the bound adds every rounding up; on the whole they cancel: two roundings to bf16 of random sign
    if value.numel() > 1000:
        assert rel_l2(got.detach().view(value.shape), value) <= 2.0**-8, what


SHAPES = [
    # tokens, experts, top_k, dim, hidden, out_dim
    (1, 1, 1, 8, 8, 8), (1, 8, 2, 64, 128, 64), (3, 4, 3, 72, 40, 24), (64, 2, 1, 64, 64, 64), (65, 3, 2, 136, 72, 200),
    (130, 5, 2, 64, 264, 64), (200, 24, 3, 104, 56, 96), (300, 2, 2, 128, 256, 128), (513, 3, 1, 264, 136, 520),
    (90, 70, 2, 32, 40, 24), (700, 4, 2, 96, 640, 96), (40, 64, 4, 32, 48, 32), (1500, 3, 2, 192, 128, 64),
    # 128 x 128 tiles with a ring of four stages and of two
    (700, 40, 2, 640, 520, 552), (2600, 8, 2, 1032, 1040, 1048),
    # 256 x 256 tiles, several a workgroup, ragged in every direction
    (26000, 3, 2, 264, 328, 296),
    # few tiles of the weights' gradients: their rows shared out, an expert's share empty or not whole
    (600, 1, 1, 72, 40, 24), (1700, 4, 2, 264, 72, 136), (5000, 2, 1, 64, 520, 200),
    # the same with a last round in 64 x 64 tiles, and in 128 x 128 ones
    (34000, 2, 2, 136, 72, 200), (40000, 2, 2, 136, 264, 200),
]


@pytest.mark.parametrize("T,E,k,C,H,N", SHAPES)
def test_forward_and_gradients(gpu, T, E, k, C, H, N):
    print(f"experts {T} {E} {k} {C} {H} {N}", flush=True)
    for seed, biases, residual in ((1, True, True), (2, False, False)):
        c = _case(T, E, k, C, H, N, seed, biases, residual)
        want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual", "dout")))
        with torch.no_grad():
            _inside(_call(_to(c, gpu, False)), want["out"], "inference")
        d = _to(c, gpu, True)
        out = _call(d)
        _inside(out, want["out"], "out")
        names = [n for n in NAMES if d[n] is not None]
        grads = torch.autograd.grad(out, [d[n] for n in names], d["dout"])
        for n, g in zip(names, grads):
            assert g.shape == d[n].shape and g.dtype == torch.bfloat16
            _inside(g, want[n], n)


@pytest.mark.parametrize("T,E,k,C,H,N", [(1, 4, 2, 1032, 4096, 1032), (5, 8, 2, 256, 1160, 72), (2, 3, 3, 2048, 24, 8),
                                         (17, 8, 4, 40, 1096, 200), (33, 40, 2, 512, 64, 1024), (20, 2, 1, 64, 136, 64)])
def test_few_rows(gpu, T, E, k, C, H, N):
    """Inference with a handful of rows an expert: contractions split over the waves of a workgroup."""
    print(f"experts, few rows {T} {E} {k} {C} {H} {N}", flush=True)
    c = _case(T, E, k, C, H, N, 14, dropped=0.05)
    want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual")))
    d = _to(c, gpu, False)
    out = _call(d)
    _inside(out, want["out"], "out")
    assert torch.equal(out, _call(d))
    d = dict(d, b1=None, b2=None, residual=None)
    want = O.mlp_bounds(c["x"], c["weights"], c["index"], c["w1"], None, c["w2"], None, None)
    _inside(_call(d), want["out"], "plain")


def test_few_rows_of_one_expert(gpu):
    """17 tokens that all choose one of 8: a whole tile of 16 rows and one of a single row."""
    c = _case(17, 8, 1, 80, 1032, 48, 17)
    c["index"] = torch.full_like(c["index"], 5)
    want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual")))
    _inside(_call(_to(c, gpu, False)), want["out"], "out")


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (16, 3, 1), (4, 40, 4), (1, 2, 16), (8, 1, 2), (5, 512, 3),
                                   (1, 3, 1), (4, 2, 1), (1, 9, 3), (2, 5, 2), (1, 2, 4), (3, 1, 1)])
def test_up_to_16_pairs(gpu, T, E, k):
    """Served without a plan: the same expert in several slots, indexes outside the range, weights of zero."""
    for seed, picks in ((18, None), (19, 0), (20, -1), (21, E)):
        c = _case(T, E, k, 72, 1040, 136, seed)
        if E < k:
            g = torch.Generator().manual_seed(seed)
            c["index"] = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
        if picks is not None:
            c["index"].view(-1)[:: 2] = picks
            c["weights"].view(-1)[1::3] = 0.0
        want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual")))
        d = _to(c, gpu, False)
        out = _call(d)
        _inside(out, want["out"], (T, E, k, picks))
        with torch.enable_grad():  # the planned products give the same up to the contraction's order
            planned = _call(dict(d, x=d["x"].clone().requires_grad_()))
        _inside(planned.detach(), want["out"], (T, E, k, picks, "planned"))


def test_nothing_chosen_and_unused_experts(gpu):
    c = _case(70, 6, 2, 64, 72, 64, 3)
    c["index"][:] = -1
    d = _to(c, gpu, True)
    out = _call(d)
    assert torch.equal(out, d["residual"])
    grads = dict(zip(NAMES, torch.autograd.grad(out, [d[n] for n in NAMES], d["dout"])))
    for n in NAMES[:-1]:
        assert (grads[n] == 0).all(), n
    assert torch.equal(grads["residual"], d["dout"])
    c["index"][:] = torch.tensor([4, 9])  # one expert for all, and one that does not exist
    d = _to(c, gpu, True)
    want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual", "dout")))
    out = _call(d)
    _inside(out, want["out"], "out")
    for n, g in zip(NAMES, torch.autograd.grad(out, [d[n] for n in NAMES], d["dout"])):
        _inside(g, want[n], n)
    for n in ("w1", "b1", "w2", "b2"):
        assert (torch.autograd.grad(_call(d), d[n], d["dout"])[0][[0, 1, 2, 3, 5]] == 0).all()


def test_no_tokens(gpu):
    c = _case(0, 3, 2, 16, 24, 16, 4)
    d = _to(c, gpu, True)
    out = _call(d)
    assert tuple(out.shape) == (0, 16)
    for n, g in zip(NAMES, torch.autograd.grad(out, [d[n] for n in NAMES], d["dout"])):
        assert g.shape == d[n].shape and (g == 0).all()


def test_the_same_expert_twice(gpu):
    """Two slots of one expert are two rows: as one slot with the weights' sum."""
    c = _case(90, 3, 2, 64, 64, 64, 5, dropped=0.0)
    c["index"][:, 1] = c["index"][:, 0]
    want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual", "dout")))
    d = _to(c, gpu, True)
    out = _call(d)
    _inside(out, want["out"], "out")
    for n, g in zip(NAMES, torch.autograd.grad(out, [d[n] for n in NAMES], d["dout"])):
        _inside(g, want[n], n)


@pytest.mark.parametrize("which", NAMES)
def test_one_gradient_alone(gpu, which):
    c = _case(150, 4, 2, 72, 80, 64, 6)
    want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual", "dout")))
    d = _to(c, gpu, False)
    d[which].requires_grad_()
    _inside(torch.autograd.grad(_call(d), d[which], d["dout"])[0], want[which], which)


def test_layouts(gpu):
    """Rows inside wider tensors, leading dimensions, weights and biases that are views, an expanded dout."""
    c = _case(60, 3, 2, 64, 48, 64, 7)
    want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual", "dout")))["out"]
    d = _to(c, gpu, False)

    def wide(t, pad):
        buf = torch.full((*t.shape[:-1], t.shape[-1] + pad), math.nan, dtype=t.dtype, device=gpu)
        buf[..., : t.shape[-1]] = t
        return buf[..., : t.shape[-1]]

    v = dict(d, x=wide(d["x"], 16), residual=wide(d["residual"], 8), w1=wide(d["w1"], 24), w2=d["w2"].transpose(1, 2).contiguous().transpose(1, 2),
             b1=wide(d["b1"], 1), weights=wide(d["weights"], 3))
    _inside(_call(v), want, "strided")
    odd = torch.empty(60 * 64 + 1, dtype=torch.bfloat16, device=gpu)[1:].view(60, 64)
    odd.copy_(d["x"])
    _inside(_call(dict(d, x=odd, residual=odd)), O.mlp_bounds(*(c[n] for n in NAMES[:2]), c["index"], *(c[n] for n in NAMES[2:6]), c["x"])["out"], "odd first element")
    lead = {n: (d[n].view(3, 4, 5, -1) if n in ("x", "weights", "index", "residual") else d[n]) for n in d}
    out = _call(lead)
    assert tuple(out.shape) == (3, 4, 5, 64)
    _inside(out, want, "leading")
    # one token for all rows, one residual, one expert's weights for all experts: their gradients are summed
    d = _to(c, gpu, False)
    leaves = [d["x"][:1].clone(), d["residual"][:1].clone(), d["w1"][:1].clone(), d["b2"][:1].clone()]
    for t in leaves:
        t.requires_grad_()
    e = dict(d, x=leaves[0].expand(60, 64), residual=leaves[1].expand(60, 64), w1=leaves[2].expand(3, 48, 64), b2=leaves[3].expand(3, 64))
    f = {n: t.detach().contiguous() for n, t in e.items()}
    for n in ("x", "residual", "w1", "b2"):
        f[n].requires_grad_()
    got = _call(e)
    assert torch.equal(got, _call(f))
    ge = torch.autograd.grad(got, leaves, d["dout"])
    gf = torch.autograd.grad(_call(f), [f[n] for n in ("x", "residual", "w1", "b2")], d["dout"])
    for a, b in zip(ge, gf):
        assert torch.equal(a, b.sum(0, keepdim=True))
    d = _to(c, gpu, True)
    ones = torch.ones((), device=gpu).bfloat16().expand(60, 64)
    full = torch.autograd.grad(_call(d), d["w2"], ones.contiguous())[0]
    assert torch.equal(torch.autograd.grad(_call(d), d["w2"], ones)[0], full)


def test_weights_of_zero(gpu):
    """A pair of weight 0 adds nothing to the output or the experts' gradients, and its weight has one."""
    c = _case(80, 3, 2, 64, 96, 64, 12, dropped=0.0)
    c["weights"][::3, 0] = 0.0
    c["weights"][5, 1] = -0.5
    c["index"][c["index"] == 2] = 1
    c["weights"][c["index"] == 1] = 0.0  # all rows of one expert
    want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual", "dout")))
    d = _to(c, gpu, True)
    out = _call(d)
    _inside(out, want["out"], "out")
    for n, g in zip(NAMES, torch.autograd.grad(out, [d[n] for n in NAMES], d["dout"])):
        _inside(g, want[n], n)
        if n in ("w1", "b1", "w2", "b2"):
            assert (g[1:] == 0).all(), n
    rows = (c["weights"] == 0).all(1)
    assert torch.equal(out.cpu()[rows], c["residual"][rows])


def test_masked_tokens_do_not_reach_others(gpu):
    """A dropped token's x may hold anything; an infinite one reaches its own row alone."""
    c = _case(100, 4, 2, 64, 64, 64, 8, dropped=0.0)
    c["index"][10] = -1
    d = _to(c, gpu, False)
    clean = _call(d)
    x = d["x"].clone()
    x[10] = math.nan
    assert torch.equal(_call(dict(d, x=x)), clean)
    x[20] = math.inf
    out = _call(dict(d, x=x))
    keep = [t for t in range(100) if t != 20]
    assert torch.equal(out[keep], clean[keep]) and not torch.isfinite(out[20]).all()


def test_repeats_bit_for_bit_and_order_of_tokens(gpu):
    c = _case(900, 5, 2, 128, 192, 128, 9)
    d = _to(c, gpu, True)
    names = list(NAMES)

    def both():
        out = _call(d)
        return [out, *torch.autograd.grad(out, [d[n] for n in names], d["dout"])]

    a, b = both(), both()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    perm = torch.randperm(900, generator=torch.Generator().manual_seed(1)).to(gpu)
    with torch.no_grad():  # a token's result does not depend on its place
        p = {n: (d[n][perm] if n in ("x", "weights", "index", "residual") else d[n]) for n in d}
        assert torch.equal(_call(p), a[0][perm])


def test_another_stream_and_graph(gpu):
    c = _case(333, 4, 2, 96, 128, 96, 10)
    d = _to(c, gpu, False)
    want = _call(d).clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _call(d)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _call(d)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        again = _call(d)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(again, want)


def test_offsets_past_32_bits(gpu):
    """2.2e9 hidden values: rows behind the 2^31st element, forward and backward, against the oracle at single
    tokens and, for the weights' gradients, against one half of the tokens at a time."""
    T, E, k, C, H, N = 270000, 2, 2, 64, 4096, 64
    g = torch.Generator(device=gpu).manual_seed(15)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=gpu) * std).bfloat16()  # noqa: E731
    d = dict(x=r(T, C), w1=r(E, H, C, std=C**-0.5), w2=r(E, N, H, std=H**-0.5), b1=r(E, H, std=0.2), b2=r(E, N, std=0.2),
             residual=None, dout=r(T, N), weights=torch.rand(T, k, generator=g, device=gpu).bfloat16())
    d["index"] = torch.randint(0, E, (T, k), generator=g, device=gpu, dtype=torch.int32)
    for n in NAMES[:-1]:
        d[n].requires_grad_()
    out = _call(d)
    names = list(NAMES[:-1])
    grads = dict(zip(names, torch.autograd.grad(out, [d[n] for n in names], d["dout"])))
    some = torch.cat([torch.arange(4), torch.randint(0, T, (40,), generator=torch.Generator().manual_seed(1)), torch.arange(T - 4, T)])
    c = {n: t.detach().cpu() if t is not None else None for n, t in d.items() if n in ("w1", "w2", "b1", "b2")}
    at = {n: d[n].detach()[some.to(gpu)].cpu() for n in ("x", "weights", "index", "dout")}
    want = O.mlp_bounds(at["x"], at["weights"], at["index"], c["w1"], c["b1"], c["w2"], c["b2"], None, at["dout"])
    pick = some.to(gpu)
    _inside(out[pick], want["out"], "out")
    for n in ("x", "weights"):
        _inside(grads[n][pick], want[n], n)
    parts = []
    for lo, hi in ((0, T // 2), (T // 2, T)):
        h = {n: (d[n].detach()[lo:hi] if n in ("x", "weights", "index", "dout") else d[n]) for n in d}
        parts.append(torch.autograd.grad(_call(h), [d[n] for n in names[2:]], h["dout"]))
    for n, a, b in zip(names[2:], *parts):  # each side rounded to bf16 once, at random
        assert rel_l2(grads[n].float(), a.float() + b.float()) <= 2.0**-8, n


def test_custom_ops_agree(gpu):
    """What a traced program calls: the same launches through torch.ops."""
    c = _case(90, 4, 2, 64, 72, 64, 13)
    d = _to(c, gpu, True)
    args = [d[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual")]
    out = torch.ops.strata_hip.expert_mlp_train(*args)[0]
    want = _call(d)
    assert torch.equal(out, want)
    for x, y in zip(torch.autograd.grad(out, [d[n] for n in NAMES], d["dout"]),
                    torch.autograd.grad(want, [d[n] for n in NAMES], d["dout"])):
        assert torch.equal(x, y)
    with torch.no_grad():
        assert torch.equal(torch.ops.strata_hip.expert_mlp_fwd(*args), want)
    l = torch.randn(50, 8, generator=torch.Generator().manual_seed(0)).to(gpu).requires_grad_()
    a, b = torch.ops.strata_hip.expert_route(l, 2), ops.expert_route(l, 2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    g = torch.ones_like(a[0])
    g[:, 0] = 2
    assert torch.equal(torch.autograd.grad(a[0], l, g)[0], torch.autograd.grad(b[0], l, g)[0])


def test_the_same_graph_twice(gpu):
    """A kept graph's second backward, after other calls, gives the first one's bits."""
    d = _to(_case(400, 4, 2, 64, 136, 72, 22), gpu, True)
    out = _call(d)
    leaves = [d[n] for n in NAMES]
    first = torch.autograd.grad(out, leaves, d["dout"], retain_graph=True)
    torch.autograd.grad(_call(d), leaves, 2 * d["dout"])
    again = torch.autograd.grad(out, leaves, d["dout"])
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_traced_by_a_compiler(gpu):
    """Forward and backward through torch.compile, x and w1 as transposed views."""
    d = _to(_case(90, 4, 2, 64, 72, 64, 14), gpu, False)
    d["x"] = d["x"].t().contiguous().t()
    d["w1"] = d["w1"].transpose(1, 2).contiguous().transpose(1, 2)
    for n in NAMES:
        d[n].requires_grad_()
    args = [d[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual")]
    want = ops.expert_mlp(*args)
    got = torch.compile(lambda *a: ops.expert_mlp(*a), backend="aot_eager", fullgraph=True)(*args)
    assert torch.equal(got, want)
    for x, y in zip(torch.autograd.grad(got, [d[n] for n in NAMES], d["dout"]), torch.autograd.grad(want, [d[n] for n in NAMES], d["dout"])):
        assert torch.equal(x, y)


def test_two_streams_at_once(gpu):
    """Two calls in flight with different choices: each has its own workspace."""
    cases = [_to(_case(2000, 8, 2, 128, 256, 128, s), gpu, True) for s in (15, 16)]

    def run(d):
        out = _call(d)
        return [out.detach(), *torch.autograd.grad(out, [d[n] for n in NAMES], d["dout"])]

    want = [run(d) for d in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(cases[i]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for r in g:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


def test_backward_op_refuses(gpu):
    d = _to(_case(8, 3, 2, 16, 24, 16, 11), gpu, False)
    out, space = torch.ops.strata_hip.expert_mlp_train(*(d[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual")))
    a = dict(dout=d["dout"], x=d["x"], weights=d["weights"], w1=d["w1"], b1=d["b1"], w2=d["w2"], b2=d["b2"], space=space, need=[True] * 6)
    assert all(t.numel() for t in torch.ops.strata_hip.expert_mlp_bwd(**a))
    for over, msg in ((dict(dout=d["dout"][:4]), "dout"), (dict(dout=d["dout"].float()), "dout"), (dict(space=space[:-4]), "space"),
                      (dict(space=space.view(torch.int32)), "space"), (dict(need=[True]), "need"), (dict(x=d["x"][:7]), "top_k"),
                      (dict(w1=d["w1"][:2]), "E, H"), (dict(weights=d["weights"].float()), "bfloat16")):
        with pytest.raises(ValueError, match=msg):
            torch.ops.strata_hip.expert_mlp_bwd(**dict(a, **over))


def test_refusals(gpu):
    c = _to(_case(8, 3, 2, 16, 24, 16, 11), gpu, False)
    for over, msg in ((dict(x=c["x"].float()), "bfloat16"), (dict(index=c["index"].long()), "int32"),
                      (dict(w1=c["w1"][:, :, :8]), r"\[E, H"), (dict(w2=c["w2"][:2]), r"\[E, N"), (dict(b1=c["b2"]), "b1"),
                      (dict(weights=c["weights"][:, :1]), "top_k"), (dict(residual=c["residual"][:4]), "residual"),
                      (dict(x=c["x"][:, :12], w1=c["w1"][:, :, :12]), "multiples"), (dict(x=c["x"].cpu()), "GPU")):
        with pytest.raises(ValueError, match=msg):
            _call(dict(c, **over))
    x = c["x"].clone().requires_grad_()
    out = _call(dict(c, x=x))
    (g,) = torch.autograd.grad(out.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


def test_compiled_for_any_number_of_tokens(gpu):
    """One compilation, several numbers of tokens: outputs and gradients as the direct calls'."""
    from torch._dynamo.testing import CompileCounterWithBackend

    base = _to(_case(8, 4, 2, 64, 72, 64, 23), gpu, False)
    shared = [base[n].requires_grad_() for n in ("w1", "b1", "w2", "b2")]
    counter = CompileCounterWithBackend("aot_eager")
    torch._dynamo.reset()
    f = torch.compile(lambda x, w, i, r: ops.expert_mlp(x, w, i, *shared, r), backend=counter, fullgraph=True, dynamic=True)
    for T in (8, 333, 65, 2000):
        d = _to(_case(T, 4, 2, 64, 72, 64, T), gpu, False)
        x = d["x"].requires_grad_()
        args = x, d["weights"], d["index"], d["residual"]
        got, want = f(*args), ops.expert_mlp(*args[:3], *shared, args[3])
        assert torch.equal(got, want), T
        for a, b in zip(torch.autograd.grad(got, [x, *shared], d["dout"]), torch.autograd.grad(want, [x, *shared], d["dout"])):
            assert torch.equal(a, b), T
    assert counter.frame_count == 1


def test_gelu_of_far_values(gpu):
    """Hidden pre-activations whose squares leave fp32: GELU's derivative is 1 or 0 there, not 0 times infinity."""
    far = torch.tensor([2.0**70, -(2.0**70), 2.0**64, -(2.0**64), 2.0**40, -(2.0**40), 2.0**120, -(2.0**120)])
    T, n = 200, 8
    ones = lambda *s: torch.ones(*s, device=gpu).bfloat16()  # noqa: E731
    b1 = far.to(gpu).bfloat16()[None].requires_grad_()
    w1 = torch.zeros(1, n, n, device=gpu).bfloat16().requires_grad_()
    w2 = (ones(1, n, n) * 2.0**-60).requires_grad_()
    x, w, i = ones(T, n).requires_grad_(), ones(T, 1), torch.zeros(T, 1, dtype=torch.int32, device=gpu)
    out = ops.expert_mlp(x, w, i, w1, b1, w2, None)
    assert torch.equal(out, (ones(T, n).float() * far.clamp_min(0).sum().item() * 2.0**-60).bfloat16())
    dx, db1, dw1, dw2 = torch.autograd.grad(out, [x, b1, w1, w2], ones(T, n))
    d = (far > 0).float().to(gpu)
    assert torch.equal(db1.float(), (d * T * n * 2.0**-60)[None]) and torch.equal(dw1.float(), (d * T * n * 2.0**-60)[None, :, None].expand(1, n, n))
    assert not dx.any() and torch.equal(dw2.float(), (far.clamp_min(0).to(gpu) * T)[None, None].expand(1, n, n))


@pytest.mark.parametrize("k,H", [(1, 9224), (1, 16392), (1, 32768), (2, 4608), (2, 4616), (3, 3064), (3, 3088), (4, 2304), (4, 2312)])
def test_fused_second_product_at_its_limits(gpu, k, H):
    """A token's pairs just under and over the width that one launch takes, and one pair of any width."""
    print(f"experts, one token {k} {H}", flush=True)
    c = _case(1, 5, k, 64, H, 72, 24, dropped=0.0)
    want = O.mlp_bounds(*(c[n] for n in ("x", "weights", "index", "w1", "b1", "w2", "b2", "residual")))
    d = _to(c, gpu, False)
    out = _call(d)
    _inside(out, want["out"], "out")
    assert torch.equal(out, _call(d))
