"""A block with experts as it is trained and served: routing, the experts' products, the clipped AdamW
step, in one run against the oracles.

The reference takes the experts that the GPU chose (a choice between near scores is not continuous) and
computes everything else by itself.  Relative errors: ten or so roundings to bf16 stand between input and
gradient, 2^-8 / sqrt(3) each at random, 0.7e-2 together: 2e-2 as for the dense block.  The router's
gradient also takes the rounding of its logits (2^-8 |l|, |l| up to 3, in the weights), of the
weights' gradient and of its own: 1.2e-2 + 3 x 2^-8 + 0.3e-2 = 2.6e-2: 4e-2.
"""

import copy

import pytest
import torch
import torch.nn.functional as F

from oracle import block as OB
from oracle import experts as OE
from oracle import optim as OO
from oracle import rope as R
from strata_amd import ops
from strata_amd import rope as P
from strata_amd.modules import ExpertMlp, StrataBlock, init_xavier_
from strata_amd.optim import AdamW

from .conftest import rel_l2

pytestmark = pytest.mark.gpu


def _reference_mlp(x, p, index, score, renorm, scale, residual):
    """Dense over the chosen experts, differentiable: x [T, C] fp32."""
    w = OE.route_weights(x @ p["router.weight"].T, index, score, renorm, scale)
    out = residual
    for e in range(p["w1"].shape[0]):
        tok, slot = (index == e).nonzero(as_tuple=True)
        h = F.gelu(x[tok] @ p["w1"][e].T + p["b1"][e], approximate="tanh")
        y = h @ p["w2"][e].T + p["b2"][e]
        out = out.index_add(0, tok, w[tok, slot][:, None] * y)
    return out


def _record(mlp):
    seen = []
    route = mlp.route

    def wrapped(x):
        out = route(x)
        seen.append(out[1].detach())
        return out

    mlp.route = wrapped
    return seen


@pytest.mark.parametrize("options", [dict(top_k=2), dict(top_k=3, score="sigmoid", groups=2, top_groups=2, renormalize=True,
                                                          scale=1.5, balance=True)], ids=["softmax", "sigmoid-balance"])
def test_block_with_experts_trains(gpu, options):
    C, H, kernel, E = 128, 2, (3, 5, 5), 8
    torch.manual_seed(0)
    blk = StrataBlock(C, H, kernel, mlp_ratio=2.0, experts=E, expert_options=options)
    init_xavier_(blk, torch.Generator().manual_seed(1))
    with torch.no_grad():
        for n, p in blk.named_parameters():
            if p.dim() == 1 or n.endswith(("b1", "b2")):
                p.uniform_(-0.1, 0.1)
        if options.get("balance"):
            blk.mlp.balance.uniform_(-0.05, 0.05)
    params = {k: v.detach().bfloat16().float().requires_grad_(True) for k, v in blk.named_parameters()}
    blk = blk.to(gpu).bfloat16()
    if options.get("balance"):
        assert blk.mlp.balance.dtype == torch.float32 and blk.mlp.balance.is_cuda
    seen = _record(blk.mlp)
    g = torch.Generator().manual_seed(2)
    B, Z, Y, X = 1, 4, 12, 12
    x = torch.randn(B, Z, Y, X, C, generator=g).bfloat16()
    dy = torch.randn(B, Z, Y, X, C, generator=g).bfloat16()
    lat, lon = P.synthetic_tile_latlon(B, Y, X, g)
    cos, sin = P.stereographic_rope_tables(lat, lon, C // H, 10000.0, P.default_rope_length_scale(1))
    c1, s1 = R.tables(lat, lon, C // H, 10000.0, R.default_rope_length_scale(1))
    opt = AdamW(blk.parameters(), lr=1e-3, max_norm=0.5)
    xg = x.to(gpu).requires_grad_(True)
    out = blk(xg, (cos.to(gpu), sin.to(gpu)))
    out.backward(dy.to(gpu))
    # reference: the oracle's block with a zeroed dense MLP is its attention half
    xr = x.float().requires_grad_(True)
    att = {k: v for k, v in params.items() if k.startswith("attn.")}
    att |= {f"mlp.layers.{i}.{n}": torch.zeros(s) for i, a, b in ((0, 8, C), (2, C, 8)) for n, s in (("weight", (a, b)), ("bias", (a,)))}
    mid = OB.block_forward(xr, att, H, kernel, c1.float(), s1.float())
    hid = F.layer_norm(mid, (C,), eps=1e-6).view(-1, C)
    index = seen[0].cpu().view(-1, options["top_k"])
    mlp = {k[4:]: v for k, v in params.items() if k.startswith("mlp.")}
    want = _reference_mlp(hid, mlp, index, options.get("score", "softmax"), True, options.get("scale", 1.0), mid.view(-1, C))
    want.backward(dy.float().view(-1, C))
    assert rel_l2(out.detach(), want.detach().view(out.shape)) <= 1e-2
    assert rel_l2(xg.grad.float(), xr.grad) <= 2e-2
    for name, p in blk.named_parameters():
        assert rel_l2(p.grad.float(), params[name].grad) <= (4e-2 if "router" in name else 2e-2), name
    # the step that uses these gradients
    before = {n: p.detach().cpu().double() for n, p in blk.named_parameters()}
    grads = {n: p.grad.detach().cpu().double() for n, p in blk.named_parameters()}
    opt.step()
    norm = OO.global_norm(grads.values())
    assert abs(float(opt.grad_norm) - norm) <= 1e-12 * norm
    coef = min(1.0, 0.5 / (norm + 1e-6))
    for n, p in blk.named_parameters():
        new, m, v = OO.adamw(before[n], grads[n], 0 * before[n], 0 * before[n], 1, 1e-3, (0.9, 0.999), 1e-8, 1e-2, coef)
        got = opt.state[p]["master"].cpu().double()
        assert ((got - new).abs() <= 2.0**-24 * (3 * before[n].abs() + 24 * 1e-3)).all(), n
        assert torch.equal(p.detach().cpu(), opt.state[p]["master"].cpu().bfloat16()), n
    # and the next one runs on what it left
    opt.zero_grad()
    blk(x.to(gpu), (cos.to(gpu), sin.to(gpu))).backward(dy.to(gpu))
    opt.step()
    assert all(torch.isfinite(p).all() for p in blk.parameters()) and int(opt.state[next(blk.parameters())]["step"]) == 2


def test_expert_mlp_served_from_a_graph(gpu):
    """Router, choice and products captured for one token and for a batch; every replay as the eager call."""
    torch.manual_seed(3)
    mlp = ExpertMlp(64, 128, 8, 2).to(gpu).bfloat16()
    g = torch.Generator().manual_seed(4)
    for tokens in (1, 77):
        x = torch.randn(tokens, 64, generator=g).bfloat16().to(gpu)
        res = torch.randn(tokens, 64, generator=g).bfloat16().to(gpu)
        with torch.no_grad():
            mlp(x, res)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = mlp(x, res)
            for k in range(3):
                x.copy_(torch.randn(tokens, 64, generator=g).bfloat16())
                graph.replay()
                torch.cuda.synchronize()
                want = mlp(x, res)
                torch.cuda.synchronize()
                assert torch.equal(out, want), (tokens, k)


def test_training_step_replayed_from_a_graph(gpu):
    """Routing, products, both backward passes, clipping and the step captured together: each replay as the
    same step made eagerly on a copy.  No graph of the captured leaves is alive at the capture."""
    torch.manual_seed(7)
    mlp = ExpertMlp(64, 128, 8, 2, score="sigmoid").to(gpu).bfloat16()
    twin = copy.deepcopy(mlp)
    g = torch.Generator().manual_seed(8)
    x, dy = (torch.randn(300, 64, generator=g).bfloat16().to(gpu) for _ in range(2))

    def state(module):
        ps = list(module.parameters())
        zeros = lambda dt=torch.float32: [torch.zeros(p.shape, dtype=dt, device=gpu) for p in ps]  # noqa: E731
        return ps, zeros(), zeros(), [p.detach().float() for p in ps], torch.zeros(1, dtype=torch.int64, device=gpu)

    def step(module, ps, m, v, master, count):
        grads = torch.autograd.grad(module(x), ps, dy)
        with torch.no_grad():
            return ops.adamw_step([p.detach() for p in ps], [t.contiguous() for t in grads], m, v, count, lr=1e-2, max_norm=0.5,
                                  masters=master)

    a, b = state(mlp), state(twin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(mlp, *a)
    torch.cuda.current_stream().wait_stream(side)
    step(twin, *b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step(mlp, *a)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = step(twin, *b)
        torch.cuda.synchronize()
        assert float(norm) == float(want) and int(a[4]) == int(b[4]) == k + 2
        for p, q in zip(mlp.parameters(), twin.parameters()):
            assert torch.equal(p, q), k
        x.copy_(torch.randn(300, 64, generator=g).bfloat16())


def test_tokens_do_not_depend_on_their_batch(gpu):
    """A token served alone, in a small batch and in a large one: the tile changes the order of no sum but
    the few-rows kernel's split of the contraction (fp32), so results agree to the last roundings."""
    torch.manual_seed(5)
    mlp = ExpertMlp(128, 256, 4, 2).to(gpu).bfloat16()
    x = torch.randn(3000, 128, generator=torch.Generator().manual_seed(6)).bfloat16().to(gpu)
    with torch.no_grad():
        w, i = mlp.route(x)
        big = mlp(x)
        assert torch.equal(mlp(x[:900]), big[:900])
        one = torch.cat([mlp(x[k:k + 1]) for k in range(4)])
        assert torch.equal(torch.cat([mlp.route(x[k:k + 1])[1] for k in range(4)]), i[:4])
    # h may round the other way beside a border (2^-8 of single values), then out: 2 x 2^-8 of the row's norm
    assert rel_l2(one, big[:4]) <= 2 * 2.0**-8
