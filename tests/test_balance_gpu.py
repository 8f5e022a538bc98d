"""The balance of the routing on the GPU against its float64 oracle.

Tolerances count roundings of half a step (u = 2^-24).  A softmax's score is within 16 u of itself; one of a sigmoid is an
exponential of logarithms of up to |l| + 1, three of them rounded twice, so within 6 |l| u more.  Sums over tokens are of
positive terms: 3 rounds, 9 exchanges and sums of a workgroup, 64 bits after that: C = 64 + 6 max|l| counts all of it.  The
log-sum-exp is off by at most (2 max|l| + 24) u.
"""

import pytest
import torch

from oracle import experts as O
from strata_amd import modules, ops
from tests.test_balance import formula, routed

pytestmark = pytest.mark.gpu
U = 2.0**-24
GB, GZ = 1e-2, 1e-3


def _check(logits, index, score, sequences, got, grad=None):
    """``got``: (balance, z, load) on the GPU of these logits, on the CPU, in their own type; ``grad``: theirs, of GB and GZ."""
    l = logits.double()
    ok = torch.isfinite(l)
    most = float(l[ok].abs().max()) if ok.any() else 0.0
    balance, z, load = O.balance(l, index, score, sequences)
    c, off = 64 + (6 * most if score == "sigmoid" else 0), U * (2 * most + 24)
    lse = torch.where(ok.any(1), torch.logsumexp(torch.where(ok, l, -torch.inf), 1), 0.0)
    got = [g.detach() for g in got]
    assert torch.equal(got[2].cpu(), load)
    assert abs(float(got[0]) - float(balance)) <= c * U * float(balance)
    n = max(int(ok.any(1).sum()), 1)
    assert abs(float(got[1]) - float(z)) <= float((2 * lse.abs() * off + off**2).sum()) / n + U * float(z)
    if grad is None:
        return
    want, size = formula(l, index, score, sequences, GB, GZ)
    half = torch.finfo(logits.dtype).eps / 2
    tol = half * want.abs() + (1 + half) * (2 * c * U * size + GZ * 2 / n * off) + 1e-38
    assert ((grad.cpu().double() - want).abs() <= tol).all(), float(((grad.cpu().double() - want).abs() / tol).max())


def _run(logits, index, score, sequences, gpu):
    leaf = logits.to(gpu).requires_grad_()
    out = ops.expert_balance(leaf, index.to(gpu), score, sequences)
    grad = torch.autograd.grad(out[:2], leaf, [torch.tensor(GB, device=gpu), torch.tensor(GZ, device=gpu)])[0]
    return out, grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,sequences,masked", [
    (1, 1, 1, 1, 0.0), (1, 8, 2, 1, 0.0), (2, 3, 1, 2, 0.3), (64, 5, 2, 1, 0.0), (1350, 24, 3, 1, 0.1), (999, 12, 4, 3, 0.5),
    (800, 64, 8, 16, 0.0), (513, 130, 4, 1, 0.9), (340, 512, 8, 20, 0.2), (300, 257, 1, 2, 0.0), (520, 16, 64, 1, 0.0)])
def test_matches_the_oracle(gpu, T, E, k, sequences, masked, score, dtype):
    print(f"balance {T} {E} {k} {sequences} {masked} {score} {dtype}", flush=True)
    logits, index = routed(T, E, k, masked, T + E, dtype)
    out, grad = _run(logits, index, score, sequences, gpu)
    _check(logits, index, score, sequences, out, grad)
    with torch.no_grad():
        again = ops.expert_balance(logits.to(gpu), index.to(gpu), score, sequences)
    assert all(torch.equal(a, b) for a, b in zip(out, again))  # the same bits on every call


def test_a_long_batch(gpu):
    """More tokens than one round of every workgroup, against the formula (the oracle goes token by token)."""
    g = torch.Generator().manual_seed(2)
    T, E, k, S = 300001 * 2, 8, 2, 2
    logits = torch.randn(T, E, generator=g) * 2
    index = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    (balance, z, load), grad = _run(logits, index, "softmax", S, gpu)
    l = logits.double()
    lse, s = torch.logsumexp(l, 1), torch.softmax(l, 1)
    part = [sum(((index[i] == e).sum().double() * E / (k * (T // S)) * s[i, e].mean()) for e in range(E)) for i in (slice(0, T // S), slice(T // S, T))]
    rounds = T // S // 256 // 256 + 2  # of a lane's own sum
    assert abs(float(balance) - float(sum(part) / S)) <= (64 + rounds) * U * 1.1
    assert abs(float(z) - float((lse**2).mean())) <= float((2 * lse.abs() * U * (2 * float(l.abs().max()) + 24)).mean()) + U * float(z)
    assert torch.equal(load.cpu(), index.flatten().bincount(minlength=E).int())
    want, size = formula(l, index, "softmax", S, GB, GZ)
    tol = U * want.abs() + 2 * 64 * U * size + GZ * 2 / T * U * (2 * float(l.abs().max()) + 24) + 1e-38
    assert ((grad.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_nothing_to_route(gpu, score):
    """No tokens at all, no token with an expert, and a sequence without one beside another."""
    for T, masked in ((0, False), (6, True)):
        logits = torch.full((T, 4), -torch.inf if masked else 0.0)
        (balance, z, load), grad = _run(logits, torch.full((T, 2), -1, dtype=torch.int32), score, 2, gpu)
        assert float(balance) == 0 and float(z) == 0 and load.tolist() == [0] * 4 and not grad.any() and grad.shape == logits.shape
    logits, index = routed(8, 4, 2, 0.0, 3, torch.float32)
    logits[:4] = -torch.inf
    out, grad = _run(logits, index, score, 2, gpu)
    _check(logits, index, score, 2, out, grad)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_logits_of_the_types_lowest_value(gpu, dtype, score):
    """They are finite: an expert of score 0 beside others, an even choice where all of them are (whose square is no number
    of 32 bits)."""
    logits, index = routed(64, 10, 2, 0.0, 4, dtype)
    logits[:, 3] = torch.finfo(dtype).min
    logits[::5, :9] = torch.finfo(dtype).min
    leaf = logits.to(gpu).requires_grad_()
    balance, z, load = ops.expert_balance(leaf, index.to(gpu), score)
    want, _, wload = O.balance(logits.double(), index, score)
    finite = float(logits.double()[logits > torch.finfo(dtype).min].abs().max())
    assert abs(float(balance) - float(want)) <= (64 + 6 * finite) * U * float(want) and torch.equal(load.cpu(), wload)
    assert torch.isfinite(torch.autograd.grad(balance, leaf, retain_graph=True)[0]).all()
    with torch.no_grad():
        lowest = torch.full((3, 4), torch.finfo(dtype).min, dtype=dtype, device=gpu)
        balance, z, _ = ops.expert_balance(lowest, torch.tensor([[0], [1], [2]], dtype=torch.int32, device=gpu), score)
    assert abs(float(balance) - 1) <= 64 * U and float(z) == float("inf")


@pytest.mark.parametrize("l", [-200.0, -1e4, 200.0])
def test_scores_far_out(gpu, l):
    """Sigmoids that are 0 (or 1) in 32 bits keep their ratios."""
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(40, 6, generator=g) + l
    index = torch.randint(0, 6, (40, 2), generator=g, dtype=torch.int32)
    out, grad = _run(logits, index, "sigmoid", 2, gpu)
    _check(logits, index, "sigmoid", 2, out, grad)


def test_strided_and_shared_rows(gpu):
    logits, index = routed(60, 16, 2, 0.0, 6, torch.float32)
    want = ops.expert_balance(logits.to(gpu), index.to(gpu))
    wide = torch.full((60, 40), torch.nan, device=gpu)
    wide[:, 3:19] = logits.to(gpu)
    got = ops.expert_balance(wide[:, 3:19], index.to(gpu).t().contiguous().t())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    shaped = ops.expert_balance(logits.to(gpu).view(3, 4, 5, 16), index.to(gpu).view(3, 4, 5, 2))
    assert all(torch.equal(a, b) for a, b in zip(shaped, want))
    row = logits[:1].to(gpu).requires_grad_()  # a broadcast input: its gradient is the sum
    out = ops.expert_balance(row.expand(60, 16), index.to(gpu))
    _check(logits[:1].expand(60, 16), index, "softmax", 1, out)
    g = torch.autograd.grad(out[1], row)[0]
    lse = torch.logsumexp(logits[0].double(), 0)
    expect = 2 * lse * torch.softmax(logits[0].double(), 0)
    assert ((g.cpu().double()[0] - expect).abs() <= U * (64 + 60) * expect.abs() + U * 64).all()


def test_replayed_from_a_graph_forward_and_backward(gpu):
    logits, index = routed(700, 24, 3, 0.1, 7, torch.bfloat16)
    l, i = logits.to(gpu).requires_grad_(), index.to(gpu)
    gs = [torch.tensor(GB, device=gpu), torch.tensor(GZ, device=gpu)]
    other = routed(700, 24, 3, 0.1, 8, torch.bfloat16)[0].to(gpu)
    _run(logits, index, "sigmoid", 7, gpu)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = ops.expert_balance(l, i, "sigmoid", 7)
        grad = torch.autograd.grad(out[:2], l, gs)[0]
        out = [o.detach() for o in out]
    for k in range(4):
        with torch.no_grad():
            l.copy_(other if k % 2 else logits.to(gpu))
        graph.replay()
        torch.cuda.synchronize()
        want, wgrad = _run(l.detach().cpu(), index, "sigmoid", 7, gpu)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(grad, wgrad), k


def test_two_streams_at_once(gpu):
    cases = [routed(5000, 64, 4, 0.0, 9 + s, torch.float32) for s in range(2)]
    want = [_run(l, i, "softmax", 4, gpu) for l, i in cases]
    at = [(l.to(gpu).requires_grad_(), i.to(gpu)) for l, i in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for s, (l, i) in zip(streams, at):
        with torch.cuda.stream(s):
            out = ops.expert_balance(l, i, "softmax", 4)
            got.append((out, torch.autograd.grad(out[:2], l, [torch.tensor(GB, device=gpu), torch.tensor(GZ, device=gpu)])[0]))
    torch.cuda.synchronize()
    for (a, ga), (b, gb) in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(ga, gb)


def test_routing_losses_of_a_block(gpu):
    """The losses collected from a routed block: those of its router's logits, and their gradient at the router's weight."""
    torch.manual_seed(0)
    block = modules.StrataBlock(128, 2, 3, experts=6, expert_options=dict(top_k=2, score="sigmoid", balance=True)).to(gpu).bfloat16()
    x = torch.randn(2, 3, 8, 8, 128, device=gpu).bfloat16()
    with modules.RoutingLosses(per_sample=True) as routing:
        block(x)
    h = ops.layer_norm(block.attn(ops.layer_norm(x, block.eps), None, residual=x), block.eps)
    logits = (h.float() @ block.mlp.router.weight.float().T).bfloat16().detach()
    # the router's logits are a bf16 product: what is collected is the loss of the block's own
    _, index = block.mlp.route(h)
    want = O.balance(logits.cpu().double().view(-1, 6), index.cpu().view(-1, 2), "sigmoid", 2)
    assert abs(float(routing.balance) - float(want[0])) <= 1e-2 * float(want[0])  # logits off by 2^-8 of up to 2 here
    assert abs(float(routing.z) - float(want[1])) <= 2e-2 * float(want[1])
    (mlp, load), = routing.load
    assert mlp is block.mlp and torch.equal(load.cpu(), want[2])
    (1e-2 * routing.balance + 1e-3 * routing.z).backward()
    assert block.mlp.router.weight.grad.abs().sum() > 0 and block.mlp.w1.grad is None


@pytest.mark.parametrize("reentrant", [False, True])
def test_routing_losses_inside_a_checkpoint(gpu, reentrant):
    """Losses that the region returns have the gradients of the plain run; collected around one that is not
    reentrant, its backward raises."""
    from torch.utils.checkpoint import CheckpointError, checkpoint

    torch.manual_seed(0)
    mlp = modules.ExpertMlp(128, 256, 6).to(gpu).bfloat16()
    x = torch.randn(90, 128, device=gpu).bfloat16().requires_grad_()

    def region(x):
        with modules.RoutingLosses() as routing:
            y = mlp(x)
        return y.float().square().mean() + routing.balance + 1e-2 * routing.z

    wanted = [x, *mlp.parameters()]
    region(x).backward()
    want = [t.grad for t in wanted]
    for t in wanted:
        t.grad = None
    checkpoint(region, x, use_reentrant=reentrant).backward()
    for t, w in zip(wanted, want):
        assert torch.equal(t.grad, w)
    if not reentrant:
        with modules.RoutingLosses() as routing:
            y = checkpoint(mlp, x, use_reentrant=False)
        with pytest.raises(CheckpointError):
            (y.float().sum() + routing.balance).backward()
