"""The balance of the routing over many sequences, which more than one workgroup adds up."""

import pytest
import torch

from strata_amd import ops
from tests.test_balance import routed
from tests.test_balance_gpu import GB, GZ, _check, _run

pytestmark = pytest.mark.gpu
U = 2.0**-24


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("per,E,k,sequences,masked", [(3, 7, 2, 64, 0.2), (2, 7, 2, 65, 0.3), (5, 24, 3, 129, 0.6), (1, 512, 4, 200, 0.0), (2, 1, 1, 1000, 0.4),
                                                      (3, 300, 2, 130, 0.9)])
def test_matches_the_oracle(gpu, per, E, k, sequences, masked, score):
    print(f"balance {per} {E} {k} {sequences} {masked} {score}", flush=True)
    logits, index = routed(per * sequences, E, k, masked, per + E, torch.float32)
    out, grad = _run(logits, index, score, sequences, gpu)
    _check(logits, index, score, sequences, out, grad)
    again, grad2 = _run(logits, index, score, sequences, gpu)
    assert all(torch.equal(a, b) for a, b in zip(out, again)) and torch.equal(grad, grad2)


@pytest.mark.parametrize("per,E,sequences", [(1, 8, 65536), (3, 40, 65536), (1, 512, 65535)])
def test_as_many_sequences_as_it_takes(gpu, per, E, sequences):
    """Against the formula in 64 bits (the oracle goes token by token); tolerances as in test_balance_gpu."""
    g = torch.Generator().manual_seed(E)
    T, k = per * sequences, min(2, E)
    logits = torch.randn(T, E, generator=g) * 2
    logits[5 * per:7 * per] = -torch.inf
    index = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    out, grad = _run(logits, index, "softmax", sequences, gpu)
    l = logits.double()
    live = torch.isfinite(l).all(1)
    s = torch.where(live[:, None], torch.softmax(l, 1), 0.0)
    named = torch.zeros(sequences, E, dtype=torch.float64).index_put_(
        (torch.arange(T).repeat_interleave(k) // per, index.flatten().long()), torch.ones(T * k, dtype=torch.float64), accumulate=True)
    count = live.view(sequences, per)[:, 0]  # a sequence is masked as a whole here
    want = (named * E / (k * per) * s.view(sequences, per, E).mean(1)).sum(1)[count].mean()
    lse = torch.logsumexp(l[live], 1)
    most = float(l[live].abs().max())
    assert torch.equal(out[2].cpu(), index.flatten().bincount(minlength=E).int())
    assert abs(float(out[0]) - float(want)) <= 64 * U * float(want)
    off = U * (2 * most + 24)
    z = float((lse**2).mean())
    assert abs(float(out[1]) - z) <= float((2 * lse.abs() * off + off**2).mean()) + U * z
    f = (named * E / (k * per * per * int(count.sum()))).repeat_interleave(per, 0)
    mean = (f * s).sum(1, keepdim=True)
    zc = GZ * 2 / int(live.sum())
    lse = torch.where(live, torch.logsumexp(l, 1), 0.0)[:, None]
    dl, size = GB * s * (f - mean) + zc * lse * s, GB * s * (f + mean) + zc * lse.abs() * s
    assert ((grad.cpu().double() - dl).abs() <= U * dl.abs() + 2 * 64 * U * size + zc * off + 1e-38).all()


def test_sequences_without_a_token(gpu):
    """Many sequences of no tokens at all, and of tokens without an expert."""
    for T in (0, 400):
        logits = torch.full((T, 5), -torch.inf)
        (balance, z, load), grad = _run(logits, torch.full((T, 2), -1, dtype=torch.int32), "softmax", 200, gpu)
        assert float(balance) == 0 and float(z) == 0 and load.tolist() == [0] * 5 and not grad.any() and grad.shape == logits.shape


def test_replayed_from_a_graph(gpu):
    logits, index = routed(600, 24, 3, 0.1, 7, torch.bfloat16)
    l, i = logits.to(gpu), index.to(gpu)
    ops.expert_balance(l, i, "sigmoid", 300)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.expert_balance(l, i, "sigmoid", 300)
    for _ in range(4):
        l.mul_(0.9).add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ops.expert_balance(l, i, "sigmoid", 300)))
        torch.cuda.synchronize()


def test_time_of_many_sequences(gpu):
    """65536 sequences take some times what one does, not hundreds of times (the plain form in torch took a twentieth of that)."""
    g = torch.Generator(device=gpu).manual_seed(1)
    logits = torch.randn(65536, 64, generator=g, device=gpu)
    index = torch.randint(0, 64, (65536, 2), generator=g, dtype=torch.int32, device=gpu)

    def shortest(sequences):
        times = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                ops.expert_balance(logits, index, "softmax", sequences)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) * 100)
        return min(times)

    one, many = shortest(1), shortest(65536)
    print(f"one sequence {one:.1f} us, 65536 {many:.1f} us", flush=True)
    assert many <= 30 * one
