"""The balance of the routing over more tokens than a grid of the backward holds."""

import pytest
import torch

from strata_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0**-24


def test_gradient_past_a_grid(gpu):
    """2^26 tokens of more than 256 experts (35 GB of logits): all alike but for some around the border of the first launch, the
    first and the last.  The tolerance is test_balance_gpu's: a bf16 result's half step, 16 u of a score and 24 u of lse."""
    E, T, S = 257, (1 << 26) + 6, 2
    border = 4 * (0xffffffff // 256)  # four tokens a workgroup
    rows = torch.tensor([0, 1, T // 2, border - 1, border, border + 3, T - 2, T - 1], device=gpu)
    x = torch.full((T, E), 0.5, dtype=torch.bfloat16, device=gpu)
    g = torch.Generator().manual_seed(1)
    x[rows] = (torch.randn(len(rows), E, generator=g) * 2).bfloat16().to(gpu)
    index = (torch.arange(T, dtype=torch.int32, device=gpu) % 251)[:, None]
    x.requires_grad_()
    balance, z, load = ops.expert_balance(x, index, "softmax", S)
    assert load.tolist() == [T // 251 + (e < T % 251) if e < 251 else 0 for e in range(E)]
    # weights near the sizes of the sums, so that the gradient is no subnormal number
    gb, gz = 2.0**20, 2.0**18
    grad = torch.autograd.grad((balance, z), x, [torch.tensor(w, device=gpu) for w in (gb, gz)])[0]
    n = T // S
    l = x.detach()[rows].cpu().double()
    lse, s = torch.logsumexp(l, 1, keepdim=True), torch.softmax(l, 1)
    f = torch.stack([index[i * n:(i + 1) * n].flatten().bincount(minlength=E).cpu().double() * E / n for i in range(S)])[(rows >= n).long().cpu()]
    mean = (f * s).sum(1, keepdim=True)
    want = gb * s * (f - mean) / (n * S) + gz * 2 * lse * s / T
    size = gb * s * (f + mean) / (n * S) + gz * 2 * lse.abs() * s / T
    tol = 2.0**-8 * want.abs() + 2 * (64 * U * size + gz * 2 / T * U * (2 * float(l.abs().max()) + 24))
    got = grad[rows].cpu().double()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())
    # all others are those of their sequence's first one
    plain = [3, T - 5]
    for a, b, at in ((0, n, plain[0]), (n, T, plain[1])):
        other = torch.ones(b - a, dtype=torch.bool, device=gpu)
        other[rows[(rows >= a) & (rows < b)] - a] = False
        for lo in range(a, b, 1 << 23):
            hi = min(lo + (1 << 23), b)
            same = (grad[lo:hi] == grad[at]).all(1)
            assert bool((same | ~other[lo - a:hi - a]).all()), (lo, hi)
