"""Orthogonalised updates of matrices with more sums of squares than a tile adds up (more than 8 M elements)."""

import pytest
import torch

from strata_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0**-24


def test_norms_of_large_matrices(gpu):
    """Without steps the result is x / |x|: two fp16 (2^-22), a rounded scale, product and result (3 u).  The last of a stack's elements
    are its largest, so that every one of its sums counts; small matrices of the same call keep theirs."""
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.randn(3, 3001, 4099, generator=g, device=gpu)
    x *= torch.tensor([1e-3, 1.0, 1e8], device=gpu)[:, None, None]
    x[:, -1, -30:] *= 3000
    y = ops.orthogonalize(x, coefficients=())
    for i in range(3):
        want = x[i].double() / x[i].double().norm()
        tol = (2.0**-22 + 3 * U) * want.abs() + 2.0**-25 / 2**12  # fp16's smallest step, of the second one, times 2^-12
        assert ((y[i].double() - want).abs() <= tol).all(), i
        assert torch.equal(y[i], ops.orthogonalize(x[i], coefficients=())), i
    assert torch.equal(ops.orthogonalize(x.mT, coefficients=()), y.mT)
    small = [torch.randn(s, generator=g, device=gpu) for s in ((200, 300), (24, 960), (2900, 2900))]
    zero = [torch.zeros_like(t) for t in (*small, x[0])]
    ops.muon_step(zero, [*small, x[0]], [torch.zeros_like(t) for t in zero], momentum=0.0, lr=1.0, weight_decay=0.0, coefficients=())
    for p, t in zip(zero, (*small, x[0])):
        want = t.double() / t.double().norm()
        tol = (2.0**-22 + 4 * U) * want.abs() + 2.0**-25 / 2**12
        assert ((-p.double() - want).abs() <= tol).all(), p.shape


def test_passes_grow_with_the_matrix_alone(gpu):
    """2^31 elements: the passes around the products read and write 30 GB, 3.5 times what a copy does.  Sums that every tile added up
    anew were a thousand GB of reads, 37 times a copy."""
    x = torch.empty(32768, 65536, dtype=torch.bfloat16, device=gpu).normal_()

    def shortest(f):
        times = []
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            f()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    copy, call = shortest(x.clone), shortest(lambda: ops.orthogonalize(x, coefficients=()))
    print(f"copy {copy:.2f} ms, call {call:.2f} ms", flush=True)
    assert call <= 12 * copy


def test_large_steps_from_a_graph(gpu):
    """The sums' own launch, captured and replayed."""
    g = torch.Generator(device=gpu).manual_seed(2)
    x = torch.randn(2100, 4096, generator=g, device=gpu).bfloat16()
    ops.orthogonalize(x, steps=1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.orthogonalize(x, steps=1)
    for _ in range(3):
        x.mul_(1.5).add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.orthogonalize(x, steps=1))
        torch.cuda.synchronize()
