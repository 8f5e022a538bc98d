"""How exact orthogonalised updates are on the GPU, against their float64 oracle.

``FINE`` bounds the error of operands of 22 bits relative to the result's norm.  X = x / |x| of noise has singular values that
all grow alike, so a step's relative errors are kept and add up as independent ones: thirty roundings (five steps, of X in
X X^T twice, of A in A A twice, of P, of X in P X), each of half a step of two fp16 (2^-22), as much for the product
of the two second ones that is left out and as much for the fp32 sums: sqrt(30) 3 2^-22 = 3.9e-6.  Operands of 16 bits are off by
sqrt(30) times the 0.4 of half a step 2^-16 that a rounding has in the mean: 3e-5.

A result y + e of bf16 differs from y rounded only where a border of the rounding lies between them: for the error e_i the
chance is |e_i| / step_i and the difference step_i, so that the mean of its square is step_i |e_i| <= 2^-7 |y_i| |e_i|, in all
at most 2^-7 |y| |e|.  Twice that is asked for.
"""

import pytest
import torch

from oracle import optim as O
from strata_amd import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
FINE = 4e-6


def noise(*shape, seed=1):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def rounded_alike(got, want, size):
    """Of ``got`` in bf16 and the exact ``want``, whose part that the products make has the norm ``size``."""
    off = float((got.double() - want.to(BF16).double()).norm())
    tol = 2 * (2.0**-7 * float(want.norm()) * FINE * size) ** 0.5
    print(f"  {off:.2e} of {tol:.2e}", flush=True)
    assert off <= tol


SHAPES = [(128, 128), (70, 400), (300, 512), (600, 513), (960, 130), (40, 3000), (64, 64)]


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_a_bf16_result_is_the_exact_one_rounded(gpu, rows, cols):
    x = noise(rows, cols).to(BF16)
    print(f"orthogonalize {rows} {cols}", flush=True)
    want, _ = O.orthogonalize(x.double())
    rounded_alike(ops.orthogonalize(x.to(gpu)).cpu(), want, float(want.norm()))


def test_a_step_of_bf16_weights_is_the_exact_one_rounded(gpu):
    """Weights of zero (a layer that starts as the identity's branch) are the update alone."""
    shapes = [(300, 512), (128, 128), (512, 300), (24, 960)]
    for start in (0.0, 0.02):
        p = [(noise(*s, seed=2) * start).to(BF16) for s in shapes]
        g, m = [noise(*s, seed=3).to(BF16) for s in shapes], [noise(*s, seed=4).float() for s in shapes]
        q = [t.to(gpu) for t in p]
        ops.muon_step(q, [t.to(gpu) for t in g], [t.to(gpu) for t in m], lr=2e-2, weight_decay=0.1, adjust="match_rms_adamw")
        for a, b, c, d in zip(p, q, g, m):
            want, _, _ = O.muon(a.double(), c.double(), d.double(), 2e-2, 0.95, True, 0.1, "match_rms_adamw")
            print(f"muon {tuple(a.shape)} from {start}", flush=True)
            # p (1 - lr decay) is off by 3 roundings of fp32 itself
            base = a.double() * (1 - 2e-3)
            rounded_alike(b.cpu(), want, float((want - base).norm()) + 3 * 2.0**-24 / FINE * float(base.norm()))


@pytest.mark.parametrize("p_dtype", [BF16, F32])
def test_narrow_matrices_beside_wide_ones_of_fewer_bits(gpu, p_dtype):
    """A side of at most 64 keeps 22 bits whatever the call's other matrices take: routers beside the other weights of a model."""
    narrow, wide = [(24, 960), (960, 64), (1, 700), (8, 1000)], [(300, 512), (130, 70)]
    for shapes in (narrow + wide[:1], narrow + wide[1:], narrow + wide):
        p = [torch.zeros(s, dtype=p_dtype, device=gpu) for s in shapes]
        g = [noise(*s, seed=5).to(p_dtype) for s in shapes]
        m = [noise(*s, seed=6).float() for s in shapes]
        ops.muon_step(p, [t.to(gpu) for t in g], [t.to(gpu) for t in m], lr=1e-2, weight_decay=0.0, precise=False)
        for i in range(len(narrow)):
            want, _, _ = O.muon(torch.zeros(shapes[i], dtype=torch.float64), g[i].double(), m[i].double(), 1e-2, decay=0.0)
            print(f"muon {shapes[i]} beside {shapes[4:]}", flush=True)
            if p_dtype == BF16:
                rounded_alike(p[i].cpu(), want, float(want.norm()))
            else:
                assert float((p[i].cpu().double() - want).norm()) <= FINE * float(want.norm())


def decaying(rows, cols, decades, seed=7):
    """Singular values that decay evenly over so many powers of ten."""
    k = min(rows, cols)
    u, v = torch.linalg.qr(noise(rows, k, seed=seed))[0], torch.linalg.qr(noise(cols, k, seed=seed + 1))[0]
    return (u * 10 ** (-decades * torch.arange(k).double() / (k - 1))) @ v.T


@pytest.mark.parametrize("rows,cols", [(128, 128), (300, 512), (512, 600), (700, 300)])
def test_operands_of_11_bits_where_singular_values_decay(gpu, rows, cols):
    """Off by less than the rounding of a bf16 result: uniform in half a step 2^-8, which is 2^-8 / sqrt(3) of a value at the start of its
    binade and half of that at its end, 0.43 2^-8 = 1.7e-3 of normal values.  The kernels' roundings taken on the CPU
    give 0.9e-3 to 1.5e-3 with X's second fp16 in three steps, and 2 to 3.5e-3 from three decades on with it in two."""
    for decades in (0, 2, 3, 4):
        x = decaying(rows, cols, decades) if decades else noise(rows, cols)
        want, _ = O.orthogonalize(x.float().double())
        got = ops.orthogonalize(x.float().to(gpu), precise=False).cpu().double()
        off = float((got - want).norm() / want.norm())
        print(f"orthogonalize {rows} {cols} over {decades} decades: {off:.2e}", flush=True)
        assert off <= 1.7e-3


@pytest.mark.parametrize("rows,cols", [(512, 600), (300, 512), (130, 257), (128, 128), (960, 960), (200, 1500), (8, 1000), (8, 200), (384, 776), (1, 500)])
def test_operands_of_22_bits(gpu, rows, cols):
    """Matrices alone, in a stack, and as the steps of fp32 weights and of masters: all of one exactness."""
    x = noise(rows, cols).float()
    want, _ = O.orthogonalize(x.double())
    size = float(want.norm())
    got = {"alone": ops.orthogonalize(x.to(gpu)), "stack": ops.orthogonalize(torch.stack([x, 2 * x, x]).to(gpu))[2]}
    zero = lambda t=F32: torch.zeros(rows, cols, dtype=t, device=gpu)  # noqa: E731
    p, master = zero(), zero()
    kw = dict(lr=1.0, momentum=0.0, weight_decay=0.0)
    ops.muon_step([p], [x.to(gpu)], [zero()], **kw)
    ops.muon_step([zero(BF16)], [x.to(gpu)], [zero()], masters=[master], **kw)
    scale = -max(1.0, rows / cols) ** 0.5
    got.update(weights=p / scale, masters=master / scale)
    for what, y in got.items():
        off = float((y.cpu().double() - want).norm()) / size
        print(f"{rows} {cols} {what}: {off:.2e}", flush=True)
        assert off <= FINE, what


@pytest.mark.parametrize("rows,cols", [(8, 1000), (384, 776), (8, 200), (128, 128)])
def test_the_second_products_have_sums_of_their_own(gpu, rows, cols):
    """A sum of X X^T on the diagonal is of positive terms.  In one sum with the products of the second fp16 it would be rounded three
    times as often as by itself (twice as off, 2.2e-6 of 8 x 1000): at most 2e-6 is what is documented."""
    x = noise(rows, cols).float()
    want, _ = O.orthogonalize(x.double())
    off = float((ops.orthogonalize(x.to(gpu)).cpu().double() - want).norm() / want.norm())
    print(f"{rows} {cols}: {off:.2e}", flush=True)
    assert off <= 2e-6


def fewer_bits(got, x):
    """``got``: the result of x with fp16 operands, within 2.1e-3 (the kernels' roundings taken on the CPU: 1.9e-3 for a side of 65,
    less for longer ones) and its own rounding."""
    want, _ = O.orthogonalize(x.double())
    off = float((got.double() - want).norm() / want.norm())
    print(f"  {tuple(x.shape)}: {off:.2e}", flush=True)
    assert off <= (2.1e-3**2 + ((2.0**-8 / 2) ** 2 if got.dtype == BF16 else 0)) ** 0.5


@pytest.mark.parametrize("count,rows,cols,dtype", [(100, 130, 260, BF16), (70, 512, 600, BF16), (150, 260, 300, F32), (64, 513, 400, BF16),
                                                   (90, 384, 260, F32), (20, 960, 1920, BF16), (300, 100, 120, BF16), (40, 400, 90, F32)])
def test_many_matrices_of_fewer_bits(gpu, count, rows, cols, dtype):
    """Enough of them for every tile of the products of one fp16: each as alone, to the bit, and some against the oracle."""
    g = torch.Generator(device=gpu).manual_seed(count)
    x = torch.randn(count, rows, cols, generator=g, device=gpu).to(dtype)
    y = ops.orthogonalize(x, precise=False)
    for i in (0, count // 2, count - 1):
        fewer_bits(y[i].cpu(), x[i].cpu())
        assert torch.equal(y[i], ops.orthogonalize(x[i], precise=False))
    assert torch.equal(ops.orthogonalize(x, precise=False), y)


def test_offsets_past_32_bits_of_fewer_bits(gpu):
    x = torch.empty(64000, 130, 256, dtype=BF16, device=gpu).fill_(0.5)
    g = torch.Generator(device=gpu).manual_seed(1)
    for i in (0, 1, 32000, 63999):
        x[i] = torch.randn(130, 256, generator=g, device=gpu)
    y = ops.orthogonalize(x, precise=False)
    for i in (0, 1, 2, 32000, 63999):
        assert torch.equal(y[i], ops.orthogonalize(x[i], precise=False)), i
    fewer_bits(y[63999].cpu(), x[63999].cpu())


def test_a_step_of_every_precision_at_once(gpu):
    """Narrow, slim and wide matrices with and without masters, in steps of 22 bits, of 11 and of each by its type (the C interface's
    ``precise`` without ``bits``): every matrix as in a call of its own, to the bit."""
    import ctypes

    from strata_amd import _lib

    shapes = [(24, 960), (100, 400), (300, 512), (512, 300), (2, 130, 200), (1, 2000), (700, 130)]
    def tensors():
        g = torch.Generator().manual_seed(3)
        r = lambda s: torch.randn(s, generator=g)  # noqa: E731
        return [dict(p=(r(s) * 0.02).to(t).to(gpu), g=r(s).to(BF16).to(gpu), m=r(s).to(gpu), w=(r(s) * 0.02).to(gpu) if i % 3 == 1 else None)
                for i, s in enumerate(shapes) for t in ((BF16,) if i % 3 == 1 else (BF16, F32))]

    def step(ts, bits):
        table = (_lib.MuonMatrix * len(ts))(*[
            (t["p"].data_ptr(), t["g"].data_ptr(), t["m"].data_ptr(), None if t["w"] is None else t["w"].data_ptr(),
             t["p"][..., 0, 0].numel(), *t["p"].shape[-2:], 1e-2, 0.1, int(t["p"].dtype == BF16) * _lib.BF16 + int(t["p"].dtype == F32) * _lib.F32, _lib.BF16,
             int(t["p"].dtype == F32 or t["w"] is not None), bits) for t in ts])
        ws = torch.empty(_lib.load().strata_hip_muon_workspace(table, len(ts)), dtype=torch.uint8, device=gpu)
        a = _lib.MuonArgs(table, len(ts), (ctypes.c_double * 15)(*O.NEWTON_SCHULZ * 5), ws.data_ptr(), 0.95, 1e-7, 5, 1, 0, 0)
        _lib.call("strata_hip_muon_step", a, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()

    for bits in (0, 11, 22):
        ts, alone = tensors(), tensors()
        step(ts, bits)
        for i, (a, b) in enumerate(zip(ts, alone)):
            step([b], bits)
            for k in "pmw":
                assert a[k] is None or torch.equal(a[k], b[k]), (bits, i, k)
