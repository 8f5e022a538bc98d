"""Which operands the products of orthogonalised updates take, without a GPU."""

import ctypes

import pytest
import torch

from oracle import optim as O
from strata_amd import _lib, ops
from strata_amd.optim import Muon


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda name, a, *t: seen.append([(a.matrices[i].precise, a.matrices[i].bits) for i in range(a.count)]))
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: torch.device("cpu"))
    return seen


def fine(precise, bits):
    return bits == 22 or (bits == 0 and precise == 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("precise", [None, True, False])
def test_fewer_bits_are_asked_for(launches, dtype, precise):
    """Operands of 22 bits for every type, unless the caller wants less."""
    x = torch.zeros(200, 300, dtype=dtype)
    ops.orthogonalize(x, precise=precise)
    ops.muon_step([x, x.clone()], [x, x], [torch.zeros(200, 300)] * 2, precise=precise,
                  masters=[torch.zeros(200, 300) if dtype == torch.bfloat16 else None, None])
    p = torch.nn.Parameter(x.clone())
    p.grad = x.clone()
    Muon([p], master=False, precise=precise).step()
    assert len(launches) == 3 and all(fine(*row) == (precise is not False) for call in launches for row in call)


@pytest.mark.parametrize("bits", [-1, 1, 16, 24])
def test_c_entries_refuse_other_bits(bits):
    lib = _lib.load()
    for entry, momentum in (("muon_step", 0x3000000), ("orthogonalize", None)):
        t = (_lib.MuonMatrix * 1)((0x1000000, 0x2000000, momentum, None, 1, 136, 136, 1e-3, 0.1, _lib.BF16, _lib.BF16, 0, bits))
        a = _lib.MuonArgs(t, 1, (ctypes.c_double * 15)(*O.NEWTON_SCHULZ * 5), 0x100, 0.95, 1e-7, 5, 1, 0, 0)
        assert getattr(lib, "strata_hip_" + entry)(ctypes.byref(a), None) == _lib.EINVAL
        assert "bits" in lib.strata_hip_last_error().decode()


def test_workspace_of_operands_of_22_bits():
    """A and P, too, are two fp16."""
    lib = _lib.load()
    size = {}
    for precise, bits in ((0, 0), (0, 11), (1, 11), (0, 22), (1, 0), (1, 22)):
        t = (_lib.MuonMatrix * 1)((0x1000000, 0x2000000, 0x3000000, None, 1, 200, 300, 1e-3, 0.1, _lib.BF16, _lib.BF16, precise, bits))
        size[precise, bits] = lib.strata_hip_muon_workspace(t, 1)
    assert size[0, 0] == size[0, 11] == size[1, 11] == 256 + 2 * (4 * 256 * 320 + 2 * 256 * 256)
    assert size[0, 22] == size[1, 0] == size[1, 22] == 256 + 2 * (4 * 256 * 320 + 4 * 256 * 256)


def test_narrow_matrices_keep_22_bits_beside_wide_ones():
    """Room for two fp16 of a router's A and P in a call of fp16 operands; P's only beside matrices that are not slim."""
    lib = _lib.load()
    row = lambda rows, cols, bits: (0x1000000, 0x2000000, 0x3000000, None, 1, rows, cols, 1e-3, 0.1, _lib.BF16, _lib.BF16, 0, bits)  # noqa: E731

    def size(*rows):
        return int(lib.strata_hip_muon_workspace((_lib.MuonMatrix * len(rows))(*rows), len(rows)))

    wide, narrow = 4 * 256 * 320 + 2 * 256 * 256, 4 * 64 * 960 + 4 * 64 * 64
    for bits in (0, 11, 22):
        assert size(row(24, 960, bits), row(200, 300, 11)) == 256 + 2 * (wide + narrow)
        assert size(row(24, 960, bits)) == 256 + 2 * (narrow - 2 * 64 * 64)


def _off(x, cut):
    """The error of products whose operands are an fp16 and the rest as another, of ``cut`` bits, as the kernels scale them."""
    def two(v, scale):
        h = (v * scale).half().double()
        step = 2.0 ** (torch.frexp(v * scale - h)[1].double() - cut)
        return h / scale, ((v * scale - h) / step).round() * step / scale

    def product(p, q):
        return (p[0] @ q[0] + p[1] @ q[0] + p[0] @ q[1]).float().double()

    a, b, c = O.NEWTON_SCHULZ
    want, _ = O.orthogonalize(x)
    X = two(x / x.norm(), 2.0**12)
    for _ in range(5):
        A = two(product(X, (X[0].T, X[1].T)), 2.0**10)
        P = two((b * (A[0] + A[1]) + c * product(A, A)).float().double(), 2.0**10)
        X = two((a * (X[0] + X[1]) + product(P, X)).float().double(), 2.0**12)
    return float((X[0] + X[1] - want).norm() / want.norm())


@pytest.mark.parametrize("rows,cols", [(60, 90), (300, 512), (8, 1000)])
def test_the_bound_notices_operands_of_16_bits(rows, cols):
    """The GPU tests ask for 4e-6 of operands of 22 bits: less than half of it as the kernels round, five times as much with second
    fp16 of four bits."""
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    assert _off(x, 11) <= 2e-6 and _off(x, 4) >= 2e-5
