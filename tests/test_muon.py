"""Orthogonalised updates without a GPU: the oracle, refusals, traces, the optimizer's states."""

import copy
import ctypes
import pickle

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from oracle import optim as O
from strata_amd import _lib, modules, ops
from strata_amd.optim import AdamW, Muon, matrices


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def products(x, coefficients=(O.NEWTON_SCHULZ,) * 5):
    """The definition: products of the matrix itself."""
    x = x / x.norm()
    for a, b, c in coefficients:
        g = x @ x.T
        x = a * x + b * g @ x + c * g @ g @ x
    return x


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 9), (9, 1), (5, 7), (40, 40), (33, 90), (90, 33)])
def test_oracle_is_the_definition(rows, cols):
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows), dtype=torch.float64)
    x[rows // 2] *= 7
    for co in ((O.NEWTON_SCHULZ,) * 5, ((1.5, -0.5, 0.0),) * 3, ((3.0, -3.2, 1.2), (2.0, -1.5, 0.5)), ()):
        got, off = O.orthogonalize(x, co)
        want = products(x, co)
        assert torch.allclose(got, want, rtol=1e-9, atol=1e-11) and 0 < off <= 0.05 * float(want.norm())
        assert O.orthogonalize(x, co, precise=True)[1] <= off / (50 if len(co) > 3 else 1)


def test_values_come_near_one():
    x = torch.randn(30, 50, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    s = torch.linalg.svdvals(O.orthogonalize(x)[0])
    assert float(s.min()) > 0.6 and float(s.max()) < 1.3
    tight = O.orthogonalize(x, ((3.4445, -4.7750, 2.0315),) * 4 + ((1.5, -0.5, 0.0),) * 4)[0]
    assert torch.allclose(tight @ tight.T, torch.eye(30, dtype=torch.float64), atol=1e-5)


def _row(i, **over):
    base = 0x1000000 * (i + 1)
    t = _lib.MuonMatrix(base, base + 0x100000, base + 0x200000, None, 1, 136, 136, 1e-3, 0.1, _lib.BF16, _lib.BF16, 0, 0)
    for k, v in over.items():
        setattr(t, k, v)
    return t


def _call(lib, entry, over=(), first=(), second=()):
    t = (_lib.MuonMatrix * 2)(_row(0, **dict(first)), _row(1, **dict(second)))
    co = (ctypes.c_double * 15)(*O.NEWTON_SCHULZ * 5)
    a = _lib.MuonArgs(t, 2, co, 0x100, 0.95, 1e-7, 5, 1, 0, 0)
    for k, v in dict(over).items():
        setattr(a, k, v)
    return getattr(lib, "strata_hip_" + entry)(ctypes.byref(a), None), lib.strata_hip_last_error().decode()


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("over,first,second,msg", [
    (dict(count=-1), {}, {}, "list"), (dict(steps=-1), {}, {}, "steps"), (dict(steps=65), {}, {}, "steps"),
    (dict(coefficients=None), {}, {}, "coefficients"), (dict(coefficients=(ctypes.c_double * 15)(NAN)), {}, {}, "finite"),
    (dict(eps=0.0), {}, {}, "eps"), (dict(eps=INF), {}, {}, "eps"), (dict(momentum=1.0), {}, {}, "momentum"),
    (dict(momentum=NAN), {}, {}, "momentum"), (dict(momentum=-0.1), {}, {}, "momentum"), (dict(adjust=2), {}, {}, "adjust"),
    (dict(workspace=None), {}, {}, "workspace"), (dict(workspace=0x180), {}, {}, "workspace"),
    ({}, dict(rows=-1), {}, "negative"), ({}, {}, dict(batch=-1), "negative"), ({}, dict(lr=NAN), {}, "finite"),
    ({}, dict(weight_decay=INF), {}, "finite"), ({}, dict(param_dtype=5), {}, "bf16 or f32"), ({}, dict(grad_dtype=7), {}, "bf16 or f32"),
    ({}, dict(param=None), {}, "null"), ({}, dict(grad=None), {}, "null"), ({}, dict(momentum=None), {}, "null"),
    ({}, dict(param_dtype=_lib.F32, master=0x9000000), {}, "master"), ({}, dict(param=0x1000001), {}, "aligned"),
    ({}, dict(momentum=0x1200002), {}, "aligned"), ({}, {}, dict(param=0x1000000), "overlap"),
    ({}, {}, dict(param=0x1000000 + 136 * 136 * 2 - 2), "overlap"), ({}, dict(batch=257), {}, "overlap"),
    ({}, dict(grad=0x1000000), {}, "gradient"), ({}, dict(grad=0x2200000), {}, "gradient"), ({}, dict(master=0x2000000), {}, "overlap"),
])
def test_c_entry_refuses(lib, over, first, second, msg):
    rc, err = _call(lib, "muon_step", over, first, second)
    assert rc == _lib.EINVAL and msg in err, (rc, err)


def test_c_entry_of_the_products_refuses(lib):
    two = dict(momentum=None)
    for first, msg in ((dict(momentum=0x1200000), "step's"), (dict(momentum=None, master=0x1300000), "master"),
                       (dict(momentum=None, grad=0x1000000), "gradient")):
        rc, err = _call(lib, "orthogonalize", {}, first, two)
        assert rc == _lib.EINVAL and msg in err, (rc, err)
    assert lib.strata_hip_orthogonalize(None, None) == lib.strata_hip_muon_step(None, None) == _lib.EINVAL


@pytest.mark.parametrize("size", [dict(rows=1 << 21), dict(cols=1 << 62), dict(rows=(1 << 15) + 1, cols=(1 << 15) + 1),
                                  dict(batch=1 << 21, rows=1, cols=1), dict(batch=1 << 20, rows=1, cols=1 << 11),
                                  dict(batch=1 << 20, rows=1, cols=300), dict(batch=1 << 62)])
def test_sizes_past_the_grids(lib, size):
    rc, err = _call(lib, "muon_step", first=size)
    assert rc == _lib.EUNSUPPORTED and "2^20" in err
    t = (_lib.MuonMatrix * 1)(_row(0, **size))
    assert lib.strata_hip_muon_workspace(t, 1) == -1


def test_workspace_and_empty_calls(lib):
    """Sums of squares, and X twice, A and P in fp16; nothing for matrices that all are small, which one workgroup takes whole."""
    t = (_lib.MuonMatrix * 4)(_row(0, rows=200, cols=65), _row(1, rows=0), _row(2, rows=65, cols=200, precise=1, batch=2), _row(3, rows=64, cols=384))
    size = 8 * 32 + 2 * (4 * 64 * 384 + 2 * 64 * 64) + 2 * (4 * 128 * 256 + 2 * 128 * 128) + 2 * 2 * (4 * 128 * 256 + 4 * 128 * 128)
    assert lib.strata_hip_muon_workspace(t, 4) == size and lib.strata_hip_muon_workspace(None, 0) == 0
    assert lib.strata_hip_muon_workspace(ctypes.byref(t[3]), 1) == 0
    none = (_lib.MuonMatrix * 2)(_row(0, rows=0), _row(1, batch=0))
    a = _lib.MuonArgs(none, 2, None, None, 0.9, 1e-7, 0, 1, 0, 0)
    assert lib.strata_hip_muon_step(ctypes.byref(a), None) == _lib.OK  # nothing to do, nothing launched
    a.count = 0
    assert lib.strata_hip_orthogonalize(ctypes.byref(a), None) == _lib.OK


def test_c_entry_returns_where_a_list_cannot_be_held(lib):
    """More matrices than host memory, or than a vector, holds: an error, no exception across the C boundary."""
    import subprocess
    import sys
    from pathlib import Path

    code = f"""
import ctypes, mmap, resource
from strata_amd import _lib
lib = _lib.load()
n = (96 << 26) // {ctypes.sizeof(_lib.MuonMatrix)}
zeros = mmap.mmap(-1, 96 << 26, flags=mmap.MAP_PRIVATE | mmap.MAP_ANONYMOUS | 0x4000)  # no pages until they are written
t = ctypes.cast(ctypes.addressof(ctypes.c_char.from_buffer(zeros)), ctypes.POINTER(_lib.MuonMatrix))
t[n - 1] = (0x1000000, 0x2000000, 0x3000000, None, 1, 200, 200, 0.1, 0.1, 0, 0, 0, 0)
resource.setrlimit(resource.RLIMIT_AS, (int(open("/proc/self/statm").read().split()[0]) * 4096 + (64 << 20),) * 2)
assert lib.strata_hip_muon_workspace(t, n) == -1
a = _lib.MuonArgs(t, n, None, 0x100, 0.9, 1e-7, 0, 1, 0, 0)
assert lib.strata_hip_muon_step(ctypes.byref(a), None) == _lib.EUNSUPPORTED
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=Path(_lib.__file__).resolve().parents[1])
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])


def test_struct_layouts_are_the_header_s(tmp_path):
    import subprocess
    from pathlib import Path

    header = Path(_lib.__file__).resolve().parents[1] / "include" / "strata_hip.h"
    structs = {"strata_hip_muon_matrix": _lib.MuonMatrix, "strata_hip_muon_args": _lib.MuonArgs,
               "strata_hip_expert_balance_args": _lib.ExpertBalanceArgs}
    lines, want = [f'#include "{header}"', "#include <stddef.h>", "#include <stdio.h>", "int main(void) {"], []
    for name, st in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(st))
        for f, _ in st._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(st, f).offset)
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(src)], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == want


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda name, a, *t: seen.append((name, a)))
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: torch.device("cpu"))
    return seen


def test_ops_refuse():
    x = torch.zeros(4, 4)
    with pytest.raises(ValueError, match="GPU"):
        ops.orthogonalize(x)
    with pytest.raises(ValueError, match="GPU"):
        ops.muon_step([x], [x], [x])
    for kw, msg in ((dict(coefficients=(1.0, 2.0)), "three"), (dict(coefficients=((1.0, 2.0),)), "three"), (dict(steps=65), "64"),
                    (dict(steps=-1), "64"), (dict(coefficients=((1.0, 0.0, 0.0),), steps=2), "triples"), (dict(eps=0.0), "eps"),
                    (dict(coefficients=(NAN, 0.0, 0.0)), "finite"), (dict(eps=NAN), "eps")):
        with pytest.raises(ValueError, match=msg):
            ops.orthogonalize(x, **kw)
        with pytest.raises(ValueError, match=msg):
            ops.muon_step([x], [x], [x], **kw)
    for kw, msg in ((dict(adjust="none"), "adjust"), (dict(momentum=1.0), "momentum"), (dict(lr=[1e-3] * 2), "one entry"),
                    (dict(masters=[]), "one entry"), (dict(weight_decay=[]), "one entry")):
        with pytest.raises(ValueError, match=msg):
            ops.muon_step([x], [x], [x], **kw)
    ops.muon_step([], [], [])


@pytest.mark.parametrize("over,msg", [
    (dict(grads=[torch.zeros(3, 4)]), "grads must be"), (dict(grads=[torch.zeros(4, 3).half()]), "grads must be"),
    (dict(momentums=[torch.zeros(4, 3).bfloat16()]), "momentums must be"), (dict(params=[torch.zeros(3, 4).T]), "params must be"),
    (dict(masters=[torch.zeros(4, 3)]), "masters belong"), (dict(momentums=[torch.zeros(12)]), "momentums must be"),
    (dict(params=[torch.zeros(12)], grads=[torch.zeros(12)], momentums=[torch.zeros(12)]), "stacks"),
    (dict(masters=[torch.zeros(4, 3).double()]), "masters must be")])
def test_step_refuses_tensors(launches, over, msg):
    x = torch.zeros(4, 3)
    with pytest.raises(ValueError, match=msg):
        ops.muon_step(**{**dict(params=[x], grads=[x], momentums=[x]), **over})
    assert not launches


def test_products_refuse_tensors(launches):
    for x, msg in ((torch.zeros(4), "rows, cols"), (torch.zeros(4, 4).half(), "dtype")):
        with pytest.raises(ValueError, match=msg):
            ops.orthogonalize(x)
    with pytest.raises(RuntimeError, match="differentiable"):
        ops.orthogonalize(torch.zeros(4, 4, requires_grad=True))
    assert not launches and ops.orthogonalize(torch.zeros(0, 4, 4)).shape == (0, 4, 4) and not launches
    with torch.no_grad():
        ops.orthogonalize(torch.zeros(4, 4, requires_grad=True))
    assert [n for n, _ in launches] == ["strata_hip_orthogonalize"]


def test_rows_of_a_step(launches):
    """What the C structure holds: stacks, rates, which matrices take operands of twice the bits."""
    p = [torch.zeros(6, 4), torch.zeros(2, 3, 5, 7).bfloat16(), torch.zeros(8, 8).bfloat16(), torch.zeros(2, 0, 3)]
    w = [None, None, torch.zeros(8, 8), None]
    g, m = [t.clone() for t in p], [torch.zeros(t.shape) for t in p]
    for precise, want in ((None, [1, 0, 1, 1]), (False, [0] * 4), (True, [1] * 4)):
        launches.clear()
        ops.muon_step(p, g, m, lr=[1.0, 2.0, 3.0, 4.0], weight_decay=0.5, masters=w, precise=precise, steps=3, adjust="match_rms_adamw")
        (name, a), = launches
        assert name == "strata_hip_muon_step" and (a.count, a.steps, a.nesterov, a.adjust) == (4, 3, 1, 1)
        rows = [a.matrices[i] for i in range(4)]
        assert [(r.batch, r.rows, r.cols, r.lr, r.weight_decay) for r in rows] == [
            (1, 6, 4, 1.0, 0.5), (6, 5, 7, 2.0, 0.5), (1, 8, 8, 3.0, 0.5), (0, 0, 3, 4.0, 0.5)]
        assert [r.precise for r in rows] == want and [r.param_dtype for r in rows] == [_lib.F32, _lib.BF16, _lib.BF16, _lib.F32]
        assert [r.master for r in rows] == [None, None, w[2].data_ptr(), None] and rows[1].grad == g[1].data_ptr()
    v = p[0]._version
    ops.muon_step(p, g, m)
    assert p[0]._version == v + 1


def test_traces_see_the_op(launches):
    x = torch.randn(3, 6, 4)
    f = lambda x: ops.orthogonalize(x, steps=3)  # noqa: E731
    assert "strata_hip.orthogonalize.default" in [str(n.target) for n in make_fx(f)(x).graph.nodes]
    assert "strata_hip::orthogonalize" in str(torch.jit.trace(f, x, check_trace=False).graph)
    assert torch.vmap(f)(x).shape == x.shape
    torch._dynamo.reset()
    assert torch.compile(f, backend="aot_eager", fullgraph=True)(x).shape == x.shape
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=True):
        y = ops.orthogonalize(torch.empty(5, 4, dtype=torch.bfloat16, device="cuda").T)
        assert y.shape == (4, 5) and y.dtype == torch.bfloat16 and y.is_contiguous()
    t = [torch.zeros(4, 4)]
    with pytest.raises(RuntimeError, match="trace"):
        make_fx(lambda p: ops.muon_step([p], t, t))(torch.zeros(4, 4))


def test_optimizer_refuses():
    p = [torch.nn.Parameter(torch.zeros(4, 4))]
    for kw, msg in ((dict(adjust="x"), "adjust"), (dict(momentum=1.0), "momentum"), (dict(eps=0.0), "eps"),
                    (dict(coefficients=(1.0,)), "three"), (dict(steps=99), "64")):
        with pytest.raises(ValueError, match=msg):
            Muon(p, **kw)
    with pytest.raises(ValueError, match="matrices"):
        Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="momentum"):
        Muon([dict(params=p, momentum=0.5)])
    opt = Muon(p)
    with pytest.raises(ValueError, match="matrices"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4))]))
    assert len(opt.param_groups) == 1


def test_optimizer_states(launches, monkeypatch):
    ps = [torch.nn.Parameter(torch.ones(4, 6, dtype=torch.bfloat16)), torch.nn.Parameter(torch.ones(2, 6, 4))]
    opt = Muon([dict(params=ps[:1], lr=0.5), dict(params=ps[1:], weight_decay=0.0)], lr=0.1, nesterov=False, steps=4)
    opt.step()
    assert not launches and not opt.state
    for p in ps:
        p.grad = torch.ones_like(p)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="eager"):
        opt.step()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert opt.step(lambda: 3.0) == 3.0
    (_, a), = launches
    assert [(a.matrices[i].lr, a.matrices[i].weight_decay, a.matrices[i].batch) for i in range(2)] == [(0.5, 0.1, 1), (0.1, 0.0, 2)]
    assert (a.steps, a.nesterov) == (4, 0)
    assert opt.state[ps[0]]["master"].dtype == opt.state[ps[0]]["momentum"].dtype == torch.float32 and "master" not in opt.state[ps[1]]
    for o in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (o.steps, o.nesterov, o.coefficients, o.adjust) == (4, False, ops.NEWTON_SCHULZ, "original")
    other = Muon([torch.nn.Parameter(p.detach().clone()) for p in ps][:1])
    other.add_param_group(dict(params=[torch.nn.Parameter(ps[1].detach().clone())]))
    other.load_state_dict(opt.state_dict())
    q = other.param_groups[0]["params"][0]
    assert other.state[q]["momentum"].dtype == torch.float32 and other.state[q]["master"] is not opt.state[ps[0]]["master"]
    assert other.param_groups[0]["lr"] == 0.5


def test_matrices_of_a_block():
    blk = modules.StrataBlock(64, 2, (3, 3, 3), experts=4)
    names = {id(p): n for n, p in blk.named_parameters()}
    some, rest = matrices(blk)
    assert {names[id(p)] for p in some} == {"attn.qkv.weight", "attn.proj.weight", "mlp.router.weight", "mlp.w1", "mlp.w2"}
    assert {names[id(p)] for p in rest} >= {"mlp.b1", "mlp.b2", "attn.qkv.bias"} and len(some) + len(rest) == len(names)
    Muon(some), AdamW(rest)
