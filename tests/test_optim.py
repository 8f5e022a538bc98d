"""Refusals of the AdamW step and its 8-bit oracle, without a GPU."""

import ctypes

import pytest
import torch

from oracle import optim as O
from strata_amd import _lib, ops
from strata_amd.optim import AdamW


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _call(lib, over=(), tensor=(), second=None):
    t = (_lib.AdamwTensor * 2)()
    for i in range(2):
        base = 0x100000 * (i + 1)
        t[i] = (base, base + 0x10000, base + 0x20000, base + 0x30000, None, None, None, 100, 1e-3, 0.1, _lib.BF16, _lib.BF16, 32, 0)
    for k, v in dict(tensor).items():
        setattr(t[0], k, v)
    for k, v in dict(second or {}).items():
        setattr(t[1], k, v)
    a = _lib.AdamwArgs(t, 2, 0x1000, 0x2000, 0x3000, 0.9, 0.95, 1e-8, 0.0)
    for k, v in dict(over).items():
        setattr(a, k, v)
    rc = lib.strata_hip_adamw_step(ctypes.byref(a), None)
    return rc, lib.strata_hip_last_error().decode()


@pytest.mark.parametrize("over,tensor,second,msg", [
    (dict(step=None), {}, {}, "step"), (dict(workspace=None), {}, {}, "workspace"), (dict(beta1=1.0), {}, {}, "betas"),
    (dict(beta2=-0.1), {}, {}, "betas"), (dict(beta1=float("nan")), {}, {}, "betas"), (dict(eps=-1.0), {}, {}, "eps"),
    (dict(max_norm=float("inf")), {}, {}, "max_norm"), (dict(max_norm=1.0, norm=None), {}, {}, "norm"),
    (dict(count=-1), {}, {}, "list"), ({}, dict(lr=float("nan")), {}, "lr"), ({}, dict(n=-1), {}, "size"),
    ({}, dict(param_dtype=5), {}, "bf16 or f32"), ({}, dict(state_bits=16), {}, "state_bits"), ({}, dict(grad=None), {}, "null"),
    ({}, dict(state_bits=8), {}, "scales"), ({}, dict(param_dtype=0, master=0x900000), {}, "master"),
    ({}, dict(param=0x100001), {}, "aligned"), ({}, {}, dict(param=0x100000), "overlap"),
    ({}, {}, dict(param=0x1000c6), "overlap"), ({}, {}, dict(exp_avg=0x120000), "overlap"),
    ({}, dict(exp_avg=0x130000), {}, "overlap"),
])
def test_c_entry_refuses(lib, over, tensor, second, msg):
    rc, err = _call(lib, over, tensor, second)
    assert rc == _lib.EINVAL and msg in err


@pytest.mark.parametrize("tensor,second,msg", [
    (dict(grad=0x100000), {}, "gradient"), (dict(grad=0x1000c6), {}, "gradient"), ({}, dict(grad=0x130000), "gradient"),
    (dict(grad=0x12018e), {}, "gradient"), (dict(param=0x1000), {}, "overlap"), (dict(exp_avg=0x1004), {}, "overlap"),
])
def test_c_entry_refuses_what_another_tensor_holds(lib, tensor, second, msg):
    """A gradient, which other workgroups read than those that write, and the step count."""
    rc, err = _call(lib, {}, tensor, second)
    assert rc == _lib.EINVAL and msg in err


def test_workspace(lib):
    t = (_lib.AdamwTensor * 3)()
    for i, n in enumerate((1, 16385, 0)):
        t[i].n = n
    assert lib.strata_hip_adamw_workspace(t, 3) == 8 + 1 + 2
    assert lib.strata_hip_adamw_workspace(None, 0) == 8


def test_ops_refuse_cpu_and_bad_lists():
    p = [torch.zeros(4)]
    step = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        ops.adamw_step(p, p, p, p, step)
    with pytest.raises(ValueError, match="one entry"):
        ops.adamw_step(p, [], p, p, step)
    with pytest.raises(ValueError, match="have one entry"):
        ops.adamw_step(p, p, p, p, step, lr=[1e-3, 1e-3])
    with pytest.raises(ValueError, match="GPU"):
        torch.ops.strata_hip.adamw_state_values(torch.zeros(4, dtype=torch.int8), torch.zeros(1))


def test_optimizer_refuses():
    p = [torch.nn.Parameter(torch.zeros(4))]
    for kw, msg in ((dict(state_bits=16), "state_bits"), (dict(betas=(1.0, 0.9)), "betas"), (dict(max_norm=0.0), "max_norm")):
        with pytest.raises(ValueError, match=msg):
            AdamW(p, **kw)
    with pytest.raises(ValueError, match="betas"):
        AdamW([dict(params=p, betas=(0.9, 0.9))])


def test_codes_are_the_nearest():
    """pack / unpack: within half a step of the root's domain, zero exact, the largest value exact to its scale."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1000, generator=g, dtype=torch.float64) * torch.exp(2 * torch.randn(1000, generator=g, dtype=torch.float64))
    x[::17] = 0
    for signed, y in ((True, x), (False, x * x)):
        codes, scale, _ = O.pack(y, signed)
        s = scale.double().repeat_interleave(O.BLOCK)[:1000]
        back = O.unpack(codes, scale)
        steps = 127 if signed else 256
        low = 0 if signed else 1
        r, q = (y.abs() / s).sqrt() * steps, (back.abs() / s).sqrt() * steps
        assert ((r.clamp(min=low) - q).abs() <= 0.5 + 1e-4).all()
        if signed:
            assert (back[y == 0] == 0).all() and (back.sign() * y.sign() >= 0).all()


def test_copies_and_pickles():
    import copy
    import pickle

    p = torch.nn.Parameter(torch.zeros(8))
    opt = AdamW([p], lr=0.5, betas=(0.8, 0.9), eps=1e-6, max_norm=2.0, state_bits=8, master=False, min_8bit=16)
    opt.state[p] = opt._new_state(p, torch.ones(1, dtype=torch.int64))
    for o in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (o.betas, o.eps, o.max_norm, o.state_bits, o.master, o.min_8bit) == ((0.8, 0.9), 1e-6, 2.0, 8, False, 16)
        q = o.param_groups[0]["params"][0]
        assert o.param_groups[0]["lr"] == 0.5 and int(o.state[q]["step"]) == 1 and o.grad_norm is None


def test_c_entry_with_counts_refuses(lib):
    """Each tensor's own count: given, aligned, apart from what is written and read."""
    t = (_lib.AdamwTensor * 2)()
    for i in range(2):
        base = 0x100000 * (i + 1)
        t[i] = (base, base + 0x10000, base + 0x20000, base + 0x30000, None, None, None, 100, 1e-3, 0.1, _lib.BF16, _lib.BF16, 32, 0)
    a = _lib.AdamwArgs(t, 2, None, 0x2000, 0x3000, 0.9, 0.95, 1e-8, 0.0)
    for steps, msg in (((0x1000, None), "step"), ((0x1000, 0x1104), "aligned"), ((0x1000, 0x100000), "overlap"),
                       ((0x1000, 0x110000), "gradient"), ((0x120008, 0x1000), "overlap")):
        rc = lib.strata_hip_adamw_step_counts(ctypes.byref(a), (ctypes.c_void_p * 2)(*steps), None)
        assert rc == _lib.EINVAL and msg in lib.strata_hip_last_error().decode(), steps
    assert lib.strata_hip_adamw_step_counts(ctypes.byref(a), None, None) == _lib.EINVAL


def test_ops_refuse_bad_counts():
    p, step = [torch.zeros(4)] * 2, torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="one for each"):
        ops.adamw_step(p, p, p, p, [step])
    with pytest.raises(ValueError, match="GPU"):
        ops.adamw_step(p, p, p, p, [step, step])


@pytest.fixture
def counted(monkeypatch):
    """AdamW whose steps only count; (the optimizer, its parameters, step(which have gradients), counts)."""
    def fake(params, grads, m, v, step, **kw):
        for t in {id(t): t for t in step}.values():
            t += 1

    monkeypatch.setattr(ops, "adamw_step", fake)
    ps = [torch.nn.Parameter(torch.zeros(4)) for _ in range(4)]
    opt = AdamW(ps)

    def step(which):
        for k, p in enumerate(ps):
            p.grad = torch.ones(4) if k in which else None
        opt.step()

    return opt, ps, step, lambda: [int(opt.state[p]["step"]) if opt.state.get(p) else 0 for p in ps]


def test_each_parameter_counts_its_own_steps(counted):
    """As torch's: late ones, ones left out for a while, a group added later; those alike share a count."""
    opt, ps, step, counts = counted
    ref = torch.optim.AdamW([p.detach().clone().requires_grad_() for p in ps])
    for which in ((0, 1), (0, 1), (0, 1, 2), (0, 2), (2, 3), (0, 1, 2, 3), (1,), (0, 1, 2, 3)):
        for k, q in enumerate(ref.param_groups[0]["params"]):
            q.grad = torch.ones(4) if k in which else None
        ref.step()
        step(which)
        want = [int(ref.state[q]["step"]) if q in ref.state else 0 for q in ref.param_groups[0]["params"]]
        assert counts() == want, which
    late = torch.nn.Parameter(torch.zeros(4))
    opt.add_param_group(dict(params=[late]))
    late.grad = torch.ones(4)
    step(range(4))
    assert int(opt.state[late]["step"]) == 1 and counts() == [w + 1 for w in want]


def test_counts_are_shared_and_survive_a_state_dict(counted):
    opt, ps, step, counts = counted
    step((0, 1))
    step((0, 1, 2, 3))
    assert opt.state[ps[0]]["step"] is opt.state[ps[1]]["step"] and opt.state[ps[2]]["step"] is opt.state[ps[3]]["step"]
    other = AdamW([torch.nn.Parameter(torch.zeros(4)) for _ in ps])
    other.load_state_dict(opt.state_dict())
    loaded = [other.state[p]["step"] for p in other.param_groups[0]["params"]]
    assert [int(t) for t in loaded] == counts() == [2, 2, 1, 1] and loaded[0] is loaded[1] and loaded[2] is loaded[3]
    assert not {id(t) for t in loaded} & {id(s["step"]) for s in opt.state.values()}


def test_a_capture_makes_no_states(counted, monkeypatch):
    """States and counts made inside a capture would be made again by every replay."""
    opt, ps, step, counts = counted
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="eager"):
        step((0, 1))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    step((0, 1))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    step((0, 1))
    with pytest.raises(RuntimeError, match="eager"):
        step((0,))
    assert counts() == [2, 2, 0, 0]


def test_the_package_needs_no_numpy():
    """Imported, and the rows of a step's tensors laid out, where numpy is not installed."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import sys
sys.modules["numpy"] = None
import ctypes, torch
from strata_amd import _lib, ops, optim, modules
rows = []
ops._require_gpu = lambda *a: None
ops._launch = lambda name, a, *r: rows.extend([getattr(a.tensors[i], f) for f, _ in _lib.AdamwTensor._fields_] for i in range(a.count))
p, q = torch.zeros(300, dtype=torch.bfloat16), torch.zeros(5)
g = [torch.zeros(300), torch.zeros(5)]
m, v = [torch.zeros(300, dtype=torch.int8), torch.zeros(5)], [torch.zeros(300, dtype=torch.uint8), torch.zeros(5)]
s, w = [torch.zeros(2), None], [torch.zeros(300), None]
ops.adamw_step([p, q], g, m, v, torch.zeros(1, dtype=torch.int64), lr=[0.1, 0.2], weight_decay=0.3, masters=w, exp_avg_scales=s, exp_avg_sq_scales=s)
a = lambda t: None if t is None else t.data_ptr()
for i, row in enumerate(rows):
    assert row == [a((p, q)[i]), a(g[i]), a(m[i]), a(v[i]), a(s[i]), a(s[i]), a(w[i]), (300, 5)[i], (0.1, 0.2)[i], 0.3,
                   (_lib.BF16, _lib.F32)[i], _lib.F32, (8, 32)[i], 0], row
rows.clear()
ops.adamw_step([], [], [], [], torch.zeros(1, dtype=torch.int64))
assert not rows
"""
    r = subprocess.run([sys.executable, "-W", "ignore", "-c", code], capture_output=True, text=True,
                       cwd=Path(_lib.__file__).resolve().parents[1])
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("count", [1 << 44, 1 << 60])
def test_c_entry_returns_where_a_list_cannot_be_held(count):
    """More tensors than host memory, or than a vector, holds: an error, no exception across the C boundary."""
    import subprocess
    import sys
    from pathlib import Path

    code = f"""
import ctypes
from strata_amd import _lib
lib = _lib.load()
t = (_lib.AdamwTensor * 1)()
a = _lib.AdamwArgs(t, {count}, 0x1000, 0x2000, 0x3000, 0.9, 0.95, 1e-8, 0.0)
assert lib.strata_hip_adamw_step(ctypes.byref(a), None) == _lib.EUNSUPPORTED
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=Path(_lib.__file__).resolve().parents[1])
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
