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
