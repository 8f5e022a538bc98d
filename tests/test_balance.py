"""The balance of the routing on the CPU: its oracle, its refusals, and what traces, transforms and watches see of it."""

import ctypes

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from oracle import experts as O
from strata_amd import _lib, modules, ops


def formula(logits, index, score, sequences, gb, gz):
    """The gradient at float64 logits [T, E], and the magnitude of what it is summed of."""
    T, E = logits.shape
    per, k = T // sequences, index.shape[1]
    ok = torch.isfinite(logits)
    some = ok.any(1)
    l = torch.where(ok, logits, -torch.inf)
    lse = torch.where(some, torch.logsumexp(l, 1), 0.0)
    soft = torch.softmax(l, 1).nan_to_num(0.0)
    s, om = soft, torch.ones_like(soft)
    if score == "sigmoid":
        s = torch.softmax(torch.where(ok, torch.nn.functional.logsigmoid(logits.nan_to_num(0.0, 0.0, 0.0)), -torch.inf), 1).nan_to_num(0.0)
        om = torch.sigmoid(-l)
    n = some.view(sequences, per).sum(1)
    f = torch.zeros(sequences, E, dtype=torch.float64)
    for g in range(sequences):
        i = index[g * per:(g + 1) * per].reshape(-1).long()
        i = i[(i >= 0) & (i < E)]
        f[g] = i.bincount(minlength=E).double() * E / (k * max(int(n[g]), 1) ** 2 * max(int((n > 0).sum()), 1))
    f = f.repeat_interleave(per, 0)
    mean = (f * s).sum(1, keepdim=True)
    zc = gz * 2 / max(int(n.sum()), 1)
    grad = torch.where(ok, gb * s * (f - mean) * om + zc * lse[:, None] * soft, 0.0)
    return grad, torch.where(ok, abs(gb) * s * (f + mean) * om + abs(zc) * lse[:, None].abs() * soft, 0.0)


def routed(T, E, k, masked, seed, dtype=torch.float64):
    """Logits with masked experts, tokens and a masked run at the start, and an index with repeated, empty and foreign entries."""
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(T, E, generator=g) * 2).to(dtype)
    if masked:
        logits[torch.rand(T, E, generator=g) < masked] = -torch.inf
        logits[::7] = torch.nan
        logits[1::11, 0] = torch.inf
    index = torch.randint(-2, E + 2, (T, k), generator=g, dtype=torch.int32)
    return logits, index


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,sequences,masked", [(1, 1, 1, 1, 0.0), (6, 4, 2, 3, 0.0), (24, 5, 3, 2, 0.3), (21, 8, 1, 3, 0.6)])
def test_oracle_gradient(score, T, E, k, sequences, masked):
    """Autograd of the oracle, the formula, and differences of the oracle agree."""
    logits, index = routed(T, E, k, masked, 1)
    leaf = logits.clone().requires_grad_()
    b, z, _ = O.balance(leaf, index, score, sequences)
    loss = 0.7 * b + 0.3 * z
    want = torch.autograd.grad(loss, leaf)[0].nan_to_num(0.0) if loss.requires_grad else torch.zeros_like(logits)
    grad, _ = formula(logits, index, score, sequences, 0.7, 0.3)
    assert torch.allclose(grad, want, rtol=1e-12, atol=1e-14)
    at = [(t, e) for t in range(T) for e in range(E) if torch.isfinite(logits[t, e])][:: max(1, T * E // 12)]
    for t, e in at:
        ends = []
        for h in (1e-5, -1e-5):
            moved = logits.clone()
            moved[t, e] += h
            b, z, _ = O.balance(moved, index, score, sequences)
            ends.append(float(0.7 * b + 0.3 * z))
        assert abs((ends[0] - ends[1]) / 2e-5 - float(grad[t, e])) <= 1e-8


def test_even_load_has_balance_one():
    index = torch.arange(8, dtype=torch.int32)[:, None]
    b, z, load = O.balance(torch.zeros(8, 8, dtype=torch.float64), index)
    assert abs(float(b) - 1) < 1e-14 and load.tolist() == [1] * 8 and abs(float(z) - torch.tensor(8.0).log() ** 2) < 1e-6


def test_refusals():
    l, i = torch.randn(6, 4), torch.zeros(6, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.expert_balance(l, i)


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda name, *a: seen.append(name))
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: torch.device("cpu"))
    return seen


@pytest.mark.parametrize("logits,index,kw,match", [
    (torch.randn(6, 4), torch.zeros(6, 2, dtype=torch.int64), {}, "index must be int32"),
    (torch.randn(6, 4), torch.zeros(5, 2, dtype=torch.int32), {}, "index must be int32"),
    (torch.randn(6, 4), torch.zeros(6, dtype=torch.int32), {}, "index must be int32"),
    (torch.randn(6, 4), torch.zeros(6, 0, dtype=torch.int32), {}, "index must be int32"),
    (torch.randn(6, 4), torch.zeros(6, 2, dtype=torch.int32), dict(score="relu"), "score"),
    (torch.randn(6, 4), torch.zeros(6, 2, dtype=torch.int32), dict(sequences=4), "whole number"),
    (torch.randn(6, 4), torch.zeros(6, 2, dtype=torch.int32), dict(sequences=0), "whole number"),
    (torch.randn(6, 4), torch.zeros(6, 2, dtype=torch.int32), dict(sequences=-1), "whole number"),
    (torch.randn(6, 4).half(), torch.zeros(6, 2, dtype=torch.int32), {}, "dtype"),
    (torch.randn(6, 0), torch.zeros(6, 2, dtype=torch.int32), {}, "experts"),
])
def test_refused_arguments(launches, logits, index, kw, match):
    with pytest.raises(ValueError, match=match):
        ops.expert_balance(logits, index, **kw)
    assert not launches


def test_a_fraction_of_a_sequence_is_refused(launches):
    with pytest.raises(TypeError, match="integer"):
        ops.expert_balance(torch.randn(6, 4), torch.zeros(6, 2, dtype=torch.int32), sequences=1.5)
    assert not launches


def test_refused_by_the_library():
    lib = _lib.load()
    a = _lib.ExpertBalanceArgs()

    def bad(code, text, call=lib.strata_hip_expert_balance):
        assert call(ctypes.byref(a), None) == code and text in lib.strata_hip_last_error().decode()

    assert lib.strata_hip_expert_balance(None, None) == _lib.EINVAL
    a.tokens, a.sequences, a.experts, a.top_k, a.ld = 6, 1, 0, 2, 8
    bad(_lib.EINVAL, "experts")
    a.experts, a.sequences = 8, 4
    bad(_lib.EINVAL, "whole number")
    a.sequences, a.dtype = 3, 9
    bad(_lib.EINVAL, "dtype")
    a.dtype, a.score = _lib.BF16, 2
    bad(_lib.EINVAL, "score")
    a.score, a.experts = 0, 513
    bad(_lib.EUNSUPPORTED, "512")
    a.experts, a.ld = 8, 7
    bad(_lib.EINVAL, "stride")
    a.ld = 8
    bad(_lib.EINVAL, "state")
    a.state = 0x1000
    bad(_lib.EINVAL, "null")
    a.logits = 0x1000
    bad(_lib.EINVAL, "null")
    a.balance = a.z = a.load = a.index = 0x1000
    bad(_lib.EINVAL, "workspace")
    a.workspace = 0x1004
    bad(_lib.EINVAL, "workspace")
    bad(_lib.EINVAL, "null", lib.strata_hip_expert_balance_bwd)
    a.tokens, a.sequences = 1 << 30, 1
    bad(_lib.EUNSUPPORTED, "2^31")
    a.tokens = a.sequences = 1 << 17
    bad(_lib.EUNSUPPORTED, "sequences")
    a.tokens = 0
    a.sequences = 1
    assert lib.strata_hip_expert_balance_bwd(ctypes.byref(a), None) == _lib.OK


def _call(l):
    return ops.expert_balance(l, torch.zeros(6, 2, dtype=torch.int32))[0]


def test_traces_and_transforms_see_the_op(launches):
    x = torch.randn(6, 4)
    assert "strata_hip.expert_balance.default" in [str(n.target) for n in make_fx(_call)(x).graph.nodes]
    grad = lambda x: torch.autograd.grad(_call(x), x)[0]  # noqa: E731
    targets = [str(n.target) for n in make_fx(grad)(x.clone().requires_grad_()).graph.nodes]
    assert "strata_hip.expert_balance_bwd.default" in targets
    with torch.no_grad():
        assert "strata_hip::expert_balance" in str(torch.jit.trace(_call, x, check_trace=False).graph)
    assert torch.vmap(_call)(torch.stack([x, x, x])).shape == (3,)


def test_either_loss_alone_has_a_gradient(launches):
    x = torch.randn(6, 4, requires_grad=True)
    for pick in (0, 1):
        launches.clear()
        out = ops.expert_balance(x, torch.zeros(6, 2, dtype=torch.int32))[pick]
        assert torch.autograd.grad(out, x)[0].shape == x.shape and launches == ["strata_hip_expert_balance", "strata_hip_expert_balance_bwd"]


def test_differentiable_once(launches):
    x = torch.randn(6, 4, requires_grad=True)
    b = ops.expert_balance(x, torch.zeros(6, 2, dtype=torch.int32))[0]
    (g,) = torch.autograd.grad(b, x, create_graph=True)
    with pytest.raises(RuntimeError, match="forward-only"):
        torch.autograd.grad(g.sum(), x)


def test_backward_takes_the_saved_tensors_as_they_come_back(launches, monkeypatch):
    """Of another place, type or layout where hooks changed them; strided logits; a graph kept and run twice."""
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda name, a, t, *r: seen.append((name, a.logits, a.dlogits, a.dtype, a.ld, a.tokens)))
    index = torch.zeros(6, 2, dtype=torch.int32)
    for change, code in ((lambda t: t.clone(), _lib.F32), (lambda t: t.bfloat16() if t.dim() == 2 else t, _lib.BF16),
                         (lambda t: t.t().contiguous().t() if t.dim() == 2 else t, _lib.F32)):
        x = torch.randn(6, 4, requires_grad=True)
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: kept.append(change(t)) or kept[-1]):
            b = ops.expert_balance(x, index)[0]
        seen.clear()
        for _ in range(2):
            g = torch.autograd.grad(b, x, retain_graph=True)[0]
        assert g.shape == x.shape and [s[0] for s in seen] == ["strata_hip_expert_balance_bwd"] * 2
        assert {s[3] for s in seen} == {code} and all(s[4:] == (4, 6) for s in seen)
        if change(x.detach()).is_contiguous():
            assert [s[1] for s in seen] == [t.data_ptr() for t in kept if t.dim() == 2]
    wide = torch.randn(6, 9, requires_grad=True)
    seen.clear()
    torch.autograd.grad(ops.expert_balance(wide[:, 1:5], index)[1], wide)
    assert [s[4] for s in seen] == [9, 9]


def test_compiled_with_its_gradient(launches):
    i = torch.zeros(6, 2, dtype=torch.int32)
    torch._dynamo.reset()
    f = torch.compile(lambda l: sum(ops.expert_balance(l, i, "sigmoid", 2)[:2]), backend="aot_eager", fullgraph=True)
    x = torch.randn(6, 4, requires_grad=True)
    assert torch.autograd.grad(f(x), x)[0].shape == x.shape


def test_routing_losses_collects(launches, monkeypatch):
    monkeypatch.setattr(ops, "gemm_bias_act", lambda x, w, *a: x @ w.T)
    mlp = modules.ExpertMlp(16, 24, 4)
    x = torch.randn(2, 3, 16)
    mlp.route(x)
    assert launches == ["strata_hip_expert_route"]
    with modules.RoutingLosses(per_sample=True) as outer:
        mlp.route(x)
        with modules.RoutingLosses() as inner:
            mlp.route(x)
            mlp.route(x)
        mlp.route(x[0])
    mlp.route(x)
    assert [m for m, _ in outer.load] == [mlp] * 2 and len(inner.load) == 2 and outer.balance.shape == () and inner.z.requires_grad
    assert launches.count("strata_hip_expert_balance") == 4 and not modules.RoutingLosses._active()
    assert modules.RoutingLosses().balance is None
    with pytest.raises(KeyError):
        with modules.RoutingLosses():
            raise KeyError
    assert not modules.RoutingLosses._active()
