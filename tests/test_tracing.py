"""The experts' operators and the 8-bit moments' values where something traces, transforms or watches the calls: it sees the
custom ops.  On the CPU, with the launches left out."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from strata_amd import ops

BF16 = torch.bfloat16


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda name, *a: seen.append(name))
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: None)
    monkeypatch.setattr(ops, "_expert_check", lambda *a: None)
    return seen


def _mlp_args(T=6, E=4, k=2, C=16, H=24):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(BF16)  # noqa: E731
    return r(T, C), r(T, k), torch.randint(0, E, (T, k), generator=g, dtype=torch.int32), r(E, H, C), None, r(E, C, H), r(E, C)


def _route(l):
    return ops.expert_route(l, 2)[0]


def _values(c):
    return ops.adamw_state_values(c, torch.ones(1))


def _calls():
    x, *rest = _mlp_args()
    return {"route": (_route, torch.randn(6, 8), "expert_route"), "mlp": (lambda x: ops.expert_mlp(x, *rest), x, "expert_mlp_fwd"),
            "values": (_values, torch.zeros(8, dtype=torch.int8), "adamw_state_values")}


@pytest.mark.parametrize("which", ["route", "mlp", "values"])
def test_make_fx_records_the_op(launches, which):
    f, x, op = _calls()[which]
    targets = [str(n.target) for n in make_fx(f)(x).graph.nodes]
    assert f"strata_hip.{op}.default" in targets, targets


@pytest.mark.parametrize("which", ["route", "mlp"])
def test_make_fx_records_the_backward(launches, which):
    f, x, op = _calls()[which]
    grad = lambda x: torch.autograd.grad(f(x).sum(), x)[0]  # noqa: E731
    targets = [str(n.target) for n in make_fx(grad)(x.clone().requires_grad_()).graph.nodes]
    op = op.replace("_fwd", "")
    assert f"strata_hip.{op}_bwd.default" in targets and any(f"strata_hip.{op}" in t and "bwd" not in t for t in targets), targets


@pytest.mark.parametrize("which", ["route", "mlp"])
def test_a_backward_alone_is_recorded(launches, which):
    """The forward outside the trace, the gradient inside."""
    f, x, op = _calls()[which]
    x = x.clone().requires_grad_()
    y = f(x)
    targets = [str(n.target) for n in make_fx(lambda d: torch.autograd.grad(y, x, d, retain_graph=True)[0])(torch.ones_like(y)).graph.nodes]
    assert f"strata_hip.{op.replace('_fwd', '')}_bwd.default" in targets, targets


@pytest.mark.parametrize("which", ["route", "mlp", "values"])
def test_jit_trace_records_the_op(launches, which):
    f, x, op = _calls()[which]
    with torch.no_grad():
        assert f"strata_hip::{op}" in str(torch.jit.trace(f, x, check_trace=False).graph)


@pytest.mark.parametrize("which", ["route", "mlp", "values"])
def test_modes_see_the_op(launches, which):
    f, x, op = _calls()[which]
    seen = []

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    for mode in (Dispatch, Function):
        seen.clear()
        with mode():
            f(x)
        assert any(op in s for s in seen), (mode, seen)


@pytest.mark.parametrize("which", ["route", "mlp", "values"])
def test_vmap(launches, which):
    f, x, _ = _calls()[which]
    assert torch.vmap(f)(torch.stack([x, x, x])).shape[0] == 3 and len(launches) >= 3


def test_batched_gradients_of_the_routing(launches):
    x = torch.randn(6, 8, requires_grad=True)
    (g,) = torch.autograd.grad(_route(x), x, torch.ones(3, 6, 2), is_grads_batched=True)
    assert g.shape == (3, 6, 8) and launches.count("strata_hip_expert_route_bwd") == 3


@pytest.mark.parametrize("which", ["route", "mlp", "values"])
def test_plain_calls_take_the_short_path(launches, monkeypatch, which):
    f, x, op = _calls()[which]

    def no(*a, **k):
        raise AssertionError("custom op called")

    for name in ("_expert_route_op", "expert_mlp_fwd", "expert_mlp_train", "_state_values_op"):
        monkeypatch.setattr(ops, name, no)
    f(x)
    with torch.device("cpu"):
        f(x)
    assert launches


def test_a_trace_of_the_step_is_refused():
    t = [torch.zeros(4)]
    with pytest.raises(RuntimeError, match="trace"):
        make_fx(lambda p: ops.adamw_step([p], t, t, t, torch.zeros(1, dtype=torch.int64)))(torch.zeros(4))


def test_compiled_inference_takes_the_inference_op(launches):
    """With gradients enabled but asked of nothing: the op that keeps nothing."""
    _, *rest = _mlp_args()
    seen = []

    def backend(gm, _example):
        seen.extend(str(n.target) for n in gm.graph.nodes)
        return gm.forward

    torch._dynamo.reset()
    torch.compile(lambda x: ops.expert_mlp(x, *rest), backend=backend, fullgraph=True)(_mlp_args()[0])
    assert any("expert_mlp_fwd" in t for t in seen) and not any("expert_mlp_train" in t for t in seen), seen


def test_training_leaves_the_number_of_tokens_open():
    """The workspace's size under fake tensors is arithmetic of the tokens, and no size becomes a constant."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext

    env = ShapeEnv()
    x, w, i, w1, b1, w2, b2 = _mlp_args(T=90)
    with FakeTensorMode(shape_env=env) as mode:
        open_rows = StatelessSymbolicContext(dynamic_sizes=[DimDynamic.DYNAMIC, DimDynamic.STATIC])
        x, w, i = (mode.from_tensor(t, symbolic_context=open_rows, static_shapes=False) for t in (x, w, i))
        w1, w2, b2 = (mode.from_tensor(t, static_shapes=True) for t in (w1, w2, b2))
        out, space = torch.ops.strata_hip.expert_mlp_train(x, w, i, w1, b1, w2, b2, None)
        grads = torch.ops.strata_hip.expert_mlp_bwd(out, x, w, w1, b1, w2, b2, space, [True, True, True, False, True, True])
    for size in (x.shape[0], out.shape[0], space.shape[0], grads[0].shape[0]):
        assert isinstance(size, torch.SymInt) and size.node.expr.free_symbols, size
    assert not env.replacements, env.replacements


@pytest.mark.parametrize("train", [False, True])
def test_compiled_once_for_every_number_of_tokens(launches, train):
    from torch._dynamo.testing import CompileCounterWithBackend

    *_, w1, b1, w2, b2 = _mlp_args()
    w1.requires_grad_(train)
    counter = CompileCounterWithBackend("aot_eager")
    torch._dynamo.reset()
    f = torch.compile(lambda x, w, i: ops.expert_mlp(x, w, i, w1, b1, w2, b2), backend=counter, fullgraph=True, dynamic=True)
    for T in (6, 90, 33, 5000):
        y = f(*_mlp_args(T)[:3])
        if train:
            torch.autograd.grad(y.sum(), w1)
    assert counter.frame_count == 1


def test_training_workspace_holds_every_plan():
    """Its size is taken for the smallest tile: no tile under a backward is smaller, no plan's workspace larger."""
    from strata_amd import _lib

    lib = _lib.load()
    for n in (1, 63, 1023, 1024, 1025, 4000, 70001, 1 << 20):
        for E in (1, 8, 60, 512):
            dact, y, plan, ws, size = ops._expert_space(n, E, 64, 64, 64, True)
            assert size - ws >= 4 * lib.strata_hip_expert_plan_workspace(n, E)
            for width in (8, 768, 4096):
                tile = lib.strata_hip_expert_tile(n, E, width, width, width, 1)
                assert tile >= ops._TRAIN_TILE and ws - plan >= 4 * ops._plan_size(n, E, tile)


def test_vmap_over_a_leaf_keeps_its_gradient(launches):
    """Under vmap the tensors' wrappers show no wish for gradients; the leaves behind them have one."""
    x, w, i, w1, _, w2, b2 = _mlp_args()
    w1.requires_grad_()
    xs = torch.stack([x, x, x]).requires_grad_()
    out = torch.vmap(lambda x: ops.expert_mlp(x, w, i, w1, None, w2, b2))(xs)
    gx, g1 = torch.autograd.grad(out.sum(), [xs, w1])
    assert gx.shape == xs.shape and g1.shape == w1.shape and launches.count("strata_hip_expert_mlp_bwd") == 3
