"""The experts' oracle: closed forms, torch's own pieces, and differences (float64, CPU); refusals of
the operators without a GPU."""

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from oracle import experts as O
from strata_amd import _lib, ops


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def test_one_expert_is_the_dense_mlp():
    x, w1, b1, w2, b2 = _rand(0, 5, 8), _rand(1, 1, 12, 8), _rand(2, 1, 12), _rand(3, 1, 8, 12), _rand(4, 1, 8)
    want = x + F.linear(F.gelu(F.linear(x, w1[0], b1[0]), approximate="tanh"), w2[0], b2[0])
    idx, one = torch.zeros(5, 1, dtype=torch.int32), torch.ones(5, 1, dtype=torch.float64)
    assert torch.allclose(O.mlp(x, one, idx, w1, b1, w2, b2, x), want, rtol=1e-12)
    # the same expert in both slots, weights that sum to one
    both = torch.tensor([[0.25, 0.75]], dtype=torch.float64).expand(5, 2)
    assert torch.allclose(O.mlp(x, both, idx.expand(5, 2), w1, b1, w2, b2, x), want, rtol=1e-12)
    assert torch.equal(O.mlp(x, one, idx - 1, w1, b1, w2, b2, x), x)  # dropped


def test_bounds_values_are_the_definition_and_its_gradients():
    x, w1, b1, w2, b2, res = _rand(0, 7, 8), _rand(1, 3, 8, 8), _rand(2, 3, 8), _rand(3, 3, 16, 8), _rand(4, 3, 16), _rand(5, 7, 16)
    wt = torch.rand(7, 2, generator=torch.Generator().manual_seed(6), dtype=torch.float64)
    idx = torch.tensor([[0, 1], [1, 1], [-1, 2], [2, 0], [-1, -1], [0, 7], [1, 2]], dtype=torch.int32)
    dout = _rand(7, 7, 16)
    leaves = [t.clone().requires_grad_() for t in (x, wt, w1, b1, w2, b2, res)]
    out = O.mlp(leaves[0], leaves[1], idx, *leaves[2:])
    grads = torch.autograd.grad(out, leaves, dout)
    got = O.mlp_bounds(x, wt, idx, w1, b1, w2, b2, res, dout)
    assert torch.allclose(got["out"][0], out, rtol=1e-11, atol=1e-12)
    for n, g in zip(("x", "weights", "w1", "b1", "w2", "b2", "residual"), grads):
        assert torch.allclose(got[n][0], g, rtol=1e-10, atol=1e-11), n
    fn = lambda *a: O.mlp(a[0], a[1], idx, *a[2:])  # noqa: E731
    assert torch.autograd.gradcheck(fn, leaves)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_closed_forms(score, renorm):
    l = _rand(1, 6, 10)
    w, i = O.route(l, 3, score, renormalize=renorm, scale=2.0)
    top = l.topk(3, dim=1)
    assert torch.equal(i.long(), top.indices)
    s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    s = s.gather(1, top.indices)
    want = 2.0 * (s / s.sum(1, keepdim=True) if renorm else s)
    assert torch.allclose(w, want, rtol=1e-12)
    lg = l.clone().requires_grad_()
    assert torch.allclose(O.route_weights(lg, i, score, renorm, 2.0), want, rtol=1e-12)
    assert torch.autograd.gradcheck(lambda a: O.route_weights(a, i, score, renorm, 2.0), lg)


def test_route_bias_groups_ties_and_masks():
    l = torch.tensor([[0.0, 1.0, 1.0, 3.0, 2.0, 2.0]], dtype=torch.float64)
    assert O.route(l, 4)[1].tolist() == [[3, 4, 5, 1]]  # of two equal keys the lower expert
    bias = torch.tensor([10.0, 0, 0, 0, 0, 0])
    w, i = O.route(l, 1, "sigmoid", bias, renormalize=False)
    assert i.tolist() == [[0]] and float(w) == 0.5  # the bias chooses and does not weigh
    # groups (0, 1), (2, 3), (4, 5): the sums of their two best are s(0)+s(1), s(1)+s(3), s(2)+s(2)
    assert O.route(l, 2, "sigmoid", None, 3, 1)[1].tolist() == [[4, 5]]
    assert O.route(l, 2, "softmax", None, 3, 1)[1].tolist() == [[3, 2]]
    m = l.clone()
    m[0, 1:] = -math.inf
    w, i = O.route(m, 3)
    assert i.tolist() == [[0, -1, -1]] and w.tolist() == [[1.0, 0.0, 0.0]]
    m[0, 0] = math.nan
    assert O.route(m, 2)[1].tolist() == [[-1, -1]]


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _route_args(**over):
    a = _lib.ExpertRouteArgs()
    a.logits = a.weights = a.index = a.dweights = a.dlogits = 0x1000
    a.tokens, a.ld, a.dtype, a.experts, a.top_k, a.score = 4, 8, _lib.BF16, 8, 2, 0
    a.groups, a.top_groups, a.renormalize, a.scale = 1, 1, 1, 1.0
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code,msg", [
    (dict(tokens=-1), _lib.EINVAL, "tokens"), (dict(top_k=0), _lib.EINVAL, "top_k"), (dict(dtype=3), _lib.EINVAL, "dtype"),
    (dict(score=2), _lib.EINVAL, "score"), (dict(experts=513, ld=513), _lib.EUNSUPPORTED, "512"),
    (dict(experts=512, ld=512, top_k=65), _lib.EUNSUPPORTED, "64"), (dict(groups=3), _lib.EINVAL, "groups"),
    (dict(groups=4, top_groups=5), _lib.EINVAL, "groups"), (dict(groups=4, top_groups=1, top_k=3), _lib.EINVAL, "exceeds"),
    (dict(top_k=9), _lib.EINVAL, "exceeds"), (dict(ld=7), _lib.EINVAL, "stride"), (dict(scale=math.inf), _lib.EINVAL, "scale"),
    (dict(tokens=1 << 31), _lib.EUNSUPPORTED, "pairs"), (dict(index=None), _lib.EINVAL, "null"),
])
def test_route_refusals(lib, over, code, msg):
    a = _route_args(**over)
    for fn in (lib.strata_hip_expert_route, lib.strata_hip_expert_route_bwd):
        assert fn(ctypes.byref(a), None) == code and msg in lib.strata_hip_last_error().decode()
    a = _route_args(tokens=0, logits=None, index=None)
    assert lib.strata_hip_expert_route(ctypes.byref(a), None) == 0


def test_plan_refusals_and_sizes(lib):
    assert lib.strata_hip_expert_plan_workspace(1024, 8) == 0 and lib.strata_hip_expert_plan_workspace(1025, 8) == 16
    for over, code in ((dict(pairs=-1), _lib.EINVAL), (dict(experts=0), _lib.EINVAL), (dict(tile=0), _lib.EINVAL),
                       (dict(experts=513), _lib.EUNSUPPORTED), (dict(offsets=None), _lib.EINVAL),
                       (dict(row_token=None), _lib.EINVAL), (dict(weights=None), _lib.EINVAL), (dict(top_k=3), _lib.EINVAL), (dict(pairs=2000, workspace=None), _lib.EINVAL)):
        a = _lib.ExpertPlanArgs(*[0x1000] * 8, 100, 2, 8, 64, 0)
        for k, v in over.items():
            setattr(a, k, v)
        assert lib.strata_hip_expert_plan(ctypes.byref(a), None) == code, over


def _mlp_args(lib, **over):
    a = _lib.ExpertMlpArgs(*[0x1000] * 16, 16, 64, 64, 2, 8, 64, 128, 64, 0)
    for k, v in over.items():
        setattr(a, k, v)
    if a.tile == 0:
        a.tile = lib.strata_hip_expert_tile(a.tokens * a.top_k, a.experts, a.dim, a.hidden, a.out_dim, a.dact is not None)
    return a


@pytest.mark.parametrize("over,code,msg", [
    (dict(tokens=-1), _lib.EINVAL, "sizes"), (dict(dim=60), _lib.EINVAL, "multiples"), (dict(hidden=4), _lib.EINVAL, "multiples"),
    (dict(out_dim=0), _lib.EINVAL, "sizes"), (dict(experts=513), _lib.EUNSUPPORTED, "512"), (dict(tile=3), _lib.EINVAL, "tile"),
    (dict(w1=0x1008), _lib.EINVAL, "aligned"), (dict(b1=0x1004), _lib.EINVAL, "aligned"), (dict(x=None), _lib.EINVAL, "null"),
    (dict(h=None), _lib.EINVAL, "null"), (dict(ldx=60), _lib.EINVAL, "stride"), (dict(ldx=56), _lib.EINVAL, "stride"),
    (dict(tokens=1 << 24), _lib.EUNSUPPORTED, "2 GiB"), (dict(x=0x1002), _lib.EINVAL, "aligned"),
])
def test_mlp_refusals(lib, over, code, msg):
    a = _mlp_args(lib, **over)
    assert lib.strata_hip_expert_mlp(ctypes.byref(a), None) == code and msg in lib.strata_hip_last_error().decode()
    b = _lib.ExpertMlpBwdArgs(a, *[0x1000] * 9)
    assert lib.strata_hip_expert_mlp_bwd(ctypes.byref(b), None) == code


@pytest.mark.parametrize("over,msg", [
    (dict(dout=None), "dout"), (dict(gz=None), "gz"), (dict(dxs=None), "dxs"),
    (dict(dw2=None), "bias gradient"), (dict(dw1=None), "bias gradient"), (dict(dx=0x1008), "aligned"),
])
def test_mlp_bwd_refusals(lib, over, msg):
    b = _lib.ExpertMlpBwdArgs(_mlp_args(lib), *[0x1000] * 9)
    for k, v in over.items():
        setattr(b, k, v)
    assert lib.strata_hip_expert_mlp_bwd(ctypes.byref(b), None) == _lib.EINVAL
    assert msg in lib.strata_hip_last_error().decode()
    if "dout" in over:
        b.fwd.out = None
        assert lib.strata_hip_expert_mlp(ctypes.byref(b.fwd), None) == _lib.EINVAL


def test_ops_refuse_cpu_tensors():
    with pytest.raises(ValueError, match="GPU"):
        ops.expert_route(torch.zeros(2, 8), 2)
    x, w = torch.zeros(2, 8).bfloat16(), torch.zeros(2, 1).bfloat16()
    w1, w2 = torch.zeros(3, 16, 8).bfloat16(), torch.zeros(3, 8, 16).bfloat16()
    with pytest.raises(ValueError, match="GPU"):
        ops.expert_mlp(x, w, torch.zeros(2, 1, dtype=torch.int32), w1, None, w2, None)


def test_expert_modules_without_a_gpu():
    from strata_amd.modules import ExpertMlp, StrataBlock, init_xavier_

    blk = StrataBlock(64, 1, (3, 3, 3), experts=4, expert_options=dict(top_k=1, balance=True))
    names = [n for n, _ in blk.named_parameters()]
    assert names == ["attn.qkv.weight", "attn.qkv.bias", "attn.proj.weight", "attn.proj.bias", "mlp.w1", "mlp.b1", "mlp.w2",
                     "mlp.b2", "mlp.router.weight"]
    init_xavier_(blk, torch.Generator().manual_seed(0))
    assert float(blk.mlp.w1.detach().abs().max()) <= (6 / (64 + 256)) ** 0.5 and not blk.mlp.b1.any()
    blk.mlp.balance[1] = 1 / 3
    blk.bfloat16()
    assert blk.mlp.balance.dtype == torch.float32 and float(blk.mlp.balance[1]) == float(torch.tensor(1 / 3))
    assert blk.mlp.w1.dtype == torch.bfloat16 and "mlp.balance" in blk.state_dict()
    with pytest.raises(ValueError, match="not a choice"):
        ExpertMlp(64, 64, 4, top_k=5)
    with pytest.raises(ValueError, match="not a choice"):
        ExpertMlp(64, 64, 8, top_k=3, groups=4, top_groups=1)
    with pytest.raises(ValueError, match="score"):
        ExpertMlp(64, 64, 4, score="tanh")
    assert [n for n, _ in StrataBlock(64, 1, (3, 3, 3)).named_parameters()][4:] == [
        "mlp.layers.0.weight", "mlp.layers.0.bias", "mlp.layers.2.weight", "mlp.layers.2.bias"]


def test_traced_shapes():
    """The custom ops under fake tensors: shapes, types and strides of what the kernels write."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=True):
        e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        w, i = ops.expert_route(e(5, 7, 8, dtype=torch.float32), 2)
        assert w.shape == i.shape == (5, 7, 2) and (w.dtype, i.dtype) == (torch.float32, torch.int32)
        assert torch.ops.strata_hip.expert_route_bwd(w, e(5, 7, 8, dtype=torch.float32), i, 2, "softmax", None, True, 1.0).shape == (5, 7, 8)
        x, wt = e(7, 5, 64).transpose(0, 1), e(5, 7, 2)
        w1, w2 = e(4, 64, 96).transpose(1, 2), e(4, 32, 96)
        out = ops.expert_mlp(x, wt, i, w1, None, w2, e(4, 32))
        assert out.shape == (5, 7, 32) and out.dtype == torch.bfloat16
        out, space = torch.ops.strata_hip.expert_mlp_train(x, wt, i, w1, None, w2, e(4, 32), None)
        tile = ops._expert_tile(70, w1, w2, True)
        assert out.shape == (5, 7, 32) and space.dtype == torch.uint8 and space.numel() == ops._expert_space(70, 4, 96, 32, tile, True)[4]
        need = [True, False, True, False, True, True]
        g = torch.ops.strata_hip.expert_mlp_bwd(out, x, wt, w1, None, w2, e(4, 32), space, need)
        assert [tuple(t.shape) for t in g] == [(5, 7, 64), (0,), (4, 96, 64), (0,), (4, 32, 96), (4, 32)]
        assert all(t.is_contiguous() for t in g)
        v = ops.adamw_state_values(e(300, dtype=torch.int8), e(2, dtype=torch.float32))
        assert v.shape == (300,) and v.dtype == torch.float32


STRUCTS = {"strata_hip_expert_route_args": _lib.ExpertRouteArgs, "strata_hip_expert_plan_args": _lib.ExpertPlanArgs,
           "strata_hip_expert_mlp_args": _lib.ExpertMlpArgs, "strata_hip_expert_mlp_bwd_args": _lib.ExpertMlpBwdArgs,
           "strata_hip_adamw_tensor": _lib.AdamwTensor, "strata_hip_adamw_args": _lib.AdamwArgs,
           "strata_hip_adamw_values_args": _lib.AdamwValuesArgs}


def test_struct_layouts_are_the_header_s(tmp_path):
    """Every field's offset and every structure's size, as a C compiler lays the header out."""
    header = Path(_lib.__file__).resolve().parents[1] / "include" / "strata_hip.h"
    lines = [f'#include "{header}"', "#include <stddef.h>", "#include <stdio.h>", "int main(void) {"]
    want = []
    for name, st in STRUCTS.items():
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


def test_kernels_without_a_plan_read_an_index_once():
    """They check the index that they read and form addresses from it: a second read would not be the checked one."""
    src = (Path(_lib.__file__).resolve().parent / "csrc" / "expert.hip").read_text()
    for kernel in ("void expert_few_kernel(", "void expert_few_out_kernel("):
        body = src[src.index(kernel):]
        assert body[: body.index("\n}\n")].count("p.index[") == 1, kernel
