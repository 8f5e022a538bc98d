"""The optimizers' states and arguments, without a GPU."""

import pytest
import torch

from strata_amd import ops
from strata_amd.optim import AdamW, Muon, matrices


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda name, *a: seen.append(name))
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: torch.device("cpu"))
    return seen


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64, torch.float16])
def test_states_are_fp32_whatever_torch_makes_by_default(launches, default):
    """A model built under ``torch.set_default_dtype`` steps all the same."""
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(default)
        for make in (Muon, AdamW, lambda ps: AdamW(ps, state_bits=8, min_8bit=1)):
            for dtype in (torch.bfloat16, torch.float32):
                p = torch.nn.Parameter(torch.ones(4, 300, dtype=dtype))
                p.grad = torch.ones_like(p)
                opt = make([p])
                opt.step()
                state = {k: v.dtype for k, v in opt.state[p].items() if k != "step"}
                assert set(state.values()) <= {torch.float32, torch.int8, torch.uint8}, state
    finally:
        torch.set_default_dtype(before)
    assert len(launches) == 6


def test_coefficients_that_can_be_read_once(launches):
    """An iterator's triples are the optimizer's, not the check's alone."""
    p = torch.nn.Parameter(torch.ones(4, 6))
    opt = Muon([p], coefficients=iter([(1.5, -0.5, 0.0)] * 3))
    assert opt.coefficients == ((1.5, -0.5, 0.0),) * 3


@pytest.mark.parametrize("steps", [2.7, 3.0, "3"])
def test_a_fraction_of_a_step_is_refused(launches, steps):
    x = torch.ones(4, 6)
    for call in (lambda: ops.orthogonalize(x, steps=steps), lambda: ops.muon_step([x], [x], [x], steps=steps), lambda: Muon([torch.nn.Parameter(x)], steps=steps)):
        with pytest.raises(TypeError, match="integer"):
            call()
    assert not launches


def test_an_embedding_that_a_linear_layer_shares_is_no_matrix():
    net = torch.nn.ModuleList([torch.nn.Linear(6, 8, bias=False), torch.nn.Embedding(9, 6), torch.nn.Linear(6, 9, bias=False)])
    net[2].weight = net[1].weight
    some, rest = matrices(net)
    assert [p is q for p, q in zip(some + rest, (net[0].weight, net[1].weight))] == [True, True] and len(some) == len(rest) == 1
