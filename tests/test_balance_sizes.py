"""Sizes that the balance of the routing does not take, without a GPU."""

import pytest
import torch

from strata_amd import _lib, ops


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda name, *a: seen.append(name))
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: torch.device("cpu"))
    return seen


@pytest.mark.parametrize("experts", [513, 1024, 2048, 2049, 1 << 20, (1 << 30) + 1, (1 << 31) - 1])
def test_workspace_of_too_many_experts(experts):
    lib = _lib.load()
    assert lib.strata_hip_expert_balance_workspace(1000, 1, experts) == -1
    assert "512 experts" in lib.strata_hip_last_error().decode()


def test_workspace_of_sizes_at_the_limits():
    ws = _lib.load().strata_hip_expert_balance_workspace
    for tokens, sequences in ((1, 1), (65536, 65536), ((1 << 31) - 1, 1)):
        for experts in (1, 8, 9, 512):
            assert ws(tokens, sequences, experts) >= sequences * (12 + 8 * experts)
    assert ws(0, 3, 8) == ws(4, 0, 8) == ws(4, 1, 0) == ws(-1, 1, 8) == ws(4, 1, -5) == 0
    assert ws(1 << 31, 1, 8) == ws(1 << 17, 1 << 17, 8) == -1


@pytest.mark.parametrize("experts", [513, 2049, 70000])
def test_too_many_experts_are_refused(launches, experts):
    with pytest.raises(_lib.StrataHipError, match="512 experts"):
        ops.expert_balance(torch.zeros(3, experts), torch.zeros(3, 1, dtype=torch.int32))
    assert not launches


@pytest.mark.parametrize("rows,sequences", [(0, 1 << 50), (0, 1 << 64), (0, (1 << 64) + 1), (6, 1 << 50), (6, -(1 << 50)), (0, 0)])
def test_numbers_of_sequences_are_checked_before_anything_is_allocated(launches, rows, sequences):
    with pytest.raises(ValueError, match="whole number"):
        ops.expert_balance(torch.zeros(rows, 4), torch.zeros(rows, 1, dtype=torch.int32), sequences=sequences)
    assert not launches


def test_too_many_sequences_are_refused(launches):
    with pytest.raises(_lib.StrataHipError, match="65536 sequences"):
        ops.expert_balance(torch.zeros(65537, 2), torch.zeros(65537, 1, dtype=torch.int32), sequences=65537)
    ops.expert_balance(torch.zeros(65536, 2), torch.zeros(65536, 1, dtype=torch.int32), sequences=65536)
    assert launches == ["strata_hip_expert_balance"]


def test_one_number_is_no_row_of_logits(launches):
    with pytest.raises(ValueError, match="index must be int32"):
        ops.expert_balance(torch.zeros(()), torch.zeros((), dtype=torch.int32))
    assert not launches
