"""CPU-only tests of the operators over ragged groups: what they refuse, before anything runs."""
import pytest
import torch

from mcmc_amd import RowGroups, group_rows, grouped_linear, philox_dropout


def groups(rows, n, order=True):
    return RowGroups(torch.arange(rows, dtype=torch.int32) if order else None, torch.linspace(0, rows, n + 1).to(torch.int32))


def test_there_is_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        group_rows(torch.zeros(4, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        grouped_linear(torch.zeros(4, 3), torch.zeros(2, 5, 3), groups(4, 2))
    with pytest.raises(RuntimeError, match="no CPU path"):
        philox_dropout(torch.zeros(4, 3), 0.1, 0)


@pytest.mark.parametrize("ids, n, text", [
    (torch.zeros(2, 2, dtype=torch.int64), 2, "1-D"),
    (torch.zeros(4, dtype=torch.int16), 2, "int32 or int64"),
    (torch.zeros(4), 2, "int32 or int64"),
    (torch.zeros(4, dtype=torch.int32), 0, "n_groups"),
    (torch.zeros(4, dtype=torch.int32), 4097, "n_groups"),
    (torch.zeros(4, dtype=torch.int32), 2 ** 32 + 1, "n_groups"),
])
def test_group_rows_refuses(ids, n, text):
    with pytest.raises(ValueError, match=text):
        group_rows(ids, n)


@pytest.mark.parametrize("change, text", [
    (dict(x=torch.zeros(3)), "x must be"),
    (dict(x=torch.zeros(4, 2)), "Expected 3 input features, got 2"),
    (dict(x=torch.zeros(4, 3, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(x=torch.zeros(4, 3, dtype=torch.float16)), "one type"),
    (dict(weight=torch.zeros(5, 3)), "weight"),
    (dict(weight=torch.zeros(2, 0, 3)), "every size"),
    (dict(bias=torch.zeros(5)), "bias"),
    (dict(bias=torch.zeros(2, 4)), "bias must be"),
    (dict(bias=torch.zeros(2, 5, dtype=torch.bfloat16)), "one type"),
    (dict(groups=groups(4, 3)), "offsets"),
    (dict(groups=groups(5, 2)), "order"),
    (dict(groups=RowGroups(None, torch.zeros(3, dtype=torch.int64))), "offsets"),
    (dict(groups=RowGroups(torch.zeros(4, dtype=torch.int64), torch.zeros(3, dtype=torch.int32))), "order"),
    (dict(groups=RowGroups(None, torch.zeros(6, dtype=torch.int32)[::2])), "contiguous"),
])
def test_grouped_linear_refuses(change, text):
    args = dict(x=torch.zeros(4, 3), weight=torch.zeros(2, 5, 3), groups=groups(4, 2), bias=torch.zeros(2, 5))
    args.update(change)
    with pytest.raises(ValueError, match=text):
        grouped_linear(**args)


@pytest.mark.parametrize("change, text", [
    (dict(x=torch.zeros(())), "dimension"),
    (dict(x=torch.zeros(4, dtype=torch.int32)), "float32, bfloat16 or float16"),
    (dict(activation="relu"), "activation"),
    (dict(seed=torch.zeros(2, dtype=torch.int64)), "one int64"),
    (dict(seed=torch.zeros(1)), "one int64"),
    (dict(pair=-1), "pair"),
    (dict(pair=2 ** 64), "pair"),
    (dict(row_begin=-1), "row_begin"),
    (dict(elem_begin=2 ** 40), "elem_begin"),
])
def test_philox_dropout_refuses(change, text):
    args = dict(x=torch.zeros(4, 3), p=0.1, seed=1)
    args.update(change)
    with pytest.raises(ValueError, match=text):
        philox_dropout(**args)


def test_row_groups_counts_its_groups():
    assert groups(10, 4).n_groups == 4
