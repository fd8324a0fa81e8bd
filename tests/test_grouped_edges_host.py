"""CPU-only tests of the grouped operators: calls that are refused, with the launches stubbed where a refusal comes after them."""
from contextlib import nullcontext
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from grouped_checks import agree, agree_as_fp32
from mcmc_amd import RowGroups, _lib, grouped, grouped_linear, philox_dropout


@pytest.fixture
def no_device(monkeypatch):
    """The operators' Python on CPU tensors: no device is looked for, nothing is launched, results are zeros."""
    monkeypatch.setattr(grouped, "_engine", lambda *a, **kw: SimpleNamespace())
    monkeypatch.setattr(grouped, "_on", lambda eng: nullcontext())
    monkeypatch.setattr(grouped, "_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(grouped, "_forward", lambda eng, x, w, b, order, offsets: x.new_zeros(x.shape[0], w.shape[1]))
    monkeypatch.setattr(grouped, "_dropout", lambda eng, x, args: (torch.zeros_like(x), x))


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", ["x", "weight", "bias", "dropout"])
def test_forward_mode_derivatives_are_refused(no_device, which, grad_mode):
    """A tangent does not show in requires_grad; without a look for it the derivative would be zero without a word."""
    args = {"x": torch.ones(4, 3), "weight": torch.ones(2, 5, 3), "bias": torch.ones(2, 5)}
    groups = RowGroups(None, torch.tensor([0, 2, 4], dtype=torch.int32))
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        assert grouped_linear(args["x"], args["weight"], groups, args["bias"]).shape == (4, 5)  # no tangent: an ordinary call
        with pytest.raises(NotImplementedError, match="jvp"):
            if which == "dropout":
                philox_dropout(forward_ad.make_dual(args["x"], torch.ones(4, 3)), 0.1, 1)
            else:
                args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
                grouped_linear(args["x"], args["weight"], groups, args["bias"])


@pytest.mark.parametrize("which", ["linear", "dropout"])
def test_tangents_of_the_output_gradient_are_refused(no_device, which):
    x, groups = torch.ones(4, 3, requires_grad=True), RowGroups(None, torch.tensor([0, 2, 4], dtype=torch.int32))
    y = philox_dropout(x, 0.1, 1) if which == "dropout" else grouped_linear(x, torch.ones(2, 5, 3), groups)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="jvp"):
            torch.autograd.grad(y, x, dual)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1.1])
def test_the_comparison_sees_every_wrong_value(bad):
    one, slack = torch.ones(3, dtype=torch.float64), torch.full((3,), 1e-3, dtype=torch.float64)
    agree(torch.ones(3), one, slack, "ones")
    got = torch.tensor([1.0, bad, 1.0])
    for check in (agree, agree_as_fp32):
        with pytest.raises(AssertionError, match="1 of 3 off"):
            check(got, one, slack, "one of them")
    for ref, tol in ((one / 0, slack), (one, slack / 0)):
        with pytest.raises(AssertionError, match="not finite"):
            agree(torch.ones(3), ref, tol, "a mistake of the test")
    with pytest.raises(AssertionError, match="infinities"):
        agree_as_fp32(torch.full((3,), 3e38), one * 1e39, slack, "beyond fp32")


@pytest.mark.parametrize("product", [0, 1])
@pytest.mark.parametrize("dtype", [_lib.DT_F32, _lib.DT_BF16, _lib.DT_F16])
def test_walks_of_many_groups_end(product, dtype):
    """Every workgroup of a forward or dx product walks all offsets: groups times workgroups is bounded, whatever the widths."""
    size = _lib.load().mcmc_grouped_linear_workspace_bytes
    for n_in, n_out in ((1, 1), (64, 64), (300, 200), (4096, 64), (64, 4096), (2048, 2048)):
        for rows, groups in ((1 << 20, 1 << 20), (1 << 30, 1 << 20), (1, 1 << 27), (1 << 10, 1 << 30), (1 << 30, 1 << 30)):
            assert size(product, dtype, rows, groups, n_in, n_out) == -1 and "too many" in _lib.last_error(), (rows, groups, n_in, n_out)
            assert size(2, dtype, rows, groups, n_in, n_out) >= 0  # the weight gradient does not walk
        for rows, groups in ((1 << 24, 63), (1 << 24, 64), (1 << 22, 512), (1 << 17, 4096), (8192, 4096), (1 << 10, 1 << 16), (0, 1 << 30)):
            assert size(product, dtype, rows, groups, n_in, n_out) >= 0, (rows, groups, n_in, n_out)
