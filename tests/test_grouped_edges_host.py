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


class Recorder:
    """A library whose calls are kept and do nothing."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return 0
        return call


def dense_copy(t):
    return torch.empty(t.shape, dtype=t.dtype).copy_(t)


def last_dimension_first(t):
    return t.clone() if t.dim() < 2 else t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize("unpack", [dense_copy, last_dimension_first])
def test_backward_reads_saved_tensors_as_they_come_back(no_device, monkeypatch, unpack):
    """Hooks on saved tensors (offloading to the host, for one) hand back other strides than were saved."""
    eng = SimpleNamespace(lib=Recorder(), ctx=SimpleNamespace(handle=None))
    monkeypatch.setattr(grouped, "_engine", lambda *a, **kw: eng)
    monkeypatch.setattr(grouped, "_stream", lambda e: 0)
    back, groups = [], RowGroups(torch.arange(4, dtype=torch.int32), torch.tensor([0, 2, 4], dtype=torch.int32))

    def unpacked(t):
        back.append(unpack(t))
        return back[-1]
    x = torch.randn(4, 9)[:, 1:4].requires_grad_()  # rows 9 apart
    w, b = torch.randn(2, 5, 3, requires_grad=True), torch.randn(2, 5, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpacked):
        y, z = grouped_linear(x, w, groups, b), philox_dropout(x, 0.1, 1, activation="elu")
    y.backward(torch.ones_like(y))
    z.backward(torch.ones_like(z))
    _, _, _, _, x_p, ld_x, *_ = eng.lib.calls["mcmc_grouped_linear_grad_weight"]
    assert ld_x == 3  # dense, whatever it was when saved
    assert unpack is not dense_copy or x_p in [t.data_ptr() for t in back]
    assert eng.lib.calls["mcmc_dropout_backward"][6] == 3
    w_p = eng.lib.calls["mcmc_grouped_linear_grad_input"][10]
    transposed = [t.data_ptr() for t in back if not t.is_contiguous()]
    assert w_p not in transposed and x_p not in transposed and eng.lib.calls["mcmc_dropout_backward"][5] not in transposed
