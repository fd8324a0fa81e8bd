"""Helpers of the grouped operators' tests: a comparison that nothing slips through."""
import torch

U = 2.0 ** -23  # twice the rounding of one fp32 addition: also covers a matrix instruction that truncates


def half_step(t, ref):
    """Half a step of type t at ref, or half its smallest subnormal."""
    info = torch.finfo(t)
    return ref.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def agree(got, ref, slack, what):
    """|got - ref| <= slack (fp32 arithmetic) + the rounding of ref +- slack to got's type; a NaN or an infinity in `got` is off, in
    `ref` or `slack` a mistake of the test."""
    assert got.shape == ref.shape, what
    assert ref.isfinite().all(), f"{what}: the reference is not finite"
    tol = slack + half_step(got.dtype, ref.abs() + slack)
    assert tol.isfinite().all(), f"{what}: the tolerance is not finite"
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - ref).abs() - tol).max()):.3e} beyond"


def agree_as_fp32(got, ref, slack, what):
    """As agree, where ref may lie beyond fp32: there got is the infinity of ref's sign."""
    top = torch.finfo(torch.float32).max
    assert not ((ref.abs() > top) & (ref.abs() < top * (1 + U))).any(), f"{what}: a reference on the border to infinity"
    over = ref.abs() > top
    assert torch.equal(got[over].double(), ref[over].sign() * float("inf")), f"{what}: not the infinities of fp32"
    agree(got[~over], ref[~over], slack[~over], what)
