"""grouped_linear and philox_dropout at the ends of their ranges, against 64-bit arithmetic.  Tolerances as in test_gpu_grouped.py: a sum of
n products kept in 32 bits is off by at most n * 2^-23 * sum|a||b|, the result by half a step of its type more."""
import pytest
import torch

from grouped_checks import U, agree, agree_as_fp32
from mcmc_amd import grouped_linear
from test_gpu_grouped import BF16, DEV, FP32, dropout_reference, keep_flags, linear_case, run_dropout, run_linear

pytestmark = pytest.mark.gpu

# which kernels: weights in LDS; the tiles (forward with K > 256, dx with N > 256, dW whole and in chunks); a contraction in parts; a handful of columns
SHAPES = [(300, 3, 40, 33), (500, 3, 256, 128), (500, 3, 300, 200), (500, 2, 200, 300), (9, 2, 2048, 64), (9, 2, 64, 2048), (600, 2, 2048, 2056),
          (60_000, 3, 64, 48), (20_000, 2, 64, 1), (20_000, 2, 11, 256)]

# operands that fp32 holds and whose products it holds, or not
BIG = {
    # products that overflow and whose terms in bf16 planes have either sign; one just below the largest number whose first term is above it
    "products": [(1 + 2.0 ** -7 - 2.0 ** -9) * 2.0 ** 100, -(1 + 2.0 ** -7 - 2.0 ** -9) * 2.0 ** 100, 2.0 ** 40, (2 - 2.0 ** -12) * 2.0 ** 63,
                 -(2 - 2.0 ** -9) * 2.0 ** 62, 0.5, 0.0, 1.0],
    # the same beside operands that round to a bf16 infinity
    "operands": [(1 + 2.0 ** -7 - 2.0 ** -9) * 2.0 ** 100, 2.0 ** 40, (2 - 2.0 ** -12) * 2.0 ** 63, 3.4e38, -3.4e38, 0.5, 0.0, 1.0, -torch.finfo(FP32).max],
}


def spread_over(values, shape):
    """values in turn along the last dimension of a zero-filled or broadcast shape."""
    v = torch.tensor(values, device=DEV, dtype=FP32)
    return v[torch.arange(shape[-1], device=DEV) % len(values)].expand(shape).contiguous()


@pytest.mark.parametrize("ordered", [False, True])
@pytest.mark.parametrize("R, G, K, N", SHAPES)
@pytest.mark.parametrize("big", BIG.values(), ids=BIG)
def test_fp32_products_at_the_top_of_the_range(big, R, G, K, N, ordered):
    """One product a sum, so that the sum is fp32's product: its value, or the infinity of its sign.  2 u: what the split leaves out and
    the addition of its six terms, of which one is not small."""
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, FP32, 800, ordered)
    zero = torch.zeros_like(b)
    rows = torch.arange(R, device=DEV)
    mine = torch.tensor(big, device=DEV, dtype=FP32)[rows % len(big)]
    # y: row r holds one value, every weight of output n is one value
    xs = torch.zeros_like(x)
    xs[rows, rows % K] = mine
    ws = spread_over(big, (G, K, N)).transpose(1, 2).contiguous()
    ref = mine.double()[:, None] * ws[0, :, 0].double()[None, :]
    agree_as_fp32(grouped_linear(xs, ws, groups, zero), ref, ref.abs() * 2 * U, "y")
    # dx: likewise
    ds = torch.zeros_like(dy)
    ds[rows, rows % N] = mine
    ws = spread_over(big, (G, N, K))
    ref = mine.double()[:, None] * ws[0, 0].double()[None, :]
    agree_as_fp32(run_linear(xs, ws, zero, ds, groups)["dx"], ref, ref.abs() * 2 * U, "dx")
    # dW: one row of each group holds anything
    xs, ds = torch.zeros_like(x), torch.zeros_like(dy)
    refw, refb = torch.zeros(G, N, K, device=DEV, dtype=torch.float64), torch.zeros(G, N, device=DEV, dtype=torch.float64)
    for g in range(G):
        of = (ids == g).nonzero()[:, 0]
        if of.numel():
            r = of[of.numel() // 2]
            xs[r], ds[r] = spread_over(big, (K,)), spread_over(big[::-1], (N,))
            refw[g], refb[g] = ds[r].double()[:, None] * xs[r].double()[None, :], ds[r].double()
    got = run_linear(xs, w, b, ds, groups)
    agree_as_fp32(got["dw"], refw, refw.abs() * 2 * U, "dw")
    agree_as_fp32(got["db"], refb, refb.abs() * U, "db")


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_dropout_gradient_where_only_a_factor_overflows(dtype, p):
    """dy / (1 - p) is beyond fp32, dy * elu'(x) / (1 - p) is not: x from -3 down to where exp(x) is 0."""
    x = -torch.linspace(3, 200, 64 * 24, device=DEV).view(64, 24).to(dtype)
    dy = torch.full_like(x, 3.3e38)
    dy[:, ::2] *= -1
    got = run_dropout(x, dy, p, 21, activation="elu")
    ref = dropout_reference(x, dy, keep_flags(21, 0, 64, 24, p), p, "elu")
    assert got["dx"].isfinite().all()
    agree(got["dx"], *ref["dx"], "dx")
