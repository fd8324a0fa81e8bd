"""grouped_linear and philox_dropout at the ends of their ranges, against 64-bit arithmetic.  Tolerances as in test_gpu_grouped.py: a sum of
n products kept in 32 bits is off by at most n * 2^-23 * sum|a||b|, the result by half a step of its type more."""
import pytest
import torch

from grouped_checks import U, agree, agree_as_fp32
from mcmc_amd import RowGroups, grouped_linear, philox_dropout
from test_gpu_grouped import (BF16, DEV, FP16, FP32, SIZES, dropout_reference, gen, keep_flags, linear_case, linear_reference, run_dropout,
                              run_linear)

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


@pytest.mark.parametrize("width", [1, 17])
def test_dropout_of_more_rows_than_a_launch_has_threads(width):
    """As many rows as the counter can name (17 columns: a third of them), forward and backward: around every 2^30th row and at the end
    the result is that of the rows alone."""
    R = 2 ** 32 if width == 1 else 2 ** 32 // 3
    x = torch.tensor([[1.5]], device=DEV, dtype=FP16).expand(R, width).requires_grad_()
    y = philox_dropout(x, 0.3, 55, pair=2)
    dx, = torch.autograd.grad(y, x, x.detach())
    for at in list(range(0, R, 2 ** 30)) + [R - 64]:
        first, last = max(0, at - 64), min(R, at + 64)
        alone = philox_dropout(x.detach()[first:last], 0.3, 55, pair=2, row_begin=first)
        assert torch.equal(y.detach()[first:last], alone) and torch.equal(dx[first:last], alone), at
        assert torch.equal(alone != 0, keep_flags(55, 2, last - first, width, 0.3, row_begin=first)), at


# ------------------------------------------------------------------------------------------------- one product a sum
ONE_HOT = [(300, 3, 11, 256), (400, 3, 64, 128), (400, 3, 128, 64), (600, 3, 256, 128), (1000, 3, 300, 200), (1000, 2, 200, 300), (1100, 2, 513, 1031),
           (2100, 2, 2048, 64), (2100, 2, 64, 2048), (16_700, 3, 1032, 1024), (4200, 2, 2048, 2056), (60_000, 3, 64, 48), (30_011, 5, 11, 256),
           (20_000, 2, 64, 1)]


def all_bits(dtype, shape, g):
    """Random signs, exponents 0 .. 3 and mantissas of every bit the type has, the last one set: no plane of an fp32 value is 0 for many."""
    bits = {FP32: 24, BF16: 8, FP16: 11}[dtype]
    m = torch.randint(2 ** (bits - 2), 2 ** (bits - 1), shape, generator=g, device=DEV) * 2 + 1
    e = torch.randint(0, 4, shape, generator=g, device=DEV) - (bits - 1)
    s = torch.randint(0, 2, shape, generator=g, device=DEV) * 2 - 1
    return (m.double() * s * torch.exp2(e.double())).to(dtype)


def powers(dtype, shape, g):
    return (torch.exp2(torch.randint(-2, 3, shape, generator=g, device=DEV).float()) * (torch.randint(0, 2, shape, generator=g, device=DEV) * 2 - 1)).to(dtype)


def same(got, ref, what):
    assert torch.equal(got, ref.to(got.dtype)), f"{what}: {int((got != ref.to(got.dtype)).sum())} of {ref.numel()} off"


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", ONE_HOT)
def test_one_product_a_sum(R, G, K, N, dtype):
    """Operands with all their bits, one product in every sum, at every place of the contraction: 16-bit products are exact in fp32, and so
    are fp32 ones with a power of two, whichever side it is on; of two full fp32 operands the sum is their product within 2 u."""
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 820)
    g, rows, zero = gen(821), torch.arange(R, device=DEV), torch.zeros_like(b)
    for left, right in ((all_bits, powers), (powers, all_bits), (all_bits, all_bits)):
        def close(got, ref, what):
            if dtype == FP32 and left is right:
                agree(got, ref, ref.abs() * 2 * U, what)
            else:
                same(got, ref, what)
        w = right(dtype, (G, N, K), g)
        mine = left(dtype, (R,), g)
        xs, ds = torch.zeros_like(x), torch.zeros_like(dy)
        xs[rows, rows % K], ds[rows, rows % N] = mine, mine
        close(grouped_linear(xs, w, groups, zero), mine.double()[:, None] * w.double()[ids, :, rows % K], "y")
        close(run_linear(xs, w, zero, ds, groups)["dx"], mine.double()[:, None] * w.double()[ids, rows % N], "dx")
        for trial in range(3):  # dW: column n of dy has one row
            xs, ds = left(dtype, (R, K), g), torch.zeros_like(dy)
            dw, db = torch.zeros(G, N, K, device=DEV, dtype=torch.float64), torch.zeros(G, N, device=DEV, dtype=torch.float64)
            for i in range(G):
                of = (ids == i).nonzero()[:, 0]
                n = min(N, of.numel())
                at = torch.randperm(of.numel(), generator=g, device=DEV)[:n]
                at[:2] = torch.tensor([of.numel() - 1, 0], device=DEV)[:n] if trial == 0 else at[:2]
                at, n = (at.unique(), at.unique().numel())
                r, cols, v = of[at], torch.arange(n, device=DEV), right(dtype, (n,), g)
                ds[r, cols] = v
                dw[i, :n], db[i, :n] = v.double()[:, None] * xs[r].double(), v.double()
            got = run_linear(xs, w, b, ds, groups)
            close(got["dw"], dw, "dw")
            same(got["db"], db, "db")


# ------------------------------------------------------------------------------------------ nothing else reaches a result
EVERYWHERE = SIZES + [(60_000, 3, 64, 48), (20_000, 9, 64, 1), (9000, 1, 200, 136), (3001, 3, 1000, 520), (600, 2, 2048, 2056), (8, 2, 4096, 512),
                      (5, 2, 2193, 10), (300, 9, 3, 3634), (16_700, 3, 1032, 1024), (4200, 16, 1032, 1000)]


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", EVERYWHERE)
def test_results_are_finite_and_near(R, G, K, N, dtype):
    """Every product in every kernel, where a NaN is off like any other wrong value."""
    for ordered, stray in ((False, 0.1), (True, 0.0)):
        x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, R + 2 * K, ordered, stray)
        got = run_linear(x, w, b, dy, groups)
        ref, mag = linear_reference(x, w, b, dy, ids)
        for n in ref:
            agree(got[n], ref[n], mag[n] * U, f"{n} ordered={ordered}")


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", [s for s in EVERYWHERE if s[1] >= 3 and s[0] >= 37])
def test_foreign_nan_and_infinities_stay_outside(R, G, K, N, dtype):
    """Rows of no group hold NaN and infinities, and so do the rows, the weights and the bias of group 1: the other groups' results are those
    of clean operands."""
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 31 + R, stray=0.1)
    clean = [t.clone() for t in (x, w, b, dy)]
    own, out = ids == 1, ids < 0
    clean[0][out | own], clean[3][out | own], clean[1][1], clean[2][1] = 0, 0, 0, 0
    ref, mag = linear_reference(*clean, ids)
    others = [i for i in range(G) if i != 1]
    for bad, worse in ((float("nan"), float("inf")), (-float("inf"), float("nan"))):
        x, w, b, dy = (t.clone() for t in clean)
        x[out], dy[out], x[own], dy[own], w[1], b[1] = bad, worse, worse, bad, worse, bad
        got = run_linear(x, w, b, dy, groups)
        for n in ("y", "dx"):
            assert not got[n][out].any(), n
            agree(got[n][~own], ref[n][~own], mag[n][~own] * U, n)
        for n in ("dw", "db"):
            agree(got[n][others], ref[n][others], mag[n][others] * U, n)
        assert got["y"][own].isnan().all() and (got["dw"][1].isnan().all() or not own.any())


@pytest.mark.parametrize("act", [None, "elu"])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("rows, width, p", [(1, 1, 0.1), (5, 8, 0.1), (33, 64, 0.0), (4, 1001, 0.25), (700, 24, 0.9), (1000, 17, 0.1)])
def test_dropout_is_finite_and_near(rows, width, p, dtype, act):
    x = (torch.randn(rows, width, generator=gen(rows), device=DEV) * 2).to(dtype)
    dy = torch.randn(rows, width, generator=gen(width), device=DEV).to(dtype)
    got, ref = run_dropout(x, dy, p, 77 + rows, activation=act, pair=3), dropout_reference(x, dy, keep_flags(77 + rows, 3, rows, width, p), p, act)
    for n in ("y", "dx"):
        agree(got[n], *ref[n], n)


# ---------------------------------------------------------------------------------------------------------- many groups
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", [(8192, 4096, 64, 64), (3000, 5000, 16, 24), (2500, 1000, 300, 130), (9, 65, 2048, 64), (9, 65, 64, 2048),
                                        (20_000, 130, 64, 48), (3, 70_000, 5, 6), (700, 64, 40, 33), (700, 63, 40, 33)])
def test_more_groups_than_a_wave_has_lanes(R, G, K, N, dtype):
    """63, 64 and more groups, most of them short or empty, rows of no group among them."""
    for ordered in (False, True):
        x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 900 + G, ordered, 0.1) if G <= 4096 else many_groups(R, G, K, N, dtype, ordered)
        got = run_linear(x, w, b, dy, groups)
        r = (ids >= 0) & (ids < G)
        X, W, B, D = x.double()[r], w.double()[ids[r]], b.double()[ids[r]], dy.double()[r]
        n = torch.bincount(ids[r], minlength=G).double()

        def put(shape, v, at):
            return torch.zeros(shape, device=DEV, dtype=torch.float64).index_add_(0, at, v)
        rows, own = r.nonzero()[:, 0], ids[r]
        ref = {"y": put((R, N), torch.bmm(W, X[:, :, None])[:, :, 0] + B, rows), "dx": put((R, K), torch.bmm(D[:, None], W)[:, 0], rows),
               "dw": put((G, N, K), D[:, :, None] * X[:, None], own), "db": put((G, N), D, own)}
        mag = {"y": put((R, N), (torch.bmm(W.abs(), X.abs()[:, :, None])[:, :, 0] + B.abs()) * (K + 1), rows),
               "dx": put((R, K), torch.bmm(D.abs()[:, None], W.abs())[:, 0] * N, rows),
               "dw": put((G, N, K), D.abs()[:, :, None] * X.abs()[:, None], own) * n[:, None, None], "db": put((G, N), D.abs(), own) * n[:, None]}
        for k in ref:
            agree(got[k], ref[k], mag[k] * U, f"{k} ordered={ordered}")
        assert not got["y"][~r].any() and not got["dx"][~r].any()


def many_groups(R, G, K, N, dtype, ordered):
    """More groups than group_rows sorts: the plan by hand."""
    g = gen(901)
    ids = torch.randint(-G // 10, G, (R,), generator=g, device=DEV)
    ids = torch.where(ids < 0, G, ids)
    if ordered:
        ids = torch.sort(ids).values
    order = torch.sort(ids, stable=True).indices.to(torch.int32)
    offsets = torch.searchsorted(torch.sort(ids).values, torch.arange(G + 1, device=DEV)).to(torch.int32)
    x, w, b, dy = (torch.randn(s, generator=g, device=DEV).to(dtype) for s in ((R, K), (G, N, K), (G, N), (R, N)))
    return x, w, b, dy, RowGroups(None if ordered else order, offsets), ids


def test_too_many_groups_are_refused():
    G = 1 << 27
    w, offsets = torch.zeros(1, 1, 1, device=DEV, dtype=BF16).expand(G, 1, 1), torch.zeros(G + 1, device=DEV, dtype=torch.int32)
    with pytest.raises(ValueError, match="too many"):
        grouped_linear(torch.zeros(1, 1, device=DEV, dtype=BF16), w, RowGroups(None, offsets))


# ------------------------------------------------------------------------------------------------- a bias alone
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", [(1, 1, 1, 1), (37, 5, 11, 256), (100, 3, 24, 40), (60_000, 3, 64, 48), (20_000, 9, 64, 1), (9000, 1, 200, 136),
                                        (3000, 8, 2048, 2048), (300, 600, 7, 33)])
def test_the_gradient_of_the_bias_alone(R, G, K, N, dtype):
    """Frozen weights: db needs neither x nor a dW, which would be G N K elements."""
    for ordered in (False, True):
        x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 950, ordered, 0.1)
        wide = torch.randn(R, N + 3, generator=gen(951), device=DEV).to(dtype)
        b.requires_grad_()
        y = grouped_linear(x, w, groups, b)
        x.fill_(float("nan"))  # not read any more
        for d in (dy, wide[:, 1:N + 1], dy[:1].expand(R, N)):
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            db, = torch.autograd.grad(y, b, d, retain_graph=True)
            assert torch.cuda.max_memory_allocated() - before <= 64 * G * N + (1 << 22)
            own = (ids >= 0) & (ids < G)
            member = torch.nn.functional.one_hot(ids[own], G).double().t().contiguous()
            ref, mag = member @ d.double()[own], member @ d.double().abs()[own]
            agree(db, ref, mag * torch.bincount(ids[own], minlength=G).double()[:, None] * U, "db")
        with pytest.raises(RuntimeError):  # x is saved for dW, and was changed since
            xs, ws = torch.zeros_like(x), w.detach().requires_grad_()
            y = grouped_linear(xs, ws, groups, b)
            xs.add_(1)
            y.sum().backward()


# ------------------------------------------------------------------------------------------ the bottom of the range
TINY = [(300, 3, 40, 33), (500, 3, 256, 128), (500, 3, 300, 200), (500, 2, 200, 300), (9, 2, 2048, 64), (9, 2, 64, 2048), (600, 2, 2048, 2056),
        (60_000, 3, 64, 48), (20_000, 2, 64, 1), (20_000, 2, 11, 256)]


@pytest.mark.parametrize("e", [-105, -112, -118, -126, -140])
@pytest.mark.parametrize("R, G, K, N", TINY)
def test_fp32_operands_at_the_bottom_of_the_range(R, G, K, N, e):
    """x and dy, then the weights, about 2^e against 2^100: operands below 2^-110 are off by up to 2^-134 each, on top of a sum's usual bound."""
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, FP32, 970)
    step = 2.0 ** -134
    for small, large in (((x, dy), (w,)), ((w,), (x, dy))):
        x2, w2, dy2 = (t * (2.0 ** e if any(t is s for s in small) else 2.0 ** 100) for t in (x, w, dy))
        got = run_linear(x2, w2, b * 0, dy2, groups)
        ref, mag = linear_reference(x2, w2, b * 0, dy2, ids)
        _, other = linear_reference(torch.ones_like(x2), w2, b * 0, torch.ones_like(dy2), ids)  # (K + 1) sum |w|, N sum |w|
        _, mine = linear_reference(x2, torch.ones_like(w2), b * 0, dy2, ids)                     # (K + 1) sum |x|, N sum |dy|
        agree(got["y"], ref["y"], mag["y"] * U + step * (other["y"] + mine["y"]) / (K + 1), "y")
        agree(got["dx"], ref["dx"], mag["dx"] * U + step * (other["dx"] + mine["dx"]) / N, "dx")
        if small[0] is x:
            n = torch.bincount(ids, minlength=G).double()[:, None]
            agree(got["db"], ref["db"], mag["db"] * U + n * step, "db")
    x2, dy2 = x * 2.0 ** e, dy * 2.0 ** 100
    for x2, dy2 in ((x2, dy2), (x * 2.0 ** 100, dy * 2.0 ** e)):
        got = run_linear(x2, w, b, dy2, groups)["dw"]
        ref, mag = linear_reference(x2, w, b, dy2, ids)
        _, a = linear_reference(x2, w, b, torch.ones_like(dy2), ids)
        _, c = linear_reference(torch.ones_like(x2), w, b, dy2, ids)
        n = torch.bincount(ids, minlength=G).double().clamp(min=1)[:, None, None]
        agree(got, ref["dw"], mag["dw"] * U + step * (a["dw"] + c["dw"]) / n, "dw")


@pytest.mark.parametrize("dtype, small, large", [(FP16, 2.0 ** -24, 2.0 ** 9), (BF16, 2.0 ** -133, 2.0 ** 40)])
@pytest.mark.parametrize("R, G, K, N", ONE_HOT)
def test_subnormal_operands_count(R, G, K, N, dtype, small, large):
    """16-bit operands of one to 64 times the type's smallest number against a power of two, one product a sum: exact."""
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 990)
    g, rows, zero = gen(991), torch.arange(R, device=DEV), torch.zeros_like(b)

    def tiny(shape):
        return (torch.randint(1, 65, shape, generator=g, device=DEV).double() * small).to(dtype)
    for left, right in ((tiny((R,)), torch.full((G, N, K), large, device=DEV, dtype=dtype)), (torch.full((R,), large, device=DEV, dtype=dtype), tiny((G, N, K)))):
        xs, ds = torch.zeros_like(x), torch.zeros_like(dy)
        xs[rows, rows % K], ds[rows, rows % N] = left, left
        same(grouped_linear(xs, right, groups, zero), left.double()[:, None] * right.double()[ids, :, rows % K], "y")
        same(run_linear(xs, right, zero, ds, groups)["dx"], left.double()[:, None] * right.double()[ids, rows % N], "dx")
    xs, ds = tiny((R, K)), torch.zeros_like(dy)
    dw, db = torch.zeros(G, N, K, device=DEV, dtype=torch.float64), torch.zeros(G, N, device=DEV, dtype=torch.float64)
    for i in range(G):
        of = (ids == i).nonzero()[:, 0][:N]
        cols = torch.arange(of.numel(), device=DEV)
        ds[of, cols] = large
        dw[i, cols], db[i, cols] = large * xs[of].double(), large
    got = run_linear(xs, w, b, ds, groups)
    same(got["dw"], dw, "dw")
    same(got["db"], db, "db")
    ds = torch.where(ds != 0, tiny(ds.shape), torch.zeros_like(ds))
    same(run_linear(xs, w, b, ds, groups)["db"], torch.zeros_like(db).index_add_(0, ids, ds.double()), "db")


# ------------------------------------------------------------------------------------------------- saved tensors elsewhere
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_saved_tensors_kept_on_the_host(dtype):
    """What the hooks bring back is dense, whatever the strides of the view that was saved."""
    x, w, b, dy, groups, ids = linear_case(300, 4, 63, 40, dtype, 995, ld=80)
    want, drop = run_linear(x, w, b, dy, groups), run_dropout(x, x, 0.2, 3, activation="elu")
    with torch.autograd.graph.save_on_cpu():
        got, again = run_linear(x, w, b, dy, groups), run_dropout(x, x, 0.2, 3, activation="elu")
    assert all(torch.equal(got[n], want[n]) for n in want) and all(torch.equal(again[n], drop[n]) for n in drop)
