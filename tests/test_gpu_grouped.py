"""group_rows, grouped_linear and philox_dropout against plain implementations in 64 bits.

Tolerances.  A sum of n fp32 products kept in 32 bits is off by at most n * u * sum|a||b|; u = 2^-23 (twice the rounding of one
addition) also covers a matrix instruction that truncates.  The products of 16-bit operands are exact in fp32.  Rounding the
result to its type t adds half a step: finfo(t).eps / 2 relative, or half the smallest subnormal."""
import math

import numpy as np
import pytest
import torch

from mcmc_amd import RowGroups, group_rows, grouped_linear, peak_weighted_loss, philox_dropout
from oracle import bnn_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -23


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def half_step(t, ref):
    info = torch.finfo(t)
    return ref.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def check(got, ref, slack, what):
    """|got - ref| <= slack (fp32 arithmetic) + the rounding of ref +- slack to got's type."""
    assert got.shape == ref.shape, what
    tol = slack + half_step(got.dtype, ref.abs() + slack)
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - ref).abs() - tol).max()):.3e} beyond"


# ------------------------------------------------------------------------------------------------------------ group_rows
def route(rows, n, seed, dtype=torch.int64, stray=0.1):
    ids = torch.randint(0, n, (rows,), generator=gen(seed), device=DEV)
    far = torch.tensor([-1, n, -2 ** 31, 2 ** 31 - 1] + ([2 ** 40, -2 ** 40] if dtype == torch.int64 else []), device=DEV)
    out = far[torch.randint(0, len(far), (rows,), generator=gen(seed + 1), device=DEV)]
    return torch.where(torch.rand(rows, generator=gen(seed + 2), device=DEV) < stray, out, ids).to(dtype)


def check_groups(groups, ids, n):
    key = ids.long().cpu()
    key = torch.where((key < 0) | (key >= n), n, key)
    order = torch.sort(key, stable=True).indices
    offsets = torch.cumsum(torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(key, minlength=n + 1)[:n]]), 0)
    assert groups.order.dtype == groups.offsets.dtype == torch.int32
    assert torch.equal(groups.order.cpu().long(), order)
    assert torch.equal(groups.offsets.cpu().long(), offsets)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows", [0, 1, 63, 65, 365, 8192, 8193, 100_003])
@pytest.mark.parametrize("n", [1, 5, 64, 1023, 1024, 4096])
def test_group_rows_is_a_stable_sort(rows, n, dtype):
    ids = route(rows, n, rows + n, dtype)
    check_groups(group_rows(ids, n), ids, n)


@pytest.mark.parametrize("kind", ["one group", "no group", "every other", "full size"])
def test_group_rows_shapes_of_ids(kind):
    rows = 3_650_000 if kind == "full size" else 20_001
    if kind == "one group":
        ids = torch.full((rows,), 3, device=DEV)
    elif kind == "no group":
        ids = torch.full((rows,), -1, device=DEV)
    elif kind == "every other":
        ids = route(2 * rows, 7, 3)[::2]  # strided
    else:
        ids = route(rows, 32, 4)
    check_groups(group_rows(ids, 7 if kind == "every other" else 32), ids, 7 if kind == "every other" else 32)


# --------------------------------------------------------------------------------------------------------- grouped_linear
def linear_case(R, G, K, N, dtype, seed=0, ordered=False, stray=0.0, empty=(), ld=None):
    g = gen(seed)
    ids = torch.randint(0, G, (R,), generator=g, device=DEV)
    for e in empty:
        ids[ids == e] = (e + 1) % G
    if stray:
        ids[torch.rand(R, generator=g, device=DEV) < stray] = -1
    if ordered:
        ids = torch.sort(torch.where(ids < 0, G, ids)).values
    x = torch.randn(R, ld or K, generator=g, device=DEV)[:, :K].to(dtype) if ld is None else torch.randn(R, ld, generator=g, device=DEV).to(dtype)[:, :K]
    w = (torch.randn(G, N, K, generator=g, device=DEV) / math.sqrt(K)).to(dtype)
    b = torch.randn(G, N, generator=g, device=DEV).to(dtype)
    dy = torch.randn(R, N, generator=g, device=DEV).to(dtype)
    groups = group_rows(ids, G)
    return x, w, b, dy, RowGroups(None, groups.offsets) if ordered else groups, ids


def linear_reference(x, w, b, dy, ids):
    """y, dx, dw, db in 64 bits, and the sums of |products| that bound each one's fp32 arithmetic, with their lengths."""
    X, W, B, D = x.double(), w.double(), b.double(), dy.double()
    G, N, K = w.shape
    R = x.shape[0]
    out = {n: torch.zeros(s, dtype=torch.float64, device=x.device) for n, s in (("y", (R, N)), ("dx", (R, K)), ("dw", (G, N, K)), ("db", (G, N)))}
    mag = {n: torch.zeros_like(v) for n, v in out.items()}
    for g in range(G):
        r = (ids == g).nonzero()[:, 0]
        n = r.numel()
        if n == 0:
            continue
        out["y"][r], mag["y"][r] = X[r] @ W[g].t() + B[g], (X[r].abs() @ W[g].abs().t() + B[g].abs()) * (K + 1)
        out["dx"][r], mag["dx"][r] = D[r] @ W[g], (D[r].abs() @ W[g].abs()) * N
        out["dw"][g], mag["dw"][g] = D[r].t() @ X[r], (D[r].abs().t() @ X[r].abs()) * n
        out["db"][g], mag["db"][g] = D[r].sum(0), D[r].abs().sum(0) * n
    return out, mag


def run_linear(x, w, b, dy, groups):
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    y = grouped_linear(x, w, groups, b)
    return dict(zip(("y", "dx", "dw", "db"), (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))))


SIZES = [  # rows, groups, in, out
    (1, 1, 1, 1), (1, 5, 7, 3), (3, 2, 1, 64), (5, 3, 64, 1), (37, 5, 11, 256), (365, 5, 256, 128), (130, 4, 65, 63), (64, 1, 64, 64), (63, 2, 33, 31),
    (200, 70, 40, 24), (257, 3, 129, 130), (1000, 8, 72, 200), (8, 16, 1024, 520), (700, 2, 513, 96), (40, 3, 2000, 17), (2049, 3, 128, 264),
]


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", SIZES)
def test_grouped_linear_and_its_gradients(R, G, K, N, dtype):
    for ordered, stray, empty in ((False, 0.0, ()), (True, 0.0, ()), (False, 0.2, (0, G - 1) if G > 2 else ()), (True, 0.3, (1,) if G > 2 else ())):
        x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, R + K, ordered, stray, empty)
        got = run_linear(x, w, b, dy, groups)
        ref, mag = linear_reference(x, w, b, dy, ids)
        for n in ref:
            check(got[n], ref[n], mag[n] * U, f"{n} ordered={ordered} stray={stray}")
        none = (ids < 0) | (ids >= G)
        assert not got["y"][none].any() and not got["dx"][none].any()
        for e in range(G):
            if not (ids == e).any():
                assert not got["dw"][e].any() and not got["db"][e].any()


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", [(60_000, 3, 64, 48), (30_011, 5, 11, 256), (20_000, 9, 64, 1), (9000, 1, 200, 136)])
def test_weight_gradients_summed_in_chunks(R, G, K, N, dtype):
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 5, stray=0.05, empty=(2,) if G > 2 else ())
    if R == 60_000:  # nearly everything in one group: chunks of very unequal groups
        ids = torch.where(torch.rand(R, generator=gen(9), device=DEV) < 0.98, 1, ids)
        groups = group_rows(ids, G)
    got = run_linear(x, w, b, dy, groups)
    ref, mag = linear_reference(x, w, b, dy, ids)
    for n in ref:
        check(got[n], ref[n], mag[n] * U, n)
    again = run_linear(x, w, b, dy, groups)
    assert all(torch.equal(got[n], again[n]) for n in got), "the same bits every time"


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("R, G, K, N", [(4096, 4, 1024, 768), (3001, 3, 1000, 520), (600, 2, 2048, 2056), (2500, 3, 520, 1032)])
def test_grouped_linear_wide(R, G, K, N, dtype):
    for ordered in (False, True):
        x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 11, ordered, 0.03)
        got = run_linear(x, w, b, dy, groups)
        ref, mag = linear_reference(x, w, b, dy, ids)
        for n in ref:
            check(got[n], ref[n], mag[n] * U, f"{n} ordered={ordered}")


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_grouped_linear_without_rows(dtype):
    x, w, b = torch.zeros(0, 7, device=DEV, dtype=dtype), torch.ones(3, 5, 7, device=DEV, dtype=dtype), torch.ones(3, 5, device=DEV, dtype=dtype)
    got = run_linear(x, w, b, torch.zeros(0, 5, device=DEV, dtype=dtype), group_rows(torch.zeros(0, dtype=torch.int64, device=DEV), 3))
    assert got["y"].shape == (0, 5) and got["dx"].shape == (0, 7)
    assert not got["dw"].any() and not got["db"].any()


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("K, N, ld", [(64, 64, 80), (64, 64, 65), (63, 40, 64), (256, 128, 264)])
def test_grouped_linear_strides(K, N, ld, dtype):
    """Views: rows further apart, starting at an odd element, expanded rows, transposed inputs and an expanded gradient."""
    R, G = 300, 4
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 21, ld=ld)
    wide = torch.randn(R, ld + 1, generator=gen(3), device=DEV).to(dtype)
    for xv in (x, wide[:, 1:K + 1], x[:1].expand(R, K), x.t().contiguous().t()):
        got = run_linear(xv, w, b, dy, groups)
        ref, mag = linear_reference(xv, w, b, dy, ids)
        for n in ref:
            check(got[n], ref[n], mag[n] * U, f"{n} strides {xv.stride()}")
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    got = run_linear(x, wt, b, dy[:1].expand(R, N), groups)
    ref, mag = linear_reference(x, wt, b, dy[:1].expand(R, N), ids)
    for n in ref:
        check(got[n], ref[n], mag[n] * U, n)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("K, N", [(64, 48), (40, 33), (256, 128)])
def test_what_a_group_does_not_own_does_not_reach_it(K, N, dtype):
    """NaN and infinities in rows of no group, in another group's rows and weights stay where they are."""
    R, G = 500, 3
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 31, stray=0.2)
    x, w, b, dy = (t.clone() for t in (x, w, b, dy))
    x[ids < 0], dy[ids < 0] = float("nan"), float("inf")
    x[ids == 1], w[1], b[1] = float("inf"), float("nan"), float("nan")
    got = run_linear(x, w, b, dy, groups)
    clean = [t.clone() for t in (x, w, b, dy)]
    clean[0][(ids < 0) | (ids == 1)] = 0
    clean[1][1] = clean[2][1] = 0
    clean[3][ids < 0] = 0
    ref, mag = linear_reference(*clean, ids)
    other = ids != 1
    assert not got["y"][ids < 0].any() and not got["dx"][ids < 0].any()
    check(got["y"][other], ref["y"][other], mag["y"][other] * U, "y")
    check(got["dx"][other], ref["dx"][other], mag["dx"][other] * U, "dx")
    for n in ("dw", "db"):
        check(got[n][[0, 2]], ref[n][[0, 2]], mag[n][[0, 2]] * U, n)
    assert got["y"][ids == 1].isnan().all()
    # a single bad value reaches its own row of y and its own column of dW
    x2, w2, b2, dy2, groups2, ids2 = linear_case(R, G, K, N, dtype, 32)
    r, c = 7, K - 1
    x2 = x2.clone()
    x2[r, c] = float("nan")
    got = run_linear(x2, w2, b2, dy2, groups2)
    assert got["y"][r].isnan().all() and not got["y"][torch.arange(R, device=DEV) != r].isnan().any()
    assert got["dw"][ids2[r], :, c].isnan().all() and int(got["dw"].isnan().sum()) == N and not got["dx"].isnan().any()


@pytest.mark.parametrize("which", ["x", "w", "b"])
def test_only_the_gradients_asked_for(which):
    x, w, b, dy, groups, ids = linear_case(100, 3, 24, 40, FP32, 41)
    leaves = {"x": x, "w": w, "b": b}
    leaves[which].requires_grad_()
    y = grouped_linear(x, w, groups, b)
    got, = torch.autograd.grad(y, leaves[which], dy)
    ref, mag = linear_reference(x.detach(), w.detach(), b.detach(), dy, ids)
    n = {"x": "dx", "w": "dw", "b": "db"}[which]
    check(got, ref[n], mag[n] * U, n)
    no_bias = grouped_linear(x.detach(), w.detach(), groups)
    zero, m = linear_reference(x.detach(), w.detach(), torch.zeros_like(b), dy, ids)
    check(no_bias, zero["y"], m["y"] * U, "no bias")


def test_grouped_linear_gradients_against_differences():
    """The product is linear in each argument: <f(a + d) - f(a - d), dy> / 2 = <grad, d> up to the rounding of the four sums."""
    x, w, b, dy, groups, ids = linear_case(150, 4, 33, 21, FP32, 51)
    got = run_linear(x, w, b, dy, groups)
    for i, n in enumerate(("dx", "dw", "db")):
        a = [x, w, b]
        d = torch.randn(a[i].shape, generator=gen(60 + i), device=DEV)
        plus, minus = list(a), list(a)
        plus[i], minus[i] = a[i] + d, a[i] - d
        fp, fm = (grouped_linear(t[0], t[1], groups, t[2]).double() for t in (plus, minus))
        diff, along = float(((fp - fm) * dy).sum() / 2), float((got[n].double() * d).sum())
        # each y is off by at most 34 u times its sum of |products| (here below 12), the inputs a +- d by u/2 of themselves
        tol = 2 * 36 * U * float((fp.abs() + fm.abs() + 12).mul(dy.abs()).sum()) + 150 * U * float((got[n].double().abs() * d.abs()).sum())
        assert abs(diff - along) <= tol, (n, diff, along, tol)


# --------------------------------------------------------------------------------------------------------- philox_dropout
def keep_flags(seed, pair, rows, width, p, row_begin=0, elem_begin=0):
    """Element by element from the oracle's Philox."""
    row = (np.arange(rows, dtype=np.int64) + row_begin).astype(np.uint32)[:, None]
    elem = (np.arange(width, dtype=np.int64) + elem_begin).astype(np.uint32)[None, :]
    row, elem = np.broadcast_arrays(row, elem)
    blk = ((elem >> np.uint32(4)) << np.uint32(1)) | ((elem >> np.uint32(2)) & np.uint32(1))
    slot = ((elem >> np.uint32(3)) & np.uint32(1)) * np.uint32(4) + (elem & np.uint32(3))
    ctr = np.stack([blk, np.full_like(elem, pair), np.full_like(elem, 0x4D41534B), row], axis=-1)
    key = np.stack([np.full_like(elem, seed & 0xFFFFFFFF), np.full_like(elem, seed >> 32)], axis=-1)
    x = orc.philox4x32_10(ctr, key)
    word = np.take_along_axis(x, (slot >> np.uint32(1)).astype(np.int64)[..., None], axis=-1)[..., 0]
    half = (word >> (np.uint32(16) * (slot & np.uint32(1)))) & np.uint32(0xFFFF)
    thr = int(np.float32(np.float32(1.0) - np.float32(p)) * np.float32(65536.0))
    return torch.from_numpy(half < thr).to(DEV)


def dropout_reference(x, dy, keep, p, act):
    s, X, D = 1.0 / (1.0 - p), x.double(), dy.double()
    if act == "elu":
        h, d = torch.where(X > 0, X, torch.expm1(X.clamp(max=0))), torch.exp(X.clamp(max=0))
        # exp(x) in fp32: the rounded argument x log2(e) moves it by |x| u, the instruction and two roundings by less than 4 u;
        # elu: exp(x) - 1 below -1/16, above it a degree-4 polynomial (truncation 1.3e-7 relative and four roundings)
        eh = torch.where(X > 0, 0 * X, torch.where(X > -0.0625, 6 * U * X.abs(), d * (X.abs() + 4) * U + U))
        ed = d * (X.abs() + 4) * U + 1e-37
    else:
        h, d, eh, ed = X, torch.ones_like(X), 0 * X, 0 * X
    zero = torch.zeros_like(X)
    return {"y": (torch.where(keep, h * s, zero), torch.where(keep, (eh + 2 * U * h.abs()) * s, zero)),
            "dx": (torch.where(keep, D * d * s, zero), torch.where(keep, D.abs() * (ed + 4 * U * d) * s, zero))}


def run_dropout(x, dy, *args, **kw):
    x = x.detach().requires_grad_()
    y = philox_dropout(x, *args, **kw)
    return {"y": y.detach(), "dx": torch.autograd.grad(y, x, dy)[0]}


def check_dropout(got, ref):
    for n in ("y", "dx"):
        check(got[n], *ref[n], n)


@pytest.mark.parametrize("act", [None, "elu"])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("rows, width, p", [(1, 1, 0.1), (3, 7, 0.5), (5, 8, 0.1), (2, 9, 0.3), (32, 256, 0.1), (33, 64, 0.0), (4, 1001, 0.25),
                                            (700, 24, 0.9), (1000, 17, 0.1), (1, 5000, 0.1)])
def test_philox_dropout(rows, width, p, dtype, act):
    x = (torch.randn(rows, width, generator=gen(rows), device=DEV) * 2).to(dtype)
    dy = torch.randn(rows, width, generator=gen(width), device=DEV).to(dtype)
    seed, pair = 0x1234_5678_9ABC_DEF0 + rows, 41
    keep = keep_flags(seed, pair, rows, width, p)
    got = run_dropout(x, dy, p, seed, activation=act, pair=pair)
    check_dropout(got, dropout_reference(x, dy, keep, p, act))
    assert not got["y"][~keep].any() and not got["dx"][~keep].any()


def test_mask_of_a_piece_is_the_whole_batch_s():
    x = torch.randn(100, 448, generator=gen(1), device=DEV)
    whole = philox_dropout(x, 0.1, 99, pair=7)
    assert torch.equal(philox_dropout(x[40:73], 0.1, 99, pair=7, row_begin=40), whole[40:73])
    for e0, e1 in ((0, 256), (256, 384), (384, 448)):  # the three hidden layers of one pair
        assert torch.equal(philox_dropout(x[:, e0:e1], 0.1, 99, pair=7, elem_begin=e0), whole[:, e0:e1])
    masks = orc.philox_keep_masks(99, 7, 100, 0.1)
    assert torch.equal((whole != 0).cpu(), torch.from_numpy(np.concatenate(masks, 1).astype(bool)))
    last = 2 ** 32 - 100  # the last rows the counter can name
    assert torch.equal(philox_dropout(x, 0.1, 99, row_begin=last) != 0, keep_flags(99, 0, 100, 448, 0.1, row_begin=last))
    assert torch.equal(philox_dropout(x[:, :32], 0.1, 99, elem_begin=2 ** 32 - 32) != 0, keep_flags(99, 0, 100, 32, 0.1, elem_begin=2 ** 32 - 32))


def test_share_of_kept_elements():
    """4.2 million draws at p = 0.1: the mean of independent flags lies within 5 standard deviations of floor(0.9 * 65536) / 65536."""
    y = philox_dropout(torch.ones(4096, 1024, device=DEV), 0.1, 3)
    q = 58982 / 65536
    assert abs(float((y != 0).double().mean()) - q) < 5 * math.sqrt(q * (1 - q) / y.numel())


@pytest.mark.parametrize("act", [None, "elu"])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_dropped_nan_and_infinity_are_zero(dtype, act):
    rows, width, p = 64, 40, 0.5
    keep = keep_flags(5, 0, rows, width, p)
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.full((rows, width), bad, device=DEV, dtype=dtype)
        got = run_dropout(x, torch.ones_like(x), p, 5, activation=act)
        assert not got["y"][~keep].any() and not got["dx"][~keep].any()
        want = torch.tensor(-1.0 if act == "elu" and bad < 0 else bad, device=DEV, dtype=dtype) / (1 - p)
        assert torch.equal(got["y"][keep].nan_to_num(1e4), want.expand(int(keep.sum())).nan_to_num(1e4))


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_philox_dropout_shapes_and_strides(dtype):
    base = torch.randn(6, 5, 50, generator=gen(2), device=DEV).to(dtype)
    flat = philox_dropout(base.reshape(30, 50), 0.2, 8, activation="elu")
    assert torch.equal(philox_dropout(base, 0.2, 8, activation="elu"), flat.view(6, 5, 50))
    assert torch.equal(philox_dropout(base[0, 0], 0.2, 8, activation="elu"), flat[0])
    rows = base.reshape(30, 50)
    for view in (rows[:, 3:20], rows[:, 1:2], rows[::2], rows.t(), rows[:1].expand(9, 50)):
        want = philox_dropout(view.contiguous(), 0.2, 8, activation="elu")
        assert torch.equal(philox_dropout(view, 0.2, 8, activation="elu"), want)
        x = view.detach().requires_grad_()
        g, = torch.autograd.grad(philox_dropout(x, 0.2, 8, activation="elu").sum(), x)  # an expanded gradient
        assert torch.equal(g, run_dropout(view.contiguous(), torch.ones(view.shape, device=DEV, dtype=dtype), 0.2, 8, activation="elu")["dx"])
    for shape in ((0, 5), (5, 0), (0,)):
        e = torch.zeros(shape, device=DEV, dtype=dtype, requires_grad=True)
        y = philox_dropout(e, 0.2, 8)
        assert y.shape == shape and torch.autograd.grad(y.sum(), e)[0].shape == shape


def test_seed_tensor_is_the_integer_seed():
    x = torch.randn(20, 100, generator=gen(3), device=DEV)
    for seed in (0, 77, 2 ** 63 + 5):
        t = torch.tensor([seed - 2 ** 64 if seed >= 2 ** 63 else seed], device=DEV)
        a, b = (run_dropout(x, torch.ones_like(x), 0.3, s, activation="elu") for s in (seed, t))
        assert torch.equal(a["y"], b["y"]) and torch.equal(a["dx"], b["dx"])
    x.requires_grad_()
    y = philox_dropout(x, 0.3, t, activation="elu")
    t.add_(1)  # the backward pass would draw another mask: refused by autograd's version check
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_elu_dropout_gradient_against_differences():
    """Central differences of the kept elements at distance 2^-6: the third derivative of exp bounds the truncation by
    h^2 / 6 * exp(x + h) * s; both values carry the fp32 error of the forward pass divided by h."""
    x = torch.randn(50, 64, generator=gen(4), device=DEV)
    x = torch.where(x.abs() < 0.05, x.sign() * 0.05 + (x == 0) * 0.05, x)  # away from the kink
    h, s = 2.0 ** -6, 1 / 0.9
    f = [philox_dropout(x + d, 0.1, 6, activation="elu").double() for d in (h, -h)]
    diff = (f[0] - f[1]) / (2 * h)
    got = run_dropout(x, torch.ones_like(x), 0.1, 6, activation="elu")["dx"]
    tol = s * (h * h / 6 * torch.exp(x.double().clamp(max=0) + h) + (x.double().abs() + 8) * 2 * U / h)
    assert ((diff - got.double()).abs() <= tol).all()


# ----------------------------------------------------------------------------------------------------------------- together
def network(G, F, dtype, seed):
    g, sizes = gen(seed), ((256, F), (128, 256), (64, 128), (1, 64))
    return [((torch.randn(G, n, k, generator=g, device=DEV) * math.sqrt(2 / k)).to(dtype), (torch.randn(G, n, generator=g, device=DEV) * 0.1).to(dtype))
            for n, k in sizes]


def members(x, ids, layers, p, seed):
    groups, h = group_rows(ids, layers[0][0].shape[0]), x
    for (w, b), e in zip(layers[:3], (0, 256, 384)):
        h = philox_dropout(grouped_linear(h, w, groups, b), p, seed, activation="elu", elem_begin=e)
    return grouped_linear(h, *layers[3][:1], groups, layers[3][1])[:, 0]


def members_reference(x, ids, layers, keeps, p):
    h = x
    for i, (w, b) in enumerate(layers):
        h = (w[ids] @ h[:, :, None])[:, :, 0] + b[ids]
        if i < 3:
            h = torch.where(h > 0, h, torch.expm1(h.clamp(max=0)))
            h = h * keeps[i] / (1 - p)
    return h[:, 0]


@pytest.mark.parametrize("dtype, tol", [(FP32, 2e-5), (BF16, 4e-2), (FP16, 6e-3)])
def test_routed_members_train_as_one_network(dtype, tol):
    """Rows routed to five members, three layers of linear -> ELU -> dropout, the output layer, the loss, every gradient; against
    autograd in 64 bits.  Bound on the norm of each gradient's error: four layers forward and four back round 8 activations by
    at most half a step each, and the loss's weights double that; 16 half steps of bf16 are 16 * 2^-8 = 6e-2, of fp16 8e-3
    (their signs differ: two thirds of that is asked); fp32: 256-term sums, 8 * 256 * u / 10."""
    R, G, F, p, seed = 333, 5, 11, 0.1, 17
    g = gen(70)
    ids = torch.randint(0, G, (R,), generator=g, device=DEV)
    x, target = torch.randn(R, F, generator=g, device=DEV).to(dtype), torch.randn(R, generator=g, device=DEV)
    layers = network(G, F, dtype, 71)
    flat = [t.detach().requires_grad_() for pair in layers for t in pair]
    xl = x.detach().requires_grad_()
    y = members(xl, ids, list(zip(flat[::2], flat[1::2])), p, seed)
    loss = peak_weighted_loss(y.float(), target)
    got = torch.autograd.grad(loss, [xl] + flat)
    keeps = [torch.from_numpy(k.astype(np.float64)).to(DEV) for k in orc.philox_keep_masks(seed, 0, R, p)]
    ref_flat = [t.detach().double().requires_grad_() for t in flat]
    xr = x.double().requires_grad_()
    yr = members_reference(xr, ids, list(zip(ref_flat[::2], ref_flat[1::2])), keeps, p)
    t64, d = target.double(), None
    d = yr - t64
    peak = (t64 > t64.mean() + 0.5 * t64.std()).double()
    w = 1 + peak * (1 + torch.sigmoid(d.abs() - d.abs().mean()))
    lossr = (d * d * w).mean()
    want = torch.autograd.grad(lossr, [xr] + ref_flat)
    assert abs(float(loss) - float(lossr)) <= tol * float(lossr)
    assert float((y.detach().double() - yr.detach()).norm()) <= tol * float(yr.detach().norm())
    for a, b in zip(got, want):
        assert float((a.double() - b).norm()) <= tol * float(b.norm())


def test_layer_by_layer_is_the_fused_forward():
    """One member and one sample through mcmc_forward_dropout's fused fp32 kernel and through the operators: the same masks, outputs
    within 1e-5 of the largest (the bar of the fused kernels' own parity tests)."""
    from mcmc_amd.engine import Engine
    from mcmc_amd import _lib
    F, rows, seed, p = 11, 257, 1234, 0.1
    layers = network(1, F, FP32, 80)
    X = torch.randn(rows, F, generator=gen(81), device=DEV)
    mu = torch.cat([t.reshape(-1) for pair in layers for t in pair])[None].contiguous()
    eng = Engine(torch.device(DEV))
    wpack = torch.empty(eng.wpack_bytes(F, _lib.DT_F32), dtype=torch.uint8, device=DEV)
    eng.sample_weights(mu, torch.zeros_like(mu), 1, F, 0, 1, _lib.NOISE_NONE, None, 0, _lib.DT_F32, wpack)
    ldY = (rows + 63) // 64 * 64
    Y = torch.zeros(1, ldY, device=DEV)
    eng.forward(_lib.DT_F32, eng.pack_x(X, _lib.DT_F32), rows, F, wpack, 1, Y, ldY, philox_dropout=(seed, p, 1, 1, 0))
    got = members(X, torch.zeros(rows, dtype=torch.int64, device=DEV), layers, p, seed)
    assert float((got - Y[0, :rows]).abs().max()) <= 1e-5 * float(Y.abs().max())


@pytest.mark.parametrize("rows", [200, 12_000])
def test_captured_training_step_replays(rows):
    """Route, forward and backward captured once; replays with new inputs, ids and seed equal the eager step, with eager work and
    synchronisation in between."""
    G, F, p = 4, 11, 0.1
    layers = network(G, F, BF16, 90)
    static = {"x": torch.zeros(rows, F, device=DEV, dtype=BF16), "ids": torch.zeros(rows, dtype=torch.int64, device=DEV),
              "seed": torch.zeros(1, dtype=torch.int64, device=DEV), "dy": torch.zeros(rows, device=DEV, dtype=BF16)}

    def step(s):
        flat = [t.detach().requires_grad_() for pair in layers for t in pair]  # leaves of their own: no eager graph shares them
        y = members(s["x"], s["ids"], list(zip(flat[::2], flat[1::2])), p, s["seed"])
        return [y.detach()] + list(torch.autograd.grad(y, flat, s["dy"]))

    def fill(i):
        g = gen(100 + i)
        static["x"].copy_(torch.randn(rows, F, generator=g, device=DEV))
        static["ids"].copy_(torch.randint(-1, G, (rows,), generator=g, device=DEV))
        static["seed"].fill_(1000 + i)
        static["dy"].copy_(torch.randn(rows, generator=g, device=DEV))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(1, 5):
        fill(i)
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in out]
        want = step(static)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(seen, want)), i


def test_two_streams_do_not_share_anything():
    """The same calls on two streams at once, different inputs: each result equals the one made alone."""
    cases = [linear_case(20_000, 5, 64, 64, BF16, 200 + i) for i in range(2)]
    ids = [route(50_000, 9, 300 + i) for i in range(2)]
    alone = [(run_linear(*c[:5]), group_rows(i, 9)) for c, i in zip(cases, ids)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append((run_linear(*cases[k][:5]), group_rows(ids[k], 9)))
    torch.cuda.synchronize()
    for k in range(2):
        for lin, grp in got[k]:
            assert all(torch.equal(lin[n], alone[k][0][n]) for n in lin)
            assert torch.equal(grp.order, alone[k][1].order) and torch.equal(grp.offsets, alone[k][1].offsets)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_offsets_beyond_32_bits(dtype):
    """Elements past 2^31 (and, in bf16, bytes past 2^32): the last rows of a wide, long batch."""
    R, K, N = (2 ** 31 + 2 ** 20) // 4096 + 3, 4096, 8
    x = torch.zeros(R, K, device=DEV, dtype=dtype)
    g = gen(400)
    x[-5:] = torch.randn(5, K, generator=g, device=DEV).to(dtype)
    w = torch.randn(2, N, K, generator=g, device=DEV).to(dtype) / 64
    ids = torch.ones(R, dtype=torch.int64, device=DEV)
    ids[-2:] = 0
    y = grouped_linear(x, w, group_rows(ids, 2))
    ref = torch.einsum("rk,rnk->rn", x[-5:].double(), w.double()[ids[-5:]])
    mag = torch.einsum("rk,rnk->rn", x[-5:].double().abs(), w.double().abs()[ids[-5:]]) * K
    check(y[-5:], ref, mag * U, "y")
    assert not y[:-5].any()
    d = philox_dropout(x, 0.5, 9, pair=1)
    keep = keep_flags(9, 1, 5, K, 0.5, row_begin=R - 5)
    assert torch.equal(d[-5:], torch.where(keep, x[-5:] * 2, torch.zeros_like(x[-5:])))
    assert not d[:-5].any()


@pytest.mark.parametrize("K, N", [(40, 33), (256, 128)])
def test_fp32_infinities_and_the_whole_range(K, N):
    """fp32 products follow fp32's rules for infinities (inf * 1 = inf, inf - inf and inf * 0 = NaN), in the rows and columns they reach
    and nowhere else, and keep their accuracy at the ends of the exponent range."""
    R, G = 300, 3
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, FP32, 500)
    x, w, dy = x.clone(), w.clone(), dy.clone()
    x[5, 3], x[9, 0] = float("inf"), -float("inf")
    w[1, 2, 1] = float("inf")
    dy[20, 4] = -float("inf")
    got = run_linear(x, w, b, dy, groups)
    ref, mag = linear_reference(x, w, b, dy, ids)
    for n in ref:
        fine = ref[n].isfinite()
        assert not fine.all()
        assert torch.equal(got[n].isnan(), ref[n].isnan()) and torch.equal(got[n].isinf(), ref[n].isinf()), n
        assert torch.equal(got[n][ref[n].isinf()].sign().double(), ref[n][ref[n].isinf()].sign()), n
        check(got[n][fine], ref[n][fine], mag[n][fine] * U, n)
    for sx, sw in ((2.0 ** 120, 2.0 ** -100), (2.0 ** -90, 2.0 ** 60), (3.4e38 / 6, 2.0 ** -20)):
        x2, w2 = torch.randn(R, K, generator=gen(1), device=DEV).clamp(-6, 6) * sx, w * 0 + sw * 0.5
        w2[:, :, ::3] *= -0.37
        got = run_linear(x2, w2, b * 0, dy.clamp(-3, 3), groups)
        ref, mag = linear_reference(x2, w2, b * 0, dy.clamp(-3, 3), ids)
        for n in ("y", "dx"):
            check(got[n], ref[n], mag[n] * U, n)


def test_gradients_of_gradients_are_refused():
    x, w, b, dy, groups, ids = linear_case(20, 2, 8, 8, FP32, 600)
    for f in (lambda t: grouped_linear(t, w, groups, b), lambda t: philox_dropout(t, 0.1, 5, activation="elu")):
        t = x.detach().requires_grad_()
        first, = torch.autograd.grad(f(t).square().sum(), t, create_graph=True)
        plain, = torch.autograd.grad(f(t).square().sum(), t)
        assert torch.equal(first.detach(), plain)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            first.sum().backward()


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", [(8, 2, 4096, 512), (15, 64, 11, 2772), (5, 2, 2193, 10), (300, 9, 3, 3634), (1, 1, 4096, 4096), (130, 1, 1000, 1111)])
def test_long_contractions_on_few_tiles(R, G, K, N, dtype):
    """Contractions split over workgroups, whose partial sums are joined afterwards; rows of no group are zero in every part."""
    for ordered, stray in ((False, 0.2 if R > 4 else 0.0), (True, 0.0)):
        x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 700, ordered, stray)
        got = run_linear(x, w, b, dy, groups)
        ref, mag = linear_reference(x, w, b, dy, ids)
        for n in ref:
            check(got[n], ref[n], mag[n] * U, n)
        assert not got["y"][ids < 0].any() and not got["dx"][ids < 0].any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", [(16_700, 3, 1032, 1024), (20_003, 5, 264, 2056), (4200, 16, 1032, 1000), (3000, 1, 4096, 4096)])
def test_enough_tiles_for_every_cu(R, G, K, N, dtype):
    """What fills the chip with 256 x 256 outputs a workgroup: y and dx of the first, y of the second, dW of the others (the last one's single group on all XCDs)."""
    for ordered in (False, True):
        x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 23, ordered, 0.03, (1,) if G > 2 else ())
        got = run_linear(x, w, b, dy, groups)
        ref, mag = linear_reference(x, w, b, dy, ids)
        for n in ref:
            check(got[n], ref[n], mag[n] * U, f"{n} ordered={ordered}")
        again = run_linear(x, w, b, dy, groups)
        assert all(torch.equal(got[n], again[n]) for n in got), "the same bits every time"


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", [(600_001, 3, 64, 16), (300_000, 4, 11, 256), (400_003, 2, 255, 31)])
def test_many_rows_past_weights_in_lds(R, G, K, N, dtype):
    """Runs of several turns of a workgroup's waves, the last one of each group short."""
    x, w, b, dy, groups, ids = linear_case(R, G, K, N, dtype, 29, False, 0.02)
    got = run_linear(x, w, b, dy, groups)
    ref, mag = linear_reference(x, w, b, dy, ids)
    for n in ref:
        check(got[n], ref[n], mag[n] * U, n)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("R, G, K, N", [(1, 1, 1, 1), (365, 5, 11, 256), (100_000, 3, 64, 1), (200_001, 7, 11, 40), (150_000, 2, 128, 64), (70_000, 5, 300, 130),
                                        (16_700, 3, 1032, 1024), (4200, 16, 1032, 1000), (3000, 1, 4096, 4096), (9, 2, 4096, 512), (5000, 100, 65, 33)])
def test_small_integers_are_exact(R, G, K, N, dtype):
    """Operands of -1, 0 and 1: every sum is an integer below 2^24, exact in 32 bits in any order, so that a row too many or too few shows
    whatever the length; the result is its one rounding to the type."""
    g = gen(31)
    ids = torch.randint(0, G, (R,), generator=g, device=DEV)
    ids[torch.rand(R, generator=g, device=DEV) < 0.5] = G // 2  # one group has half of the rows
    ids[torch.rand(R, generator=g, device=DEV) < 0.05] = -1
    x, w, b, dy = (torch.randint(-1, 2, s, generator=g, device=DEV).to(dtype) for s in ((R, K), (G, N, K), (G, N), (R, N)))
    got = run_linear(x, w, b, dy, group_rows(ids, G))
    ref, _ = linear_reference(x, w, b, dy, ids)
    for n in ref:
        assert torch.equal(got[n], ref[n].to(dtype)), n
