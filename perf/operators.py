"""What the operators of ``mcmc_amd.grouped`` are measured on: rows routed to members (``group_rows``), one linear layer per
member over ragged groups of rows (``grouped_linear``) and the counter-based dropout behind a layer's activation
(``philox_dropout``), each beside its plain form in elementary torch operations.

``own`` selects the side: False computes the plain form in 32 bits, True calls the framework."""
from __future__ import annotations

import math

import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_TAG = 0x4D41534B  # 'MASK', third counter word of the mask stream
_LOW = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    route = {"op": "route", "ids": "int64"}
    lin = {"op": "linear", "bias": True, "skew": 0.0, "unrouted": 0.0, "ordered": False}
    drop = {"op": "dropout", "act": "elu", "p": 0.1, "pair": 3}
    return [
        # one year of days handed to the five members of the default ensemble: latency
        {"name": "route-365x5", **route, "rows": 365, "groups": 5, "skew": 0.5, "unrouted": 0.0},
        # every day of 10,000 series, one member per cluster of stores, some days held out
        {"name": "route-3.65Mx32", **route, "rows": 3_650_000, "groups": 32, "skew": 1.0, "unrouted": 0.02},
        # first layer (11 features -> 256) of five members over one year, predict
        {"name": "first-fp32-365", **lin, "train": False, "dtype": "fp32", "rows": 365, "groups": 5, "k": 11, "n": 256},
        # one new row for each of a few members of a wide network: single-token serving, bound by the weights
        {"name": "wide-bf16-8rows", **lin, "train": False, "dtype": "bf16", "rows": 8, "groups": 16, "k": 4096, "n": 4096},
        # second layer (256 -> 128) over every day of 10,000 series, predict
        {"name": "second-bf16-3.65M", **lin, "train": False, "dtype": "bf16", "rows": 3_650_000, "groups": 8, "k": 256, "n": 128, "skew": 0.5},
        # the same layer's training step at the batch the large-batch kernels are measured at (8 members x 65,536 rows)
        {"name": "second-fp32-train", **lin, "train": True, "dtype": "fp32", "rows": 524_288, "groups": 8, "k": 256, "n": 128, "skew": 0.5},
        # output layer (64 -> 1), training
        {"name": "output-bf16-train", **lin, "train": True, "dtype": "bf16", "rows": 1_048_576, "groups": 8, "k": 64, "n": 1, "skew": 0.5},
        # many small experts with unequal and empty groups, odd row count, training
        {"name": "experts-fp16-train", **lin, "train": True, "dtype": "fp16", "rows": 8_191, "groups": 64, "k": 2048, "n": 1408, "skew": 1.0,
         "unrouted": 0.01},
        # few wide experts over a large batch that is already in order, training: bound by the matrix pipe
        {"name": "wide-bf16-train", **lin, "train": True, "dtype": "bf16", "rows": 32_768, "groups": 8, "k": 4096, "n": 4096, "skew": 0.25,
         "ordered": True},
        # activation and dropout of one mini-batch of 32 rows: latency
        {"name": "drop-fp32-32x256", **drop, "train": False, "dtype": "fp32", "rows": 32, "width": 256},
        # the same behind the widest layer of a large batch, training
        {"name": "drop-bf16-1Mx256", **drop, "train": True, "dtype": "bf16", "rows": 1_048_576, "width": 256},
        # plain dropout over odd rows (a width with no common factor with any tile), training
        {"name": "drop-fp16-odd", **drop, "train": True, "dtype": "fp16", "rows": 36_501, "width": 1001, "act": "none", "p": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "linear", "linear", "linear", "dropout"])
    unrouted = rng.choice([0.0, 0.0, rng.uniform(0.0, 0.2)])
    if op == "route":
        return {"op": op, "ids": rng.choice(["int64", "int32"]), "rows": _log(rng, 1, 3_650_000), "groups": _log(rng, 1, 1024),
                "skew": rng.uniform(0.0, 2.0), "unrouted": unrouted}
    train = rng.random() < 0.6
    if op == "dropout":
        width = _log(rng, 1, 8192)
        return {"op": op, "train": train, "dtype": rng.choice(list(_DT)), "rows": _log(rng, 1, max(1, min(2_000_000, (1 << 27) // width))),
                "width": width, "act": rng.choice(["elu", "none"]), "p": rng.choice([0.1, rng.uniform(0.01, 0.9)]), "pair": rng.randrange(1000)}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    k, n = _log(rng, 1, 4096), _log(rng, 1, 4096)
    groups = _log(rng, 1, max(1.0, min(64.0, 1.8e8 / (k * n))))
    products, values = (2.0e11, 1.2e8) if dtype == "fp32" else (5.0e11, 2.4e8)  # of one direction; on the wider side of the layer
    rows = _log(rng, 1, max(1.0, min(3_650_000.0, products / (k * n), values / max(k, n))))
    return {"op": op, "train": train, "dtype": dtype, "rows": rows, "groups": groups, "k": k, "n": n, "bias": rng.random() < 0.7,
            "skew": rng.uniform(0.0, 1.0), "unrouted": unrouted, "ordered": rng.random() < 0.4}


def work(case):
    r = case["rows"]
    if case["op"] == "route":
        return {"bytes": r * ((8 if case["ids"] == "int64" else 4) + 4) + 4 * (case["groups"] + 1), "flops": 0}
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "dropout":
        passes = 2 + ((3 if case["act"] == "elu" else 2) if case["train"] else 0)
        return {"bytes": passes * r * case["width"] * e, "flops": 0}
    k, n, g = case["k"], case["n"], min(case["groups"], r)  # a group without rows is neither read nor (without a gradient) written
    x, y, w = r * k * e, r * n * e, g * k * n * e
    index = 4 * r * (not case["ordered"])
    wb = case["groups"] * k * n * e
    return {"bytes": (x + y + w + index) + ((2 * x + y + w + wb + index) if case["train"] else 0), "flops": (6 if case["train"] else 2) * r * k * n}


# --------------------------------------------------------------------------------------------------------------- inputs
def _ids(case, gen, dev):
    """Each row's group; the groups' shares are exp(skew * normal) (equal at skew 0), a share `unrouted` of the rows is in none."""
    share = torch.exp(case["skew"] * torch.randn(case["groups"], generator=gen, device=dev))
    edges = torch.cumsum(share / share.sum(), 0)
    ids = torch.searchsorted(edges, torch.rand(case["rows"], generator=gen, device=dev)).clamp_(max=case["groups"] - 1)
    if case["unrouted"]:
        ids[torch.rand(case["rows"], generator=gen, device=dev) < case["unrouted"]] = -1
    return ids


def _elu_like(shape, gen, dev):
    """What a hidden layer hands on: ELU of a unit normal, a tenth of it dropped."""
    h = torch.nn.functional.elu(torch.randn(shape, generator=gen, device=dev))
    return h.mul_(torch.rand(shape, generator=gen, device=dev) >= 0.1).mul_(1 / 0.9)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    if case["op"] == "route":
        s["ids"] = _ids(case, gen, dev).to(torch.int64 if case["ids"] == "int64" else torch.int32)
        return s
    dt = _DT[case["dtype"]]
    if case["op"] == "dropout":
        shape = (case["rows"], case["width"])
        s["x"] = torch.randn(shape, generator=gen, device=dev).to(dt).requires_grad_(case["train"])
        s["seed"] = (seed * 0x9E3779B97F4A7C15 + 12345) & 0xFFFFFFFFFFFFFFFF
        if case["train"]:
            s["dy"] = (torch.randn(shape, generator=gen, device=dev) * 0.05).to(dt)
        return s
    R, G, K, N = case["rows"], case["groups"], case["k"], case["n"]
    ids = _ids(case, gen, dev)
    key = torch.where(ids < 0, torch.full_like(ids, G), ids)
    counts = torch.bincount(key, minlength=G + 1)[:G]
    s["offsets"] = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)]).to(torch.int32)
    s["order"] = None if case["ordered"] else torch.sort(key, stable=True).indices.to(torch.int32)
    s["most"] = int(counts.max())  # rows of the largest group: the host of a program that routes knows its group sizes
    s["x"] = _elu_like((R, K), gen, dev).to(dt).requires_grad_(case["train"])
    s["weight"] = (torch.randn((G, N, K), generator=gen, device=dev) * math.sqrt(2.0 / K)).to(dt).requires_grad_(case["train"])
    s["bias"] = (torch.randn((G, N), generator=gen, device=dev) * 0.1).to(dt).requires_grad_(case["train"]) if case["bias"] else None
    if case["train"]:
        s["dy"] = (torch.randn((R, N), generator=gen, device=dev) * 0.05).to(dt)
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_route(s):
    ids, G = s["ids"].to(torch.int64), s["groups"]
    key = torch.where((ids < 0) | (ids >= G), torch.full_like(ids, G), ids)
    counts = torch.bincount(key, minlength=G + 1)[:G]
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)])
    return {"order": torch.sort(key, stable=True).indices.to(torch.int32), "offsets": offsets.to(torch.int32)}


def _plain_linear(s):
    """Every group padded to the largest, then one batched product in fp32."""
    x, w, dt = s["x"].detach().float(), s["weight"].detach().float(), s["x"].dtype
    R, G, most = x.shape[0], w.shape[0], max(1, s["most"])
    off = s["offsets"].to(torch.int64)
    order = torch.arange(R, device=x.device) if s["order"] is None else s["order"].to(torch.int64)
    at = off[:-1, None] + torch.arange(most, device=x.device)
    live = (at < off[1:, None])[..., None]
    slot = order[at.clamp(max=R - 1)]  # [G, most]: the row in each place of the padded batch
    place = torch.arange(R, device=x.device)
    g = torch.searchsorted(off, place, right=True) - 1
    routed = (g < G)[:, None]
    g = g.clamp(max=G - 1)
    j = (place - off[g]).clamp(max=most - 1)

    def pad(t):
        return torch.where(live, t[slot], torch.zeros((), device=t.device))

    def unpad(t):
        out = torch.empty(R, t.shape[2], device=t.device)
        out[order] = torch.where(routed, t[g, j], torch.zeros((), device=t.device))
        return out

    xp = pad(x)
    yp = torch.bmm(xp, w.transpose(1, 2))
    if s["bias"] is not None:
        yp = yp + s["bias"].detach().float()[:, None, :]
    out = {"y": unpad(yp).to(dt)}
    if s["train"]:
        dyp = pad(s["dy"].float())
        out["dx"] = unpad(torch.bmm(dyp, w)).to(dt)
        out["dweight"] = torch.bmm(dyp.transpose(1, 2), xp).to(dt)
        if s["bias"] is not None:
            out["dbias"] = dyp.sum(1).to(dt)
    return out


def _plain_keep(s):
    """The keep flags [rows, width] of the 'MASK' stream: Philox4x32-10 in 64-bit integers, 16 bits per element."""
    R, W, dev = s["rows"], s["width"], s["x"].device
    blocks = 2 * ((W + 15) // 16)
    row = torch.arange(R, device=dev)[:, None].expand(R, blocks)
    c = [torch.arange(blocks, device=dev)[None, :].expand(R, blocks), torch.full((), s["pair"], device=dev), torch.full((), _TAG, device=dev), row]
    k0, k1 = s["seed"] & _LOW, s["seed"] >> 32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & _LOW) ^ c[1] ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c[3] ^ k1, a & _LOW]
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack(c, -1)  # [R, blocks, 4]; halves: low then high of each word
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).view(R, blocks // 2, 2, 2, 4)  # 16-column tile, block, eight, four
    flags = halves < int((torch.tensor(1.0) - torch.tensor(s["p"])).item() * 65536.0)
    return flags.transpose(2, 3).reshape(R, blocks * 8)[:, :W]  # column = 16 tile + 8 eight + 4 block + four


def _plain_dropout(s):
    x, dt = s["x"].detach().float(), s["x"].dtype
    keep, scale, zero = _plain_keep(s), 1.0 / (1.0 - s["p"]), torch.zeros((), device=x.device)
    neg = torch.expm1(x)
    h = torch.where(x > 0, x, neg) if s["act"] == "elu" else x
    out = {"y": torch.where(keep, h * scale, zero).to(dt)}
    if s["train"]:
        d = torch.where(x > 0, torch.ones((), device=x.device), neg + 1.0) if s["act"] == "elu" else 1.0
        out["dx"] = torch.where(keep, s["dy"].float() * d * scale, zero).to(dt)
    return out


# ------------------------------------------------------------------------------------------------- the framework's calls
def _own_route(s):
    from mcmc_amd import group_rows
    groups = group_rows(s["ids"], s["groups"])
    return {"order": groups.order, "offsets": groups.offsets}


def _own_linear(s):
    from mcmc_amd import RowGroups, grouped_linear
    y = grouped_linear(s["x"], s["weight"], RowGroups(s["order"], s["offsets"]), s["bias"])
    out = {"y": y}
    if s["train"]:
        leaves = [s["x"], s["weight"]] + ([s["bias"]] if s["bias"] is not None else [])
        out.update(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, leaves, s["dy"])))
    return out


def _own_dropout(s):
    from mcmc_amd import philox_dropout
    y = philox_dropout(s["x"], s["p"], s["seed"], activation=None if s["act"] == "none" else s["act"], pair=s["pair"])
    out = {"y": y}
    if s["train"]:
        out["dx"], = torch.autograd.grad(y, s["x"], s["dy"])
    return out


def run(state):
    if own:
        out = {"route": _own_route, "linear": _own_linear, "dropout": _own_dropout}[state["op"]](state)
        return {k: v.detach() for k, v in out.items()}
    return {"route": _plain_route, "linear": _plain_linear, "dropout": _plain_dropout}[state["op"]](state)


# ------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] == "route":
        return None  # whole numbers: compared as they are
    s = prepare(case, seed)
    x = s["x"].detach().double()
    if case["op"] == "dropout":
        keep, scale = _exact_keep(s), 1.0 / (1.0 - case["p"])
        elu = case["act"] == "elu"
        h = torch.where(x > 0, x, torch.expm1(x.clamp(max=0.0))) if elu else x
        out = {"y": keep * h * scale}
        if case["train"]:
            out["dx"] = keep * s["dy"].double() * (torch.exp(x.clamp(max=0.0)) if elu else 1.0) * scale
        return out
    w, off = s["weight"].detach().double(), s["offsets"].tolist()
    b = None if s["bias"] is None else s["bias"].detach().double()
    order = torch.arange(case["rows"], device=x.device) if s["order"] is None else s["order"].long()
    y = x.new_zeros(case["rows"], case["n"])
    dy = s["dy"].double() if case["train"] else None
    dx, dw, db = (torch.zeros_like(x), torch.zeros_like(w), y.new_zeros(case["groups"], case["n"])) if case["train"] else (None, None, None)
    for g in range(case["groups"]):
        rows = order[off[g]:off[g + 1]]
        if rows.numel():
            xg = x[rows]
            y[rows] = xg @ w[g].t() if b is None else torch.addmm(b[g], xg, w[g].t())
            if case["train"]:
                dyg = dy[rows]
                dx[rows], dw[g], db[g] = dyg @ w[g], dyg.t() @ xg, dyg.sum(0)
    out = {"y": y}
    if case["train"]:
        out.update({"dx": dx, "dweight": dw}, **({} if b is None else {"dbias": db}))
    return out


def _exact_keep(s):
    """The mask stream once more, element by element: which block and which 16 bits belong to a column, the 64-bit product from
    two 16-bit halves."""
    dev, W = s["x"].device, s["width"]
    col = torch.arange(W, device=dev)
    block, slot = ((col >> 4) << 1) | ((col >> 2) & 1), 4 * ((col >> 3) & 1) + (col & 3)
    threshold = int((torch.tensor(1.0) - torch.tensor(s["p"])).item() * 65536.0)
    keep = torch.empty(s["rows"], W, dtype=torch.bool, device=dev)

    def product(m, v):
        low, high = m * (v & 0xFFFF), m * (v >> 16)
        low, high = (low + ((high & 0xFFFF) << 16)), (high >> 16)
        return (high + (low >> 32)) & _LOW, low & _LOW

    step = max(1, (1 << 24) // W)
    for r0 in range(0, s["rows"], step):
        row = torch.arange(r0, min(s["rows"], r0 + step), device=dev)[:, None]
        v0, v1 = (block + 0 * row), torch.full_like(row, s["pair"])
        v2, v3 = torch.full_like(row, _TAG), row
        for i in range(10):
            h0, l0 = product(0xD2511F53, v0)
            h1, l1 = product(0xCD9E8D57, v2)
            v0, v1, v2, v3 = h1 ^ v1 ^ ((s["seed"] + i * 0x9E3779B9) & _LOW), l1, h0 ^ v3 ^ (((s["seed"] >> 32) + i * 0xBB67AE85) & _LOW), l0
        word = torch.where(slot < 2, v0, torch.where(slot < 4, v1, torch.where(slot < 6, v2, v3)))
        keep[r0:r0 + step] = ((word >> (16 * (slot & 1))) & 0xFFFF) < threshold
    return keep
