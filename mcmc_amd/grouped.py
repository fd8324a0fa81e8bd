"""Layers whose rows belong to groups: one member (or expert) per group, each with its own share of the rows.

The reference hands every member the whole batch (bayesian_ensemble.py:160-169).  Here the rows are routed first and a layer's
product runs over the ragged groups in one launch:

    groups = group_rows(ids, n_members)                       # ids[r] = the member of row r
    h = x
    for i, (w, b) in enumerate(hidden):                       # w [members, out, in], b [members, out]
        h = philox_dropout(grouped_linear(h, w, groups, b), 0.1, seed, activation="elu", elem_begin=elem[i])
    y = grouped_linear(h, w_out, groups, b_out)

All arithmetic is in libmcmc_hip.so (``mcmc_group_rows``, ``mcmc_grouped_linear_*``, ``mcmc_dropout_*``); gradients are ordinary
autograd, of the first order and in reverse mode (other derivatives are refused).  There is no CPU path.  Every call runs on the
current stream of its tensors' device and allocates what it needs from torch, nothing is kept from one call for the next, so calls
may be captured into HIP graphs (after a first call outside the capture, which loads the kernels; a backward pass, as torch has
it, only while no eager graph of the same leaves is alive).
"""
from __future__ import annotations

import math
from contextlib import nullcontext
from typing import NamedTuple, Optional, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .engine import Engine

_DT = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
_ACT = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "elu": _lib.ACT_ELU}
_U64 = 0xFFFFFFFFFFFFFFFF
_MAX_GROUPS = 4096       # MCMC_GROUP_ROWS_MAX_GROUPS
_MAX_DIM = 1 << 30       # MCMC_GROUPED_MAX_ROWS, MCMC_GROUPED_MAX_DIM
_ENGINES = {}


# The calls on small batches last as long as their Python: pointers and the stream go to the library as plain integers (ctypes
# converts those fastest), sizes are taken once, and what needs no gradient does not pass through autograd.
def _engine(t: torch.Tensor, what: str, **others: Optional[torch.Tensor]) -> Engine:
    """The engine of t's device; every other tensor has to live there too."""
    dev = t.get_device()
    for name, o in ((what, t), *others.items()):
        if o is not None and o.get_device() != dev or dev < 0:
            if not o.is_cuda:
                raise RuntimeError(f"{name} must live on a HIP device (got {o.device}); mcmc_amd has no CPU path")
            raise ValueError(f"{name} lives on {o.device}, {what} on {t.device}")
    eng = _ENGINES.get(dev)
    if eng is None:
        eng = _ENGINES[dev] = Engine(torch.device("cuda", dev))
    return eng


_HERE = nullcontext()


def _on(eng: Engine):
    return _HERE if torch._C._cuda_getDevice() == eng.device.index else torch.cuda.device(eng.device)


def _stream(eng: Engine) -> int:
    return torch._C._cuda_getCurrentRawStream(eng.device.index)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _dtype(t: torch.Tensor, what: str) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}") from None


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor whose rows are contiguous; the distance between rows is free (views and expanded rows are read in place)."""
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _flat(t: torch.Tensor) -> torch.Tensor:
    """[..., width] as [rows, width] (empty tensors included)."""
    return t if t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


def _has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """A forward-mode tangent does not show in requires_grad, and holds whatever the grad mode.  (Outside a dual level, number -1, there are
    none; the callers look at the level themselves, a call less.)"""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _once(backward):
    """Gradients of gradients are refused like once_differentiable does it, but its bookkeeping (20 us a call) is paid only by a
    backward pass that records a graph; so are tangents of dy."""
    recorded = once_differentiable(backward)

    def run(ctx, dy):
        if forward_ad._current_level >= 0 and _has_tangent(dy):
            raise NotImplementedError("the gradients of mcmc_amd's grouped operators have no forward-mode derivative (jvp)")
        return recorded(ctx, dy) if torch.is_grad_enabled() else backward(ctx, dy)
    return run


def _wants_grad(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether the call has to pass through autograd: for a gradient, or to be refused there (no operator has a jvp)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return forward_ad._current_level >= 0 and _has_tangent(*tensors)


class RowGroups(NamedTuple):
    """Which rows belong to which group.  Group g owns the rows ``order[offsets[g]:offsets[g + 1]]``; what ``order`` lists from
    ``offsets[-1]`` on belongs to no group.

    order: int32 [rows], every row once, or None where the rows lie group after group already.
    offsets: int32 [n_groups + 1], from 0, not decreasing, at most rows."""
    order: Optional[torch.Tensor]
    offsets: torch.Tensor

    @property
    def n_groups(self) -> int:
        return self.offsets.shape[0] - 1


def group_rows(ids: torch.Tensor, n_groups: int) -> RowGroups:
    """Sort the rows stably by group: ``ids`` [rows] (int32 or int64) names each row's group; an id outside 0..n_groups-1 puts the
    row into no group (``grouped_linear`` gives it zeros).  At most 4,096 groups."""
    if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be a 1-D int32 or int64 tensor, got {ids.dtype} {tuple(ids.shape)}")
    n_groups, rows = int(n_groups), ids.shape[0]
    if not 1 <= n_groups <= _MAX_GROUPS:
        raise ValueError(f"n_groups must be in [1, {_MAX_GROUPS}], got {n_groups}")
    eng = _engine(ids, "ids")
    with _on(eng):
        ids = ids.contiguous()
        ws_bytes = _lib.check(eng.lib.mcmc_group_rows_workspace_bytes(rows, n_groups), "mcmc_group_rows_workspace_bytes")
        order = torch.empty(rows, dtype=torch.int32, device=ids.device)
        offsets = torch.empty(n_groups + 1, dtype=torch.int32, device=ids.device)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=ids.device) if ws_bytes else None
        _lib.check(eng.lib.mcmc_group_rows(eng.ctx.handle, ids.data_ptr(), ids.element_size(), rows, n_groups, order.data_ptr(), offsets.data_ptr(),
                                           _ptr(ws), _stream(eng)), "mcmc_group_rows")
    return RowGroups(order, offsets)


# ---- grouped_linear ---------------------------------------------------------------------------------------------------------
def _workspace_bytes(eng: Engine, product: int, dt: int, R: int, G: int, K: int, N: int) -> int:
    return _lib.check(eng.lib.mcmc_grouped_linear_workspace_bytes(product, dt, R, G, K, N), "mcmc_grouped_linear_workspace_bytes")


def _workspace(n: int, dev) -> Optional[torch.Tensor]:
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _forward(eng: Engine, x, weight, bias, order, offsets):
    (R, K), (G, N, _), dev = x.shape, weight.shape, x.device
    dt, y = _DT[x.dtype], torch.empty((R, N), dtype=x.dtype, device=dev)
    ws = _workspace(_workspace_bytes(eng, _lib.GROUPED_FORWARD, dt, R, G, K, N), dev)
    _lib.check(eng.lib.mcmc_grouped_linear_forward(eng.ctx.handle, dt, x.data_ptr(), x.stride(0), R, _ptr(order), offsets.data_ptr(), G, K, N,
                                                   weight.data_ptr(), _ptr(bias), y.data_ptr(), _ptr(ws), _stream(eng)), "mcmc_grouped_linear_forward")
    return y


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, eng, x, weight, bias, order, offsets):
        with _on(eng):
            x, weight = _rows(x), weight.contiguous()
            y = _forward(eng, x, weight, None if bias is None else bias.contiguous(), order, offsets)
        need_x, need_w, need_b = ctx.needs_input_grad[1:4]
        (R, K), (G, N, _), dt = x.shape, weight.shape, _DT[x.dtype]
        K_w = K if need_w else 1  # inputs of the weight gradient: db alone comes with one column of it, see backward
        ctx.eng, ctx.sizes, ctx.needs = eng, (dt, R, G, K, K_w, N), (need_x, need_w, need_b)
        ctx.ws = (_workspace_bytes(eng, _lib.GROUPED_GRAD_INPUT, dt, R, G, K, N) if need_x else 0,
                  _workspace_bytes(eng, _lib.GROUPED_GRAD_WEIGHT, dt, R, G, K_w, N) if need_w or need_b else 0)
        # what each gradient reads: dx the weights, dW the inputs
        ctx.save_for_backward(x if need_w else None, weight if need_x else None, order, offsets)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        eng, (dt, R, G, K, K_w, N), (ws_x, ws_w) = ctx.eng, ctx.sizes, ctx.ws
        x, weight, order, offsets = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs
        dx = dw = db = None
        with _on(eng):
            lib, handle, stream, dtype, dev = eng.lib, eng.ctx.handle, _stream(eng), dy.dtype, dy.device
            ld_dy = N
            if not dy.is_contiguous():
                dy = _rows(dy)
                ld_dy = dy.stride(0)
            # what was saved may come back with other strides (hooks on saved tensors)
            order, offsets = None if order is None else order.contiguous(), offsets.contiguous()
            dy_p, order_p, offsets_p = dy.data_ptr(), _ptr(order), offsets.data_ptr()
            if need_x:
                weight = weight.contiguous()
                dx = torch.empty((R, K), dtype=dtype, device=dev)
                ws = _workspace(ws_x, dev)
                _lib.check(lib.mcmc_grouped_linear_grad_input(handle, dt, dy_p, ld_dy, R, order_p, offsets_p, G, K, N, weight.data_ptr(), dx.data_ptr(),
                                                              _ptr(ws), stream), "mcmc_grouped_linear_grad_input")
            if need_w or need_b:
                # db alone: dy stands for an x of one column, so that dy is read once and next to nothing else is done
                ld_x = K
                if not need_w:
                    x, ld_x = dy, ld_dy
                elif not x.is_contiguous():
                    x = _rows(x)
                    ld_x = x.stride(0)
                dw = torch.empty((G, N, K_w), dtype=dtype, device=dev)
                db = torch.empty((G, N), dtype=dtype, device=dev) if need_b else None
                ws = _workspace(ws_w, dev)
                _lib.check(lib.mcmc_grouped_linear_grad_weight(handle, dt, dy_p, ld_dy, x.data_ptr(), ld_x, R, order_p, offsets_p, G, K_w, N, dw.data_ptr(),
                                                               _ptr(db), _ptr(ws), stream), "mcmc_grouped_linear_grad_weight")
        return None, dx, dw if need_w else None, db, None, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, groups: RowGroups, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One linear layer per group: ``y[r] = weight[g] @ x[r] + bias[g]`` with g the group of row r; rows of no group are 0.

    x [rows, in]; weight [n_groups, out, in]; bias [n_groups, out]; all of one type (float32, bfloat16 or float16; sums are
    kept in 32 bits and rounded once; float32 values below 2^-110 = 8e-34 count with an absolute error of up to 2^-134, not with
    float32's relative one).  Differentiable in x, weight and bias; a group without rows gets zero gradients.

    Made for up to a few hundred groups: every workgroup walks the offsets, so that the time grows with groups times rows beyond
    (8,192 rows, 64 -> 64: up to 512 groups the same, 4,096 groups ten times as long), and a call that would walk for seconds is
    refused (2^20 groups of one row each)."""
    order, offsets = groups
    xs, ws = x.shape, weight.shape
    if len(xs) != 2 or len(ws) != 3 or (bias is not None and bias.dim() != 2):
        raise ValueError(f"x must be [rows, in], weight [groups, out, in], bias [groups, out]; got {tuple(xs)}, {tuple(ws)}"
                         + ("" if bias is None else f", {tuple(bias.shape)}"))
    _dtype(x, "x")
    (R, K), (G, N, weight_in) = xs, ws
    if min(G, N, weight_in) < 1 or max(G, N, weight_in, R) > _MAX_DIM:
        raise ValueError(f"every size of weight must be in [1, 2^30] and rows at most 2^30, got {tuple(ws)} and {R} rows")
    if K != weight_in:
        raise ValueError(f"Expected {weight_in} input features, got {K}")
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise ValueError(f"x, weight and bias must have one type, got {x.dtype}, {weight.dtype}" + ("" if bias is None else f", {bias.dtype}"))
    if bias is not None and bias.shape != (G, N):
        raise ValueError(f"bias must be {(G, N)}, got {tuple(bias.shape)}")
    if offsets.dtype != torch.int32 or offsets.shape != (G + 1,) or not offsets.is_contiguous():
        raise ValueError(f"groups.offsets must be a contiguous int32 [{G + 1}] tensor (n_groups + 1), got {offsets.dtype} {tuple(offsets.shape)}")
    if order is not None and (order.dtype != torch.int32 or order.shape != (R,) or not order.is_contiguous()):
        raise ValueError(f"groups.order must be None or a contiguous int32 [{R}] tensor (rows), got {order.dtype} {tuple(order.shape)}")
    eng = _engine(x, "x", weight=weight, bias=bias, order=order, offsets=offsets)
    if _wants_grad(x, weight, bias):
        return _GroupedLinear.apply(eng, x, weight, bias, order, offsets)
    with _on(eng):
        return _forward(eng, _rows(x), weight.contiguous(), None if bias is None else bias.contiguous(), order, offsets)


# ---- philox_dropout ---------------------------------------------------------------------------------------------------------
def _dropout(eng: Engine, x, args):
    """y [rows, width] and the 2-D x it was made from."""
    p, seed, seed_dev, act, pair, row_begin, elem_begin = args
    x = _rows(_flat(x))
    R, W = x.shape
    y = torch.empty((R, W), dtype=x.dtype, device=x.device)
    _lib.check(eng.lib.mcmc_dropout_forward(eng.ctx.handle, _DT[x.dtype], act, x.data_ptr(), x.stride(0), R, W, seed, _ptr(seed_dev), p, pair, row_begin,
                                            elem_begin, y.data_ptr(), W, _stream(eng)), "mcmc_dropout_forward")
    return y, x


class _PhiloxDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, eng, x, seed_dev, args):
        with _on(eng):
            y, x2 = _dropout(eng, x, args)
        ctx.eng, ctx.args, ctx.sizes = eng, args, x2.shape
        ctx.save_for_backward(x2 if args[3] != _lib.ACT_NONE else None, seed_dev)
        return y.view(x.shape)

    @staticmethod
    @_once
    def backward(ctx, dy):
        eng, (p, seed, _, act, pair, row_begin, elem_begin) = ctx.eng, ctx.args
        x, seed_dev = ctx.saved_tensors
        R, W = ctx.sizes
        with _on(eng):
            dx = torch.empty_like(dy, memory_format=torch.contiguous_format)
            x = None if x is None else _rows(x)  # hooks on saved tensors may have changed its strides
            ld = W
            if not dy.is_contiguous():
                dy = _rows(_flat(dy))
                ld = dy.stride(0)
            _lib.check(eng.lib.mcmc_dropout_backward(eng.ctx.handle, _DT[dy.dtype], act, dy.data_ptr(), ld, _ptr(x), 0 if x is None else x.stride(0), R, W,
                                                     seed, _ptr(seed_dev), p, pair, row_begin, elem_begin, dx.data_ptr(), W, _stream(eng)),
                       "mcmc_dropout_backward")
        return None, dx, None, None


def philox_dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], *, activation: Optional[str] = None, pair: int = 0,
                   row_begin: int = 0, elem_begin: int = 0) -> torch.Tensor:
    """``act(x) * keep / (1 - p)`` with the mask drawn from the framework's counter-based stream where it is used, forward and
    backward, and never stored.

    The last dimension of x holds a row's elements, the others count rows (row-major).  Column c of row r is element
    ``elem_begin + c`` of row ``row_begin + r`` of ``pair``: a batch cut into pieces draws the same masks as the whole with
    ``row_begin`` set, and elem_begin (a multiple of 16) 0 / 256 / 384 with a pair's global id gives the masks of ``mcmc_train_forward``'s three
    hidden layers.  A dropped element is 0 whatever x holds there.

    activation: None or "elu" (alpha 1), applied before the dropout.  p in [0, 1), taken in float32; the keep probability is
    (1 - p) rounded down to a multiple of 2^-16 while the scale stays 1 / (1 - p), as in the fused kernels: the mean is low by up to
    2^-16 / (1 - p) of itself (1.5e-4 at p = 0.9), and from p > 1 - 2^-16 on everything is dropped.  seed: a 64-bit integer, or a
    one-element int64 tensor on x's device that is read when the kernel runs, so that a captured graph can be replayed with other
    masks (keep its value until the backward pass has run)."""
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    _dtype(x, "x")
    if activation not in _ACT:
        raise ValueError(f"activation must be None or 'elu', got {activation!r}")
    for name, v in (("pair", pair), ("row_begin", row_begin), ("elem_begin", elem_begin)):
        if not 0 <= int(v) <= 1 << 32:
            raise ValueError(f"{name} must be in [0, 2^32), got {v}")
    seed_dev = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"a seed tensor must hold one int64, got {seed.dtype} {tuple(seed.shape)}")
        seed, seed_dev = 0, seed
    eng = _engine(x, "x", seed=seed_dev)
    args = (float(p), int(seed) & _U64, seed_dev, _ACT[activation], int(pair), int(row_begin), int(elem_begin))
    if _wants_grad(x):
        return _PhiloxDropout.apply(eng, x, seed_dev, args)
    with _on(eng):
        return _dropout(eng, x, args)[0].view(x.shape)
