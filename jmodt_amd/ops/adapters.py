"""Low-rank adapters of many requests at once beside a shared projection (csrc/adapters.hip): rows of different frames, each with the
adapter of its sensor rig (or with none), through one dense layer of `ops/rows.py`:

    out[r] = base[r] + scales[a] * B_a (A_a x[r])       a = ids[r], base = the shared projection's output for row r

`AdapterPlan` finds the rows of every adapter on the device (no host synchronisation) and serves every layer of a step;
`adapter_forward` / `adapter_grad` are the two directions, `adapter_linear` the differentiable layer, whose input can be kept in
8 bits for the backward (`ops/rows8.py`).  float32, bfloat16 or float16 rows; sums and the rank-sized activations are float32; every
result is rounded once and the same bits every time.  No CPU path.
"""
from typing import Optional, Tuple, Union

import torch
from torch.autograd import Function

from .. import _lib as L
from . import rows as R
from .rows8 import TYPES, Rows8, _kept, _matrix, _on_device, checkpoint_rows, linear_wgrad8

_f32, _i32 = torch.float32, torch.int32
MAX_RANK, MAX_ADAPTERS = 128, 1023


class AdapterPlan:
    """The rows of every adapter, in device memory: ids (M,) int32, the adapter of each row; a value outside 0 .. adapters - 1 is a
    row without one.  Built on the current stream; ids may be reused afterwards."""

    def __init__(self, ids: torch.Tensor, adapters: int):
        adapters = int(adapters)
        if not 1 <= adapters <= MAX_ADAPTERS:
            raise ValueError(f"{adapters} adapters; 1 .. {MAX_ADAPTERS} are supported")
        _on_device(ids, "ids")
        if ids.dtype != _i32 or ids.dim() != 1 or not ids.is_contiguous():
            raise TypeError(f"ids must be a contiguous 1-D int32 tensor, got {ids.dtype} {tuple(ids.shape)}")
        lib = L.load()
        self.rows, self.adapters = ids.shape[0], adapters
        self.data = torch.empty((lib.jm_adapter_plan_elems(self.rows, adapters),), dtype=_i32, device=ids.device)
        L.check(lib.jm_adapter_plan(self.rows, adapters, ids.data_ptr(), self.data.data_ptr(), L.stream_ptr()), "AdapterPlan")


def _weights(a, b, scales, plan, dtype, k: int, n: int, m: int):
    """checks of the adapters' tensors -> (rank, adapters)"""
    if not isinstance(plan, AdapterPlan):
        raise TypeError(f"plan: expected AdapterPlan, got {type(plan).__name__}")
    _on_device(plan.data, "plan")
    for t, name in ((a, "a"), (b, "b")):
        _on_device(t, name)
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype} like the rows, got {t.dtype}")
        if t.dim() != 3 or not t.is_contiguous():
            raise RuntimeError(f"{name} must be a contiguous 3-D tensor, got {tuple(t.shape)}")
    count, rank = a.shape[0], a.shape[1]
    if tuple(a.shape) != (count, rank, k) or tuple(b.shape) != (count, n, rank):
        raise ValueError(f"a {tuple(a.shape)}, b {tuple(b.shape)}: expected (adapters, rank, {k}) and (adapters, {n}, rank)")
    if not 1 <= rank <= MAX_RANK:
        raise ValueError(f"rank {rank}; 1 .. {MAX_RANK} are supported")
    if plan.adapters != count:
        raise ValueError(f"a plan of {plan.adapters} adapters for {count}")
    if plan.rows != m:
        raise ValueError(f"a plan of {plan.rows} rows for {m}")
    _on_device(scales, "scales")
    if scales.dtype != _f32 or tuple(scales.shape) != (count,) or not scales.is_contiguous():
        raise TypeError(f"scales must be a contiguous float32 tensor of ({count},), got {scales.dtype} {tuple(scales.shape)}")
    return rank, count


def _span(t: torch.Tensor) -> Tuple[int, int]:
    p, s = t.data_ptr(), t.element_size()
    if t.numel() == 0:
        return p, p
    return p, p + s * (1 + sum((d - 1) * st for d, st in zip(t.shape, t.stride())))


def _disjoint(out: torch.Tensor, other: torch.Tensor, name: str) -> None:
    """refuses an output that shares elements with an input (columns beside each other in rows of one buffer are fine)"""
    a0, a1 = _span(out)
    b0, b1 = _span(other)
    if a0 >= b1 or b0 >= a1:
        return
    if out.dim() == 2 and other.dim() == 2 and out.element_size() == other.element_size() and out.shape[0] > 1 and other.shape[0] > 1:
        ld = out.stride(0)
        if ld == other.stride(0):
            d = ((b0 - a0) // out.element_size()) % ld          # columns from out's first to other's first
            if d >= out.shape[1] and d + other.shape[1] <= ld:
                return
    raise RuntimeError(f"out shares memory with {name}")


def _result(base, out, m: int, n: int, like: torch.Tensor, others):
    """(base address, base row stride, out): checks of base / out, out allocated when not given"""
    pb, ldb = None, 0
    if base is not None:
        pb, ldb = _matrix(base, "base", like.dtype)
        if tuple(base.shape) != (m, n):
            raise ValueError(f"base {tuple(base.shape)}: expected ({m}, {n})")
    if out is None:
        return pb, ldb, torch.empty((m, n), dtype=like.dtype, device=like.device)
    _matrix(out, "out", like.dtype)
    if tuple(out.shape) != (m, n):
        raise ValueError(f"out {tuple(out.shape)}: expected ({m}, {n})")
    same = base is not None and out.data_ptr() == base.data_ptr() and out.stride() == base.stride()
    for t, name in others + ([(base, "base")] if base is not None and not same else []):
        _disjoint(out, t, name)
    return pb, ldb, out


def adapter_forward(base: Optional[torch.Tensor], x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor, plan: AdapterPlan,
                    out: Optional[torch.Tensor] = None, want_t: bool = False):
    """base (M, N) or None (zero), x (M, K), a (adapters, R, K), b (adapters, N, R), scales (adapters,) float32 ->
    out = base + scales[a] B_a (A_a x) row by row; rows without an adapter: base.  out: a tensor to write (base itself: in place),
    else a new one.  want_t: (out, t), t (M, R) float32 = A_a x, zero in rows without an adapter — what `adapter_grad` needs."""
    px, ldx = _matrix(x, "x")
    m, k = x.shape
    n = b.shape[1] if isinstance(b, torch.Tensor) and b.dim() == 3 else 0
    rank, count = _weights(a, b, scales, plan, x.dtype, k, n, m)
    pb, ldb, out = _result(base, out, m, n, x, [(x, "x"), (a, "a"), (b, "b"), (scales, "scales")] if out is not None else [])
    t = torch.empty((m, rank), dtype=_f32, device=x.device) if want_t else None
    L.check(L.load().jm_adapter_forward(m, k, n, rank, count, TYPES[x.dtype], px, ldx, a.data_ptr(), b.data_ptr(), scales.data_ptr(), plan.data.data_ptr(),
                                        pb, ldb, out.data_ptr(), out.stride(0) if m > 1 else n, t.data_ptr() if want_t else None, L.stream_ptr()),
            "adapter_forward")
    return (out, t) if want_t else out


def adapter_grad(dy: torch.Tensor, x: Union[torch.Tensor, Rows8], t: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor, plan: AdapterPlan,
                 base: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """the gradients of adapter_forward: dy (M, N), x (M, K) or its kept form, t from the forward ->
    (dx (M, K) = base + scales[a] A_a^T (B_a^T dy), da like a, db like b).  base: the shared projection's data gradient, or None;
    out: a tensor for dx (base itself: in place).  An adapter without rows gets zeros."""
    pdy, ldd = _matrix(dy, "dy")
    m, n = dy.shape
    kept = isinstance(x, Rows8)
    if kept:
        _kept(x, "x")
        px, ldx = None, 0
        pc, ldc, pe = x.codes.data_ptr(), x.codes.shape[1], x.exps.data_ptr()
    else:
        px, ldx = _matrix(x, "x", dy.dtype)
        pc, ldc, pe = None, 0, None
    if x.shape[0] != m:
        raise ValueError(f"dy of {m} rows for an input of {x.shape[0]}")
    k = x.shape[1]
    rank, count = _weights(a, b, scales, plan, dy.dtype, k, n, m)
    _on_device(t, "t")
    if t.dtype != _f32 or tuple(t.shape) != (m, rank) or not t.is_contiguous():
        raise TypeError(f"t must be a contiguous float32 tensor of ({m}, {rank}), got {t.dtype} {tuple(t.shape)}")
    others = [] if out is None else [(dy, "dy"), (t, "t"), (a, "a"), (b, "b"), (scales, "scales")] + ([(x.codes, "x"), (x.exps, "x")] if kept else [(x, "x")])
    pb, ldb, dx = _result(base, out, m, k, dy, others)
    da, db = torch.empty_like(a), torch.empty_like(b)
    lib = L.load()
    nbytes = lib.jm_adapter_grad_workspace_bytes(m, k, n, rank, count, TYPES[dy.dtype])
    ws = torch.empty(((nbytes + 3) // 4,), dtype=_f32, device=dy.device)
    if not kept and m == 0:
        px = a.data_ptr()          # (an empty tensor has no address; nothing is read)
    L.check(lib.jm_adapter_grad(m, k, n, rank, count, TYPES[dy.dtype], pdy, ldd, px, max(ldx, k), pc, ldc, pe, (m + 15) // 16 * 16, t.data_ptr(), a.data_ptr(), b.data_ptr(),
                                scales.data_ptr(), plan.data.data_ptr(), pb, ldb, dx.data_ptr(), dx.stride(0) if m > 1 else k, da.data_ptr(), db.data_ptr(),
                                ws.data_ptr(), nbytes, L.stream_ptr()), "adapter_grad")
    return dx, da, db


class _AdapterLinear(Function):
    """apply(x, w, bias, a, b, scales, plan, keep): the dense layer and its adapters; keep: x is kept in 8 bits for the backward"""

    @staticmethod
    def forward(ctx, x, w, bias, a, b, scales, plan, keep):
        y = R.linear_forward(x, w, bias)
        a, b = a.contiguous(), b.contiguous()
        y, t = adapter_forward(y, x, a, b, scales, plan, out=y, want_t=True)
        ctx.plan, ctx.keep, ctx.channels, ctx.has_bias = plan, keep, x.shape[1], bias is not None
        if keep:
            x8 = checkpoint_rows(x)
            ctx.save_for_backward(x8.codes, x8.exps, w, a, b, scales, t)
        else:
            ctx.save_for_backward(x, w, a, b, scales, t)
        return y

    @staticmethod
    def backward(ctx, dy):
        saved = ctx.saved_tensors
        if ctx.keep:
            x, (w, a, b, scales, t) = Rows8(saved[0], saved[1], ctx.channels), saved[2:]
        else:
            x, (w, a, b, scales, t) = saved[0], saved[1:]
        if dy.dim() != 2 or dy.stride(1) != 1 or dy.stride(0) % 4 or dy.stride(0) < dy.shape[1] or dy.data_ptr() % 16:
            dy = dy.contiguous()
        need = ctx.needs_input_grad
        base = R.linear_dgrad(dy, w, 0, w.shape[1]) if need[0] else None
        dx = da = db = dw = dbias = None
        if need[0] or need[3] or need[4]:
            dx, da, db = adapter_grad(dy, x, t, a, b, scales, ctx.plan, base=base, out=base)
        if need[1] or (ctx.has_bias and need[2]):
            dw, dbias = linear_wgrad8(dy, x, want_bias=ctx.has_bias) if ctx.keep else R.linear_wgrad(dy, [x], want_bias=ctx.has_bias)
        return (dx if need[0] else None, dw if need[1] else None, dbias if ctx.has_bias and need[2] else None, da if need[3] else None,
                db if need[4] else None, None, None, None)


def adapter_linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor,
                   plan: AdapterPlan, keep: str = "float32") -> torch.Tensor:
    """y (M, N) = x w^T + bias + scales[a] B_a (A_a x): ops.rows.linear_forward and the rows' adapters, float32, differentiable in x, w,
    bias, a and b (a frozen projection: w and bias without requires_grad).  keep = "e4m3": x is kept in 8 bits for the backward
    (da and dw from the kept values), "float32": as it is.  Widths are multiples of 4, as everywhere in ops.rows."""
    if keep not in ("float32", "e4m3"):
        raise ValueError(f"keep must be 'float32' or 'e4m3', got {keep!r}")
    if isinstance(scales, torch.Tensor) and scales.requires_grad:
        raise ValueError("scales are constants of the layer: their gradient is not computed")
    return _AdapterLinear.apply(x, w, bias, a, b, scales, plan, keep == "e4m3")
