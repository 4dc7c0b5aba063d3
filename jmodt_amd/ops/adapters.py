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
from torch.autograd.function import once_differentiable

from .. import _lib as L
from . import rows as R
from .rows8 import TYPES, Rows8, _bytes, _disjoint, _kept, _matrix, _on_device, checkpoint_rows, linear_wgrad8

_f32, _i32 = torch.float32, torch.int32
MAX_RANK, MAX_ADAPTERS, MAX_ROWS = 128, 1023, 1 << 28


class AdapterPlan:
    """The rows of every adapter, in device memory: ids (M,) int32, the adapter of each row; a value outside 0 .. adapters - 1 is a
    row without one.  Built on the current stream; ids may be reused afterwards.  On another stream: order it behind this one and
    keep the plan until it is done (or `data.record_stream`), as with every tensor."""

    def __init__(self, ids: torch.Tensor, adapters: int):
        adapters = int(adapters)
        if not 1 <= adapters <= MAX_ADAPTERS:
            raise ValueError(f"{adapters} adapters; 1 .. {MAX_ADAPTERS} are supported")
        _on_device(ids, "ids")
        if ids.dtype != _i32 or ids.dim() != 1 or not ids.is_contiguous():
            raise TypeError(f"ids must be a contiguous 1-D int32 tensor, got {ids.dtype} {tuple(ids.shape)}")
        if ids.shape[0] > MAX_ROWS:
            raise ValueError(f"{ids.shape[0]} rows; at most {MAX_ROWS} are supported")
        lib = L.load()
        self.rows, self.adapters = ids.shape[0], adapters
        self.data = torch.empty((lib.jm_adapter_plan_elems(self.rows, adapters),), dtype=_i32, device=ids.device)
        L.check(lib.jm_adapter_plan(self.rows, adapters, ids.data_ptr(), self.data.data_ptr(), L.stream_ptr()), "AdapterPlan")


def _weights(a, b, scales, plan, dtype, k: int, n: int, m: int):
    """checks of the adapters' tensors -> (rank, adapters)"""
    if not isinstance(plan, AdapterPlan):
        raise TypeError(f"plan: expected AdapterPlan, got {type(plan).__name__}")
    dev = L._current_device()
    try:
        here = plan.data.get_device() == dev and a.get_device() == dev and b.get_device() == dev and scales.get_device() == dev
    except AttributeError:
        here = False
    if not here:
        for v, name in ((plan.data, "plan"), (a, "a"), (b, "b"), (scales, "scales")):
            _on_device(v, name)
    if a.dtype != dtype or b.dtype != dtype:
        raise TypeError(f"a and b must be {dtype} like the rows, got {a.dtype} and {b.dtype}")
    if a.dim() != 3 or not a.is_contiguous() or b.dim() != 3 or not b.is_contiguous():
        raise RuntimeError(f"a and b must be contiguous 3-D tensors, got {tuple(a.shape)} and {tuple(b.shape)}")
    count, rank, ka = a.shape
    if ka != k or b.shape != (count, n, rank):
        raise ValueError(f"a {tuple(a.shape)}, b {tuple(b.shape)}: expected (adapters, rank, {k}) and (adapters, {n}, rank)")
    if not 1 <= rank <= MAX_RANK:
        raise ValueError(f"rank {rank}; 1 .. {MAX_RANK} are supported")
    if plan.adapters != count or plan.rows != m:
        raise ValueError(f"a plan of {plan.rows} rows and {plan.adapters} adapters for {m} and {count}")
    if scales.dtype != _f32 or scales.shape != (count,) or not scales.is_contiguous():
        raise TypeError(f"scales must be a contiguous float32 tensor of ({count},), got {scales.dtype} {tuple(scales.shape)}")
    return rank, count


def _result(base, out, m: int, n: int, like: torch.Tensor, others):
    """(base address, base row stride, out, its address, its row stride): checks of base / out, out allocated when not given"""
    pb, ldb = None, 0
    if base is not None:
        mb, nb, pb, ldb = _matrix(base, "base", like.dtype)
        if mb != m or nb != n:
            raise ValueError(f"base {tuple(base.shape)}: expected ({m}, {n})")
    if out is None:
        out = torch.empty_like(base) if ldb == n else torch.empty((m, n), dtype=like.dtype, device=like.device)
        return pb, ldb, out, out.data_ptr(), n
    if out is base:
        po, ldo = pb, ldb
    else:
        mo, no, po, ldo = _matrix(out, "out", like.dtype)
        if mo != m or no != n:
            raise ValueError(f"out {tuple(out.shape)}: expected ({m}, {n})")
    size = _bytes(out)
    if base is not None and not (po == pb and ldo == ldb):
        _disjoint(po, size, out, base, "base")
    for t, name in others:
        _disjoint(po, size, out, t, name)
    return pb, ldb, out, po, ldo


def adapter_forward(base: Optional[torch.Tensor], x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor, plan: AdapterPlan,
                    out: Optional[torch.Tensor] = None, want_t: bool = False):
    """base (M, N) or None (zero), x (M, K), a (adapters, R, K), b (adapters, N, R), scales (adapters,) float32 ->
    out = base + scales[a] B_a (A_a x) row by row; rows without an adapter: base.  out: a tensor to write (base itself: in place),
    else a new one.  want_t: (out, t), t (M, R) float32 = A_a x, zero in rows without an adapter — what `adapter_grad` needs.
    A value that is not finite reaches its own row (in x) or its adapter's rows (in a, b) only; in bfloat16 and float16, where t enters as a
    sum of several values, an infinity in b gives NaN."""
    m, k, px, ldx = _matrix(x, "x")
    n = b.shape[1] if isinstance(b, torch.Tensor) and b.dim() == 3 else 0
    rank, count = _weights(a, b, scales, plan, x.dtype, k, n, m)
    pb, ldb, out, po, ldo = _result(base, out, m, n, x, ((x, "x"), (a, "a"), (b, "b"), (scales, "scales"), (plan.data, "plan")))
    t = torch.empty((m, rank), dtype=_f32, device=x.device) if want_t else None
    L.check(L.load().jm_adapter_forward(m, k, n, rank, count, TYPES[x.dtype], px, ldx, a.data_ptr(), b.data_ptr(), scales.data_ptr(), plan.data.data_ptr(),
                                        pb, ldb, po, ldo, t.data_ptr() if want_t else None, L.stream_ptr()), "adapter_forward")
    return (out, t) if want_t else out


def adapter_grad(dy: torch.Tensor, x: Union[torch.Tensor, Rows8, None], t: Optional[torch.Tensor], a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor,
                 plan: AdapterPlan, base: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                 need: Tuple[bool, bool, bool] = (True, True, True)) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """the gradients of adapter_forward: dy (M, N), x (M, K) or its kept form, t from the forward ->
    (dx (M, K) = base + scales[a] A_a^T (B_a^T dy), da like a, db like b).  base: the shared projection's data gradient, or None;
    out: a tensor for dx (base itself: in place).  need: which of the three are wanted, the same bits; the others are None and not computed
    (base and out belong to dx; x may be None without da, t without db).  An adapter without rows gets zeros.  Infinities in x or dy
    (bfloat16) may give NaN in da and db."""
    m, n, pdy, ldd = _matrix(dy, "dy")
    if len(need) != 3:
        raise ValueError(f"need: three truth values for dx, da and db, got {need!r}")
    px, ldx, pc, ldc, pe, lde = None, 0, None, 0, None, 0
    others = [(dy, "dy"), (a, "a"), (b, "b"), (scales, "scales")]
    if isinstance(x, Rows8):
        mx, k, pc, ldc, pe, lde = _kept(x, "x")
        others.append((x.data, "x"))
    elif x is not None or need[1]:
        mx, k, px, ldx = _matrix(x, "x", dy.dtype)
        others.append((x, "x"))
        if m == 0:
            px = a.data_ptr()          # (an empty tensor has no address; nothing is read)
    else:
        mx, k = m, a.shape[2] if isinstance(a, torch.Tensor) and a.dim() == 3 else 0
    if mx != m:
        raise ValueError(f"dy of {m} rows for an input of {mx}")
    rank, count = _weights(a, b, scales, plan, dy.dtype, k, n, m)
    if t is not None or need[2]:
        _on_device(t, "t")
        if t.dtype != _f32 or t.shape != (m, rank) or not t.is_contiguous():
            raise TypeError(f"t must be a contiguous float32 tensor of ({m}, {rank}), got {t.dtype} {tuple(t.shape)}")
        others.append((t, "t"))
    pb, ldb, dx, po, ldo = None, 0, None, None, 0
    if need[0]:
        pb, ldb, dx, po, ldo = _result(base, out, m, k, dy, others + [(plan.data, "plan")])
    elif base is not None or out is not None:
        raise ValueError("base and out belong to dx, which is not wanted")
    da, db = torch.empty_like(a) if need[1] else None, torch.empty_like(b) if need[2] else None
    lib = L.load()
    kind = TYPES[dy.dtype]
    nbytes = lib.jm_adapter_grad_workspace_bytes(m, k, n, rank, count, kind)
    ws = torch.empty(((nbytes + 3) // 4,), dtype=_f32, device=dy.device)
    L.check(lib.jm_adapter_grad_select((1 if need[0] else 0) | (2 if need[1] else 0) | (4 if need[2] else 0), m, k, n, rank, count, kind, pdy, ldd, px, ldx, pc, ldc,
                                       pe, lde, None if t is None else t.data_ptr(), a.data_ptr(), b.data_ptr(), scales.data_ptr(), plan.data.data_ptr(), pb, ldb, po, ldo,
                                       da.data_ptr() if need[1] else None, db.data_ptr() if need[2] else None, ws.data_ptr(), nbytes, L.stream_ptr()), "adapter_grad")
    return dx, da, db


class _AdapterLinear(Function):
    """apply(x, w, bias, a, b, scales, plan, keep): the dense layer and its adapters; keep: x is kept in 8 bits for the backward (where w
    or a needs it at all)"""

    @staticmethod
    def forward(ctx, x, w, bias, a, b, scales, plan, keep):
        need = ctx.needs_input_grad
        y = R.linear_forward(x, w, bias)
        a, b = a.contiguous(), b.contiguous()
        y, t = adapter_forward(y, x, a, b, scales, plan, out=y, want_t=True) if need[4] else (adapter_forward(y, x, a, b, scales, plan, out=y), None)
        ctx.plan, ctx.keep, ctx.shape = plan, keep, tuple(x.shape)
        kept = None if not (need[1] or need[3]) else checkpoint_rows(x).data if keep else x
        ctx.save_for_backward(kept, w, a, b, scales, t)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, a, b, scales, t = ctx.saved_tensors
        if ctx.keep and x is not None:
            x = Rows8(x, *ctx.shape)
        dy = R._gradient(dy)
        need = ctx.needs_input_grad
        dx = da = db = dw = dbias = None
        if need[0] or need[3] or need[4]:
            base = R.linear_dgrad(dy, w, 0, w.shape[1]) if need[0] else None
            dx, da, db = adapter_grad(dy, x, t, a, b, scales, ctx.plan, base=base, out=base, need=(need[0], need[3], need[4]))
        if need[1]:
            dw, dbias = linear_wgrad8(dy, x, want_bias=need[2]) if ctx.keep else R.linear_wgrad(dy, [x], want_bias=need[2])
        elif need[2]:
            dbias = R.colsum(dy)
        return dx, dw, dbias, da, db, None, None, None


def adapter_linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor,
                   plan: AdapterPlan, keep: str = "float32") -> torch.Tensor:
    """y (M, N) = x w^T + bias + scales[a] B_a (A_a x): ops.rows.linear_forward and the rows' adapters, float32, differentiable in x, w,
    bias, a and b (a frozen projection: w and bias without requires_grad).  keep = "e4m3": x is kept in 8 bits for the backward
    (da and dw from the kept values), "float32": as it is.  Widths are multiples of 4 and there is at least one row, as everywhere in ops.rows.
    Forward and backward can be captured into a HIP graph together; as with every autograd function, no eager graph of the same leaves may be
    alive then (autograd keeps a leaf's accumulation on the stream of its first live graph) — take torch.autograd.grad on fresh leaves."""
    if keep not in ("float32", "e4m3"):
        raise ValueError(f"keep must be 'float32' or 'e4m3', got {keep!r}")
    if isinstance(scales, torch.Tensor) and scales.requires_grad:
        raise ValueError("scales are constants of the layer: their gradient is not computed")
    # (nothing is kept where no backward can follow)
    if not (torch.is_grad_enabled() and any(isinstance(v, torch.Tensor) and v.requires_grad for v in (x, w, bias, a, b))):
        y = R.linear_forward(x, w, bias)
        return adapter_forward(y, x, a.contiguous(), b.contiguous(), scales, plan, out=y)
    return _AdapterLinear.apply(x, w, bias, a, b, scales, plan, keep == "e4m3")
