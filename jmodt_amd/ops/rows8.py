"""Row activations kept in 8 bits between the forward and the backward pass (csrc/rows8.hip): what `ops/rows.py` keeps in float32
(4 bytes an element), kept as e4m3 codes with one power-of-two scale per 32 channels of a row (1.03 bytes), and the backward's use of
it — the weight gradient from the codes, the ReLU's mask from the codes.

The format.  For a block of 32 channels of a row: amax = the largest finite |x|; the scale 2^e = the smallest power of two with
amax <= 448 * 2^e, e >= -100; a code is x / 2^e rounded to the nearest e4m3 value (ties to even: at most 2^-4 of the value, within
2^14 of the block's maximum).  A value that is not zero never becomes zero, so the sign pattern survives and the mask of a ReLU is
exact (of a ReLU's outputs only +infinity is not finite, and its gradient passes); a value that is not finite becomes NaN (e4m3 has no
infinity).  Kept values are exact in bfloat16 and float32.

No CPU path: every entry raises on tensors that are not on the current GPU.
"""
import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib as L

_f32, _u8 = torch.float32, torch.uint8
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # JM_F32, JM_BF16, JM_F16
BLOCK = 32
MAX_ROWS, MAX_CHANNELS = 1 << 30, 1 << 22


def _on_device(t, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a GPU tensor (jmodt_amd has no CPU path); got device {t.device}")
    if t.get_device() != L._current_device():
        raise RuntimeError(f"{name} lives on {t.device} but the current device is cuda:{L._current_device()}; "
                           "wrap the call in `with torch.cuda.device(tensor.device):`")


def _matrix(t, name: str, dtype: Optional[torch.dtype] = None) -> Tuple[int, int, int, int]:
    """(rows, channels, address, row stride) of a 2-D row tensor: unit column stride, any row stride >= its width, any alignment"""
    try:
        if t.get_device() == L._current_device() and t.dim() == 2 and t.is_contiguous() and (t.dtype is dtype or (dtype is None and t.dtype in TYPES)):
            m, c = t.shape
            if 0 < c <= MAX_CHANNELS and m <= MAX_ROWS:
                return m, c, t.data_ptr(), c
    except AttributeError:
        pass                                                 # (not a tensor: refused below, like everything else that is not the usual case)
    _on_device(t, name)
    if t.dim() != 2:
        raise TypeError(f"{name} must be 2-D (rows, channels), got {tuple(t.shape)}")
    if dtype is None:
        if t.dtype not in TYPES:
            raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    elif t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    m, c = t.shape
    if c == 0:
        raise ValueError(f"{name} has no channels")
    if m > MAX_ROWS or c > MAX_CHANNELS:
        raise ValueError(f"{name}: {m} rows of {c} channels; at most {MAX_ROWS} rows and {MAX_CHANNELS} channels are supported")
    if c > 1 and t.stride(1) != 1:
        raise RuntimeError(f"{name} must have unit column stride")
    ld = t.stride(0) if m > 1 else c
    if ld < c:
        raise RuntimeError(f"{name}: rows {ld} apart overlap (width {c}); pass a contiguous tensor")
    return m, c, t.data_ptr(), ld


def _bytes(t: torch.Tensor) -> int:
    """from the tensor's first byte to behind its last one"""
    if t.is_contiguous():
        return t.numel() * t.element_size()
    return t.element_size() * (1 + sum((d - 1) * st for d, st in zip(t.shape, t.stride()))) if t.numel() else 0


def _disjoint(p: int, size: int, out: torch.Tensor, other: torch.Tensor, name: str) -> None:
    """refuses an output (`size` bytes at p) that shares elements with an input; columns beside each other in rows of one buffer are fine"""
    q = other.data_ptr()
    if q >= p + size or q + _bytes(other) <= p:
        return
    if other.dim() == 2 and out.element_size() == other.element_size() and out.shape[0] > 1 and other.shape[0] > 1:
        ld = out.stride(0)
        if ld == other.stride(0):
            d = ((q - p) // out.element_size()) % ld          # columns from out's first to other's first
            if d >= out.shape[1] and d + other.shape[1] <= ld:
                return
    raise RuntimeError(f"out shares memory with {name}")


def _sizes(m: int, c: int) -> Tuple[int, int, int]:
    """(bytes of a row of codes, blocks of a row, bytes of a block's scale column)"""
    return (c + 15) & ~15, (c + BLOCK - 1) // BLOCK, (m + 15) & ~15


class Rows8:
    """A kept row tensor of `shape` = (rows, channels) in one buffer, `data` (uint8): `codes` (rows, channels rounded up to 16), zeros behind
    the channels, then `exps`, (rows, ceil(channels / 32)) scale bytes stored column by column, a column padded to 16 rows; a block's scale is
    2^(exps - 127).  `data` is what an autograd function saves."""
    __slots__ = ("data", "shape")

    def __init__(self, data: torch.Tensor, rows: int, channels: int):
        rows, channels = int(rows), int(channels)
        if not isinstance(data, torch.Tensor) or data.dtype != _u8 or data.dim() != 1 or not data.is_contiguous():
            raise TypeError("data must be a contiguous 1-D uint8 tensor")
        if not 0 <= rows <= MAX_ROWS or not 0 < channels <= MAX_CHANNELS:
            raise ValueError(f"({rows}, {channels}) rows and channels")
        ld, nb, mp = _sizes(rows, channels)
        if data.shape[0] != rows * ld + nb * mp:
            raise ValueError(f"({rows}, {channels}) takes {rows * ld + nb * mp} bytes, got {data.shape[0]}")
        if data.data_ptr() % 16:
            raise RuntimeError("data must be 16-byte aligned")
        self.data, self.shape = data, (rows, channels)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, exps: torch.Tensor) -> "Rows8":
        """from codes (rows, channels) and exps (rows, ceil(channels / 32)), e.g. read from a file.  They are taken as they are: scale bytes as
        checkpoint_rows writes them are 27 .. 247 (0 and 255 are no scales)"""
        if codes.dtype != _u8 or codes.dim() != 2 or exps.dtype != _u8 or exps.dim() != 2:
            raise TypeError("codes and exps must be 2-D uint8 tensors")
        m, c = codes.shape
        ld, nb, mp = _sizes(m, c)
        if tuple(exps.shape) != (m, nb) or c == 0:
            raise ValueError(f"{c} channels need exps of ({m}, {nb}), got {tuple(exps.shape)}")
        out = cls(torch.zeros((m * ld + nb * mp,), dtype=_u8, device=codes.device), m, c)
        out.codes[:, :c] = codes
        out.exps.copy_(exps)
        return out

    @property
    def codes(self) -> torch.Tensor:
        m, c = self.shape
        ld = (c + 15) & ~15
        return self.data.as_strided((m, ld), (ld, 1))

    @property
    def exps(self) -> torch.Tensor:
        m, c = self.shape
        ld, nb, mp = _sizes(m, c)
        return self.data.as_strided((m, nb), (1, mp), self.data.storage_offset() + m * ld)

    @property
    def device(self):
        return self.data.device

    def nbytes(self) -> int:
        return self.data.numel()


def _kept(x8, name: str) -> Tuple[int, int, int, int, int, int]:
    """(rows, channels, address of the codes, bytes of their rows, address of the scales, bytes of their columns)"""
    if not isinstance(x8, Rows8):
        raise TypeError(f"{name}: expected Rows8, got {type(x8).__name__}")
    if x8.data.get_device() != L._current_device():
        _on_device(x8.data, name)
    m, c = x8.shape
    ld = (c + 15) & ~15
    p = x8.data.data_ptr()
    return m, c, p, ld, p + m * ld, (m + 15) & ~15


def checkpoint_rows(x: torch.Tensor) -> Rows8:
    """x (M, C) float32 / bfloat16 / float16 (any row stride) -> its kept form.  Not differentiable: it stands for x in x's backward."""
    m, c, px, ldx = _matrix(x, "x")
    ld, nb, mp = _sizes(m, c)
    data = torch.empty((m * ld + nb * mp,), dtype=_u8, device=x.device)
    pc = data.data_ptr()
    L.check(L.load().jm_rows8_pack(m, c, TYPES[x.dtype], px, ldx, pc, ld, pc + m * ld, mp, L.stream_ptr()), "checkpoint_rows")
    out = Rows8.__new__(Rows8)
    out.data, out.shape = data, (m, c)
    return out


def restore_rows(x8: Rows8, dtype: torch.dtype = _f32) -> torch.Tensor:
    """the kept values (M, C), exact in float32 and bfloat16, rounded once in float16"""
    m, c, pc, ld, pe, mp = _kept(x8, "x8")
    if dtype not in TYPES:
        raise TypeError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    out = torch.empty((m, c), dtype=dtype, device=x8.data.device)
    L.check(L.load().jm_rows8_restore(m, c, TYPES[dtype], pc, ld, pe, mp, out.data_ptr(), c, L.stream_ptr()), "restore_rows")
    return out


def relu_mask8(dy: torch.Tensor, y8: Rows8, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """kept y > 0 ? dy : 0 in float32 (a new tensor, or `out`, which may be dy): the gradient through a ReLU from its kept output.  A kept
    value that is not finite counts as positive (a ReLU's output is never below zero: it was +infinity)"""
    m, c, pdy, ldd = _matrix(dy, "dy", _f32)
    m8, c8, pc, ld, _, _ = _kept(y8, "y8")
    if (m, c) != (m8, c8):
        raise ValueError(f"dy {tuple(dy.shape)} for a kept output {y8.shape}")
    if out is None:
        out = torch.empty((m, c), dtype=_f32, device=dy.device)
    mo, co, po, ldo = _matrix(out, "out", _f32)
    if (mo, co) != (m, c):
        raise ValueError(f"out {tuple(out.shape)}: expected ({m}, {c})")
    if po != pdy or ldo != ldd:
        _disjoint(po, _bytes(out), out, dy, "dy")
    _disjoint(po, _bytes(out), out, y8.data, "y8")
    L.check(L.load().jm_rows8_relu_mask(m, c, pdy, ldd, pc, ld, po, ldo, L.stream_ptr()), "relu_mask8")
    return out


def linear_wgrad8(dy: torch.Tensor, x8: Rows8, want_bias: bool = True, out: Optional[torch.Tensor] = None,
                  col0: int = 0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(dw (N, K) = dy^T x, dbias (N) or None) in float32, dy (M, N) float32 / bfloat16 / float16, x (M, K) kept: ops.rows.linear_wgrad
    with the input as `checkpoint_rows` left it.  Rows of dy are at most 2^22 elements apart.  out / col0: write the block
    into columns col0 .. of an (N, >= col0 + K) tensor."""
    m, n, pdy, ldd = _matrix(dy, "dy")
    m8, k, pc, ld, pe, mp = _kept(x8, "x8")
    if m8 != m:
        raise ValueError(f"dy of {m} rows for a kept input of {m8}")
    lib = L.load()
    device = dy.device
    if out is None:
        dw = torch.empty((n, k), dtype=_f32, device=device)
        pw, ldw = dw.data_ptr(), k
    else:
        dw = out
        nw, kw, pw, ldw = _matrix(out, "out", _f32)
        if nw != n or col0 < 0 or col0 + k > kw:
            raise ValueError(f"out {tuple(out.shape)} for columns {col0} .. {col0 + k - 1} of ({n}, ...)")
        pw += 4 * col0
        block = out[:, col0:col0 + k]
        for t, name in ((dy, "dy"), (x8.data, "x8")):
            _disjoint(pw, _bytes(block), block, t, name)
    db = torch.empty((n,), dtype=_f32, device=device) if want_bias else None
    nbytes = lib.jm_rows8_wgrad_workspace_bytes(m, n, k)
    ws = torch.empty((nbytes // 4,), dtype=_f32, device=device) if nbytes else None
    L.check(lib.jm_rows8_linear_wgrad(m, n, k, TYPES[dy.dtype], pdy, ldd, pc, ld, pe, mp, pw, ldw, db.data_ptr() if want_bias else None,
                                      ws.data_ptr() if nbytes else None, nbytes, L.stream_ptr()), "linear_wgrad8")
    return dw, db


class _RowsMLP8(Function):
    """ops.rows._RowsMLP with its inputs and its hidden activations kept in 8 bits: apply(x1, x2 or None, acts, held, k1, box, W_0, b_0, W_1,
    b_1, ...), acts in {0 none, 1 ReLU}.  The forward's values are the float32 route's own; of the gradients only dW_l see the rounding of
    the kept activations (the masks are exact, dx and db need none of them).  Only what a gradient needs is kept and computed: an input for
    its layer's weight, an output for the mask of its ReLU, and nothing below the last layer that something trains in.
    held: those of "x1", "x2", "y" that are kept in float32 elsewhere and saved as they are; k1: x1's kept form where there is one; box: a list
    that takes y's (or None)."""

    @staticmethod
    def forward(ctx, x1, x2, acts, held, k1, box, *wb):
        from . import rows as R
        Ws, bs, nl = wb[0::2], wb[1::2], len(acts)
        need = ctx.needs_input_grad
        need_w, train = need[6::2], [w or b for w, b in zip(need[6::2], need[7::2])]
        # the last layer that the backward walks down to; -1: through all of them, to the inputs
        ctx.low = -1 if need[0] or need[1] else train.index(True) if True in train else nl
        keep = []
        for x, name, k in ((x1, "x1", k1), (x2, "x2", None)):
            keep.append(None if x is None or not need_w[0] else x if name in held else k or checkpoint_rows(x))
        cur, cur2 = x1, x2
        for l, act in enumerate(acts):
            cur, cur2 = R.linear_forward(cur, Ws[l], bs[l], act, x2=cur2), None
            if (act == 1 and l >= ctx.low) or (l + 1 < nl and need_w[l + 1]):
                keep.append(cur if l + 1 == nl and "y" in held else checkpoint_rows(cur))
            else:
                keep.append(None)
        box.append(keep[-1] if isinstance(keep[-1], Rows8) else None)
        ctx.acts, ctx.k = acts, (x1.shape[1], None if x2 is None else x2.shape[1])
        ctx.shapes = [k.shape if isinstance(k, Rows8) else None for k in keep]
        ctx.save_for_backward(*[k.data if isinstance(k, Rows8) else k for k in keep], *Ws)
        return cur

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        from . import rows as R
        acts, nl, need = ctx.acts, len(ctx.acts), ctx.needs_input_grad
        kept = [d if s is None else Rows8(d, *s) for d, s in zip(ctx.saved_tensors, ctx.shapes)]
        Ws = ctx.saved_tensors[nl + 2:]
        inputs, ys = kept[:2], kept[2:]

        def wgrad(x, want_bias, out=None, col0=0):
            if isinstance(x, Rows8):
                return linear_wgrad8(dy, x, want_bias=want_bias, out=out, col0=col0)
            return R.linear_wgrad(dy, [x], want_bias=want_bias, out=out, col0=col0)

        dy = R._gradient(dy)
        if acts[-1] == 1:
            dy = relu_mask8(dy, ys[-1]) if isinstance(ys[-1], Rows8) else R.relu_mask(dy, ys[-1])
        grads = [None] * (2 * nl)
        for l in range(nl - 1, max(ctx.low, 0) - 1, -1):
            need_w, need_b = need[6 + 2 * l], need[7 + 2 * l]
            if need_w and l > 0:
                grads[2 * l], grads[2 * l + 1] = wgrad(ys[l - 1], need_b)
            elif need_w:
                k1, k2 = ctx.k
                dw = torch.empty(Ws[0].shape, dtype=_f32, device=dy.device)
                grads[0], grads[1] = wgrad(inputs[0], need_b, out=dw)
                if k2 is not None:
                    wgrad(inputs[1], False, out=dw, col0=k1)
            elif need_b:
                grads[2 * l + 1] = R.colsum(dy)
            if l > max(ctx.low, 0):
                dy = R.linear_dgrad(dy, Ws[l], 0, Ws[l].shape[1])
                if acts[l - 1] == 1:
                    relu_mask8(dy, ys[l - 1], out=dy)
        dx1 = R.linear_dgrad(dy, Ws[0], 0, ctx.k[0]) if need[0] else None
        dx2 = R.linear_dgrad(dy, Ws[0], ctx.k[0], ctx.k[1]) if need[1] else None
        return (dx1, dx2, None, None, None, None, *grads)
