"""Row activations kept in 8 bits between the forward and the backward pass (csrc/rows8.hip): what `ops/rows.py` keeps in float32
(4 bytes an element), kept as e4m3 codes with one power-of-two scale per 32 channels of a row (1.03 bytes), and the backward's use of
it — the weight gradient from the codes, the ReLU's mask from the codes.

The format.  For a block of 32 channels of a row: amax = the largest finite |x|; the scale 2^e = the smallest power of two with
amax <= 448 * 2^e, e >= -100; a code is x / 2^e rounded to the nearest e4m3 value (ties to even: at most 2^-4 of the value, within
2^14 of the block's maximum).  A value that is not zero never becomes zero, so the sign pattern survives and the mask of a ReLU is
exact; a value that is not finite becomes NaN (e4m3 has no infinity).  Kept values are exact in bfloat16 and float32.

No CPU path: every entry raises on tensors that are not on the current GPU.
"""
import ctypes
from typing import Optional, Tuple

import torch

from .. import _lib as L

_f32, _u8 = torch.float32, torch.uint8
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # JM_F32, JM_BF16, JM_F16
BLOCK = 32


def _on_device(t, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a GPU tensor (jmodt_amd has no CPU path); got device {t.device}")
    if t.device.index != L._current_device():
        raise RuntimeError(f"{name} lives on {t.device} but the current device is cuda:{L._current_device()}; "
                           "wrap the call in `with torch.cuda.device(tensor.device):`")


def _matrix(t, name: str, dtype: Optional[torch.dtype] = None) -> Tuple[int, int]:
    """(address, row stride) of a 2-D row tensor: unit column stride, any row stride >= its width, any alignment"""
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
    if c > 1 and t.stride(1) != 1:
        raise RuntimeError(f"{name} must have unit column stride")
    ld = t.stride(0) if m > 1 else c
    if ld < c:
        raise RuntimeError(f"{name}: rows {ld} apart overlap (width {c}); pass a contiguous tensor")
    return t.data_ptr(), ld


def _exps(m: int, c: int, device) -> torch.Tensor:
    """(m, blocks of c) scale bytes, column by column in memory"""
    return torch.empty(((c + BLOCK - 1) // BLOCK, (m + 15) // 16 * 16), dtype=_u8, device=device).t()[:m]


class Rows8:
    """A kept row tensor: `codes` (rows, ld) uint8, ld = the channels rounded up to 16, zeros behind the channels; `exps`
    (rows, ceil(channels / 32)) uint8, column by column in memory, a column padded to 16 rows; a block's scale is 2^(exps - 127); `shape` = (rows, channels)."""
    __slots__ = ("codes", "exps", "shape")

    def __init__(self, codes: torch.Tensor, exps: torch.Tensor, channels: int):
        channels = int(channels)
        if not (isinstance(codes, torch.Tensor) and isinstance(exps, torch.Tensor)):
            raise TypeError("codes and exps must be tensors")
        if codes.dtype != _u8 or exps.dtype != _u8 or codes.dim() != 2 or exps.dim() != 2:
            raise TypeError("codes and exps must be 2-D uint8 tensors")
        m, ld = codes.shape
        if channels <= 0 or ld != (channels + 15) // 16 * 16 or tuple(exps.shape) != (m, (channels + BLOCK - 1) // BLOCK):
            raise ValueError(f"{channels} channels need codes (m, {(channels + 15) // 16 * 16}) and exps (m, {(channels + BLOCK - 1) // BLOCK}); "
                             f"got {tuple(codes.shape)} and {tuple(exps.shape)}")
        if codes.device != exps.device:
            raise RuntimeError(f"codes on {codes.device}, exps on {exps.device}")
        if not codes.is_contiguous() or codes.data_ptr() % 16:
            raise RuntimeError("codes must be contiguous and 16-byte aligned")
        if exps.data_ptr() % 16 or (m > 1 and exps.stride(0) != 1) or (exps.shape[1] > 1 and exps.stride(1) != (m + 15) // 16 * 16):
            raise RuntimeError("exps must be (blocks, rows rounded up to 16) in memory: Rows8.from_codes lays them out")
        self.codes, self.exps, self.shape = codes, exps, (m, channels)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, exps: torch.Tensor) -> "Rows8":
        """from codes (rows, channels) without padding, e.g. read from a file"""
        if codes.dtype != _u8 or codes.dim() != 2:
            raise TypeError("codes must be a 2-D uint8 tensor")
        m, c = codes.shape
        padded = torch.zeros((m, (c + 15) // 16 * 16), dtype=_u8, device=codes.device)
        padded[:, :c] = codes
        columns = _exps(m, c, codes.device)
        columns.copy_(exps)
        return cls(padded, columns, c)

    @property
    def device(self):
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + self.exps.numel()


def _kept(x8, name: str) -> Rows8:
    if not isinstance(x8, Rows8):
        raise TypeError(f"{name}: expected Rows8, got {type(x8).__name__}")
    _on_device(x8.codes, name)
    return x8


def checkpoint_rows(x: torch.Tensor) -> Rows8:
    """x (M, C) float32 / bfloat16 / float16 (any row stride) -> its kept form.  Not differentiable: it stands for x in x's backward."""
    px, ldx = _matrix(x, "x")
    m, c = x.shape
    codes = torch.empty((m, (c + 15) // 16 * 16), dtype=_u8, device=x.device)
    exps = _exps(m, c, x.device)
    L.check(L.load().jm_rows8_pack(m, c, TYPES[x.dtype], px, ldx, codes.data_ptr(), codes.shape[1], exps.data_ptr(), (m + 15) // 16 * 16, L.stream_ptr()), "checkpoint_rows")
    return Rows8(codes, exps, c)


def restore_rows(x8: Rows8, dtype: torch.dtype = _f32) -> torch.Tensor:
    """the kept values (M, C), exact in float32 and bfloat16, rounded once in float16"""
    _kept(x8, "x8")
    if dtype not in TYPES:
        raise TypeError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    m, c = x8.shape
    out = torch.empty((m, c), dtype=dtype, device=x8.device)
    L.check(L.load().jm_rows8_restore(m, c, TYPES[dtype], x8.codes.data_ptr(), x8.codes.shape[1], x8.exps.data_ptr(), (m + 15) // 16 * 16, out.data_ptr(), c, L.stream_ptr()),
            "restore_rows")
    return out


def relu_mask8(dy: torch.Tensor, y8: Rows8) -> torch.Tensor:
    """kept y > 0 ? dy : 0 as a new float32 tensor: the gradient through a ReLU from its kept output"""
    pdy, ldd = _matrix(dy, "dy", _f32)
    _kept(y8, "y8")
    if tuple(dy.shape) != y8.shape:
        raise ValueError(f"dy {tuple(dy.shape)} for a kept output {y8.shape}")
    m, c = dy.shape
    out = torch.empty((m, c), dtype=_f32, device=dy.device)
    L.check(L.load().jm_rows8_relu_mask(m, c, pdy, ldd, y8.codes.data_ptr(), y8.codes.shape[1], out.data_ptr(), c, L.stream_ptr()), "relu_mask8")
    return out


def linear_wgrad8(dy: torch.Tensor, x8: Rows8, want_bias: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(dw (N, K) = dy^T x, dbias (N) or None) in float32, dy (M, N) float32 / bfloat16 / float16, x (M, K) kept: ops.rows.linear_wgrad
    with the input as `checkpoint_rows` left it"""
    pdy, ldd = _matrix(dy, "dy")
    _kept(x8, "x8")
    m, n = dy.shape
    if x8.shape[0] != m:
        raise ValueError(f"dy of {m} rows for a kept input of {x8.shape[0]}")
    k = x8.shape[1]
    lib = L.load()
    dw = torch.empty((n, k), dtype=_f32, device=dy.device)
    db = torch.empty((n,), dtype=_f32, device=dy.device) if want_bias else None
    nbytes = lib.jm_rows8_wgrad_workspace_bytes(m, n, k)
    ws = torch.empty((nbytes // 4,), dtype=_f32, device=dy.device) if nbytes else None
    L.check(lib.jm_rows8_linear_wgrad(m, n, k, TYPES[dy.dtype], pdy, ldd, x8.codes.data_ptr(), x8.codes.shape[1], x8.exps.data_ptr(), (m + 15) // 16 * 16, dw.data_ptr(), k,
                                      db.data_ptr() if want_bias else None, ws.data_ptr() if ws is not None else None, nbytes, L.stream_ptr()),
            "linear_wgrad8")
    return dw, db
