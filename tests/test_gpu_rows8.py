"""Row activations kept in 8 bits (ops/rows8.py) against the definition in 64 bits.

Tolerances.  The kept form is a defined rounding: codes and scales are compared bit by bit.  A weight gradient sums m products that are
exact in float32 (or held to 24 bits): each addition is off by at most u = 2^-24 of its partial sum, whose size is at most S = sum |dy||x|;
m of them with independent signs stay within (8 + 2 sqrt(m)) u S."""
import math

import numpy as np
import pytest
import torch

from jmodt_amd.ops import rows8 as R8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def decode_table():
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v[c] = (m / 8.0 * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)) * (-1.0 if c & 128 else 1.0)
    v[127] = v[255] = np.nan
    return v


TABLE = decode_table()


def encode_ref(x):
    """(codes, exps) by the definition, from the table of e4m3 values: nearest, ties to the even code"""
    x = x.double().cpu().numpy()
    m, c = x.shape
    nb = (c + 31) // 32
    codes, exps = np.zeros((m, c), np.uint8), np.zeros((m, nb), np.uint8)
    pos = TABLE[:127]                                      # 0 .. 448 ascending
    for j in range(nb):
        p = x[:, 32 * j:32 * j + 32]
        fin = np.isfinite(p)
        amax = np.where(fin, np.abs(p), 0.0).max(axis=1) if p.size else np.zeros(m)
        e = np.full(m, -100)
        for r in range(m):
            if amax[r] > 0:
                k = math.frexp(amax[r])[1] - 9
                while amax[r] > 448.0 * 2.0 ** k:
                    k += 1
                while amax[r] <= 448.0 * 2.0 ** (k - 1):
                    k -= 1
                e[r] = max(-100, k)
        v = np.where(fin, p, 0.0) / (2.0 ** e.astype(float))[:, None]
        a = np.abs(v)
        hi = np.searchsorted(pos, a).clip(1, 126)
        lo = hi - 1
        dl, dh = a - pos[lo], pos[hi] - a
        code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
        code = np.where((code == 0) & (p != 0) & fin, 1, code)
        code = np.where(np.signbit(p) & (p != 0), code | 128, code)
        codes[:, 32 * j:32 * j + 32] = np.where(fin, code, 127)
        exps[:, j] = e + 127
    return codes, exps


def values(codes, exps):
    return TABLE[codes] * np.repeat(2.0 ** (exps.astype(float) - 127), 32, axis=1)[:, :codes.shape[1]]


def make(m, c, dtype, seed=0, relu=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, c, generator=g, device="cuda") * torch.exp(2 * torch.randn(m, 1, generator=g, device="cuda"))
    x = x.clamp(min=0) if relu else x
    return x.to(dtype)


DT = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,c", [(0, 8), (1, 1), (3, 5), (7, 16), (5, 31), (5, 33), (130, 64), (65, 196), (9, 515), (2000, 32)])
def test_keep(m, c, dtype):
    x = make(m, c, dtype, seed=m + c)
    k = R8.checkpoint_rows(x)
    codes, exps = encode_ref(x)
    neg0 = (codes & 127) == 0                              # (a zero's sign is not kept track of)
    got = k.codes.cpu().numpy()
    assert got.shape[1] % 16 == 0 and not got[:, c:].any()
    assert np.array_equal(np.where(neg0, 0, codes), np.where(neg0, got[:, :c] & 127, got[:, :c]))
    assert np.array_equal(exps, k.exps.cpu().numpy())
    for out in DT:
        r = R8.restore_rows(k, out)
        want = torch.from_numpy(values(codes, exps)).to(out)
        assert r.dtype == out and torch.equal(r.cpu().abs(), want.abs()) and torch.equal(r.cpu() < 0, want < 0)


def test_keep_special_values():
    """not finite, zeros of both signs, denormals, the border of the scale, ties, blocks far apart in one row, huge and tiny blocks"""
    inf, nan = float("inf"), float("nan")
    rows = [[nan, 1.0, inf, -inf, -0.0, 0.0, 1e-30, -1e-30], [0.0] * 8, [1e-45, -1e-45] + [0.0] * 6, [448.0, 449.0, 464.0, 432.0, 440.0, -456.0, 17.0, 18.0],
            [3.4028234663852886e38, 1.0, -1e38, 1e-45, 0.0, 0.0, 0.0, -1.0], [inf] * 8, [nan] * 8, [2.0 ** -120, 2.0 ** -110, 2.0 ** -101, 0, 0, 0, 0, 0],
            [448.0 * 2 ** -100, 2.0 ** -109, 2.0 ** -110, -2.0 ** -111, 0, 0, 0, 0], [1.75, 1.7500001, 1.0625, 1.1875, 0.0009765625, 0.0029296875, -0.001, 0]]
    x = torch.tensor(rows, device="cuda")
    wide = torch.cat([x, x * 0, x.flip(0), x, x.flip(1)], dim=1)      # 40 channels: blocks of 32 and of 8
    for t in (x, wide, x.to(torch.bfloat16), wide.to(torch.float16)):
        k = R8.checkpoint_rows(t)
        codes, exps = encode_ref(t)
        got = k.codes.cpu().numpy()[:, :t.shape[1]]
        z = (codes & 127) == 0
        assert np.array_equal(exps, k.exps.cpu().numpy())
        assert np.array_equal(np.where(z, 0, codes), np.where(z, got & 127, got))
        assert torch.equal((R8.restore_rows(k) > 0), (t > 0) & torch.isfinite(t))


@pytest.mark.parametrize("dtype", DT)
def test_keep_strided_and_unaligned(dtype):
    buf = make(40, 97, dtype, seed=3)
    for x in (buf[:, 1:96], buf[1::3, 5:38], buf[7:8, 3:], buf[:, 96:97]):
        a, b = R8.checkpoint_rows(x), R8.checkpoint_rows(x.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.exps, b.exps)


def test_relu_mask():
    y = make(77, 45, torch.float32, seed=5, relu=True)
    y[3] = 1e-38
    y[4, :] = 0
    k = R8.checkpoint_rows(y)
    dy = torch.randn(77, 52, device="cuda")[:, 2:47]
    assert torch.equal(R8.relu_mask8(dy, k), torch.where(y > 0, dy, torch.zeros_like(dy)))


def wgrad_case(m, n, k, dtype, seed, lead=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dy = (torch.randn(m, n + lead, generator=g, device="cuda") * torch.exp(2 * torch.randn(m, 1, generator=g, device="cuda"))).to(dtype)[:, lead:]
    x8 = R8.checkpoint_rows(make(m, k, torch.float32, seed=seed + 1, relu=True))
    return dy, x8


def wgrad_check(dy, x8, got):
    x = R8.restore_rows(x8).double()
    d = dy.double()
    m = max(1, dy.shape[0])
    want, size = torch.mm(d.t().contiguous(), x), torch.mm(d.abs().t().contiguous(), x.abs())
    tol = (8 + 2 * math.sqrt(m)) * U
    dw, db = got
    assert dw.dtype == torch.float32 and dw.shape == want.shape
    assert ((dw.double() - want).abs() <= tol * size + 1e-40).all()
    if db is not None:
        assert ((db.double() - d.sum(0)).abs() <= tol * d.abs().sum(0) + 1e-40).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 4, 4), (2, 64, 64), (31, 3, 5), (33, 65, 130), (257, 128, 128), (1000, 196, 131), (4099, 17, 300),
                                   (20000, 4, 7), (2500, 300, 33)])
def test_wgrad(m, n, k, dtype):
    dy, x8 = wgrad_case(m, n, k, dtype, m + n + k, lead=n % 3)
    got = R8.linear_wgrad8(dy, x8)
    wgrad_check(dy, x8, got)
    again = R8.linear_wgrad8(dy, x8, want_bias=False)
    assert torch.equal(again[0], got[0]) and again[1] is None


def test_wgrad_no_rows():
    dw, db = R8.linear_wgrad8(torch.empty(0, 12, device="cuda"), R8.checkpoint_rows(torch.empty(0, 20, device="cuda")))
    assert dw.shape == (12, 20) and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", DT)
def test_wgrad_values_that_are_not_finite(dtype):
    """an infinite or NaN gradient reaches its own rows of dw only; a NaN kept value its own column"""
    dy, x8 = wgrad_case(100, 70, 40, dtype, 9)
    clean = R8.linear_wgrad8(dy, x8)
    x = R8.restore_rows(x8)
    dy = dy.clone()
    dy[5, 3] = float("inf")
    dy[50, 66] = float("nan")
    dw, db = R8.linear_wgrad8(dy, x8)
    keep = [j for j in range(70) if j not in (3, 66)]
    assert torch.equal(dw[keep], clean[0][keep]) and torch.equal(db[keep], clean[1][keep])
    assert torch.isnan(dw[66]).all() and torch.isnan(db[66]) and torch.isinf(db[3])
    pos = x[5] > 0
    assert torch.isinf(dw[3][pos]).all() and torch.isnan(dw[3][~pos]).all()
    x[7, 11] = float("nan")
    dw = R8.linear_wgrad8(clean_dy := torch.nan_to_num(dy, 0.0, 0.0, 0.0), R8.checkpoint_rows(x))[0]
    ref = R8.linear_wgrad8(clean_dy, x8)[0]
    cols = [j for j in range(40) if j != 11]
    assert torch.isnan(dw[:, 11]).all() and torch.equal(dw[:, cols], ref[:, cols])


def test_wgrad_small_and_large_magnitudes():
    """blocks of very different scale in one row, gradients from 1e-30 to 1e30"""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(500, 96, generator=g, device="cuda") * torch.tensor([1e-20, 1.0, 1e12], device="cuda").repeat_interleave(32)
    dy = torch.randn(500, 40, generator=g, device="cuda") * torch.logspace(-30, 18, 40, device="cuda")
    x8 = R8.checkpoint_rows(x)
    wgrad_check(dy, x8, R8.linear_wgrad8(dy, x8))


def test_on_another_stream_and_in_a_graph():
    dy, x8 = wgrad_case(3000, 96, 80, torch.float32, 2)
    x = R8.restore_rows(x8)
    want = R8.linear_wgrad8(dy, x8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = R8.linear_wgrad8(dy, R8.checkpoint_rows(x))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k = R8.checkpoint_rows(x)
        out = R8.linear_wgrad8(dy, k)
        back = R8.restore_rows(k)
    for step in range(4):
        x.copy_(make(3000, 80, torch.float32, seed=20 + step))
        graph.replay()
        torch.cuda.synchronize()
        k2 = R8.checkpoint_rows(x)
        ref = R8.linear_wgrad8(dy, k2)
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1]) and torch.equal(back, R8.restore_rows(k2))


def test_refusals():
    x = torch.randn(6, 20, device="cuda")
    k = R8.checkpoint_rows(x)
    for bad, err in ((x.double(), TypeError), (x[None], TypeError), (x.t(), RuntimeError), (x[:1].expand(6, 20), RuntimeError), (x.cpu(), RuntimeError),
                     (x[:, :0], ValueError), (None, TypeError)):
        with pytest.raises(err):
            R8.checkpoint_rows(bad)
        with pytest.raises(err):
            R8.linear_wgrad8(bad, k)
    with pytest.raises(ValueError):
        R8.linear_wgrad8(x[:5], k)
    with pytest.raises(TypeError):
        R8.linear_wgrad8(x, x)
    with pytest.raises(TypeError):
        R8.restore_rows(k, torch.float64)
    with pytest.raises(ValueError):
        R8.relu_mask8(x[:, :19], k)
    with pytest.raises(TypeError):
        R8.relu_mask8(x.half(), k)
    with pytest.raises(ValueError):
        R8.Rows8(k.data, 6, 40)
    with pytest.raises(ValueError):
        R8.Rows8(k.data, 5, 20)
    with pytest.raises(TypeError):
        R8.Rows8(k.codes, 6, 20)
    with pytest.raises(ValueError):
        R8.Rows8.from_codes(k.codes[:, :20], k.exps[:5])
    with pytest.raises(TypeError):
        R8.Rows8.from_codes(k.codes.int(), k.exps)
    again = R8.Rows8.from_codes(k.codes[:, :20], k.exps)
    assert torch.equal(again.codes, k.codes) and torch.equal(again.exps, k.exps) and again.nbytes() == k.nbytes()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,c", [(1, 1), (3, 1), (9, 2), (40, 3), (5, 9), (2, 33)])
def test_keep_at_the_end_of_a_buffer(m, c, dtype):
    """rows that end where their storage ends, between guard values that must neither be used nor changed"""
    buf = torch.full((m * c + 64,), float("nan"), device="cuda", dtype=dtype)
    x = buf[32:32 + m * c].view(m, c)
    x.copy_(make(m, c, dtype, seed=m * c))
    k = R8.checkpoint_rows(x)
    codes, exps = encode_ref(x)
    assert np.array_equal(codes & 127, k.codes.cpu().numpy()[:, :c] & 127) and np.array_equal(exps, k.exps.cpu().numpy())
    assert torch.isnan(buf[:32]).all() and torch.isnan(buf[32 + m * c:]).all()


@pytest.mark.parametrize("m,c", [(1, 1), (3, 4), (50, 7), (33, 130), (5000, 64)])
def test_relu_mask_strides_and_in_place(m, c):
    y = make(m, c, torch.float32, seed=m, relu=True)
    k = R8.checkpoint_rows(y)
    wide = torch.randn(2 * m, 2 * c + 5, device="cuda")
    dy, out = wide[::2, 1:1 + c], wide[::2, 3 + c:3 + 2 * c]
    want, before = torch.where(y > 0, dy, torch.zeros_like(dy)), wide.clone()
    assert R8.relu_mask8(dy, k, out=out) is out and torch.equal(out, want)
    before[::2, 3 + c:3 + 2 * c] = want
    assert torch.equal(wide, before)                      # nothing beside it was written
    assert R8.relu_mask8(dy, k, out=dy) is dy and torch.equal(dy, want)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (5, 4, 16), (65, 66, 40), (200, 131, 130), (20000, 8, 8)])
def test_wgrad_at_the_end_of_a_buffer(m, n, k, dtype):
    """gradient rows between guard values that are NaN: rows behind the last one are read as zeros, whatever lies there"""
    dy, x8 = wgrad_case(m, n, k, dtype, 3)
    want = R8.linear_wgrad8(dy, x8)
    for lead in (64, 65):
        buf = torch.full((m * n + 128 + 64 * n,), float("nan"), device="cuda", dtype=dtype)
        inside = buf[lead:lead + m * n].view(m, n)
        inside.copy_(dy)
        got = R8.linear_wgrad8(inside, x8)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_outputs_over_inputs_are_refused():
    x = torch.randn(40, 24, device="cuda")
    with pytest.raises(RuntimeError):                     # other rows of dy
        R8.relu_mask8(x[:-1], R8.checkpoint_rows(x[1:]), out=x[1:])
    data = torch.empty(40 * 32 + 48 + 40 * 24 * 4, device="cuda", dtype=torch.uint8)
    over = R8.Rows8(data[:40 * 32 + 48], 40, 24)
    with pytest.raises(RuntimeError):                     # the kept rows
        R8.relu_mask8(x, over, out=data[16:16 + 40 * 24 * 4].view(torch.float32).view(40, 24))
    big = torch.randn(24, 24, device="cuda")
    with pytest.raises(RuntimeError):
        R8.linear_wgrad8(big, R8.checkpoint_rows(big), out=big)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", [(16400, 512, 512), (65600, 129, 256), (4200, 1000, 1030)])
def test_wgrad_of_large_products_from_unaligned_rows(m, n, k, dtype):
    """sizes that take the large tiles; rows behind an offset of one element (16-bit rows that are not 4-byte aligned)"""
    dy, x8 = wgrad_case(m, n, k, dtype, 5)
    want = R8.linear_wgrad8(dy, x8)
    wgrad_check(dy, x8, want)
    wide = torch.full((m, n + 3 - n % 2), float("nan"), device="cuda", dtype=dtype)
    wide[:, 1:1 + n] = dy
    got = R8.linear_wgrad8(wide[:, 1:1 + n], x8)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_keep_and_mask_of_many_rows():
    """more items than the element-wise kernels have threads"""
    y = make(70000, 129, torch.float32, seed=8, relu=True)
    k = R8.checkpoint_rows(y)
    codes, exps = encode_ref(y)
    assert np.array_equal(codes & 127, k.codes.cpu().numpy()[:, :129] & 127) and np.array_equal(exps, k.exps.cpu().numpy())
    assert torch.equal(R8.restore_rows(k).cpu(), torch.from_numpy(values(k.codes.cpu().numpy()[:, :129], exps)).float())
    dy = torch.randn(70000, 129, device="cuda")
    assert torch.equal(R8.relu_mask8(dy, k), torch.where(y > 0, dy, torch.zeros_like(dy)))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", [(1100, 2000, 2100), (300, 40, 50), (9000, 130, 70), (16400, 500, 520)])
def test_wgrad_into_columns(m, n, k, dtype):
    """large and small tiles, with one split of the rows and with many, into columns of a wider tensor"""
    dy, x8 = wgrad_case(m, n, k, dtype, 6)
    want = R8.linear_wgrad8(dy, x8)
    wgrad_check(dy, x8, want)
    wide = torch.full((n, k + 11), 7.0, device="cuda")
    out, db = R8.linear_wgrad8(dy, x8, out=wide, col0=5)
    assert out is wide and torch.equal(wide[:, 5:5 + k], want[0]) and torch.equal(db, want[1])
    assert (wide[:, :5] == 7).all() and (wide[:, 5 + k:] == 7).all()
