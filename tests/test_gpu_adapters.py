"""Low-rank adapters beside a shared projection (ops/adapters.py) against the formulas in 64 bits.

Tolerances, u = 2^-24, h = half a step of the rows' type relative to the value (torch.finfo(t).eps / 2):
  t            a sum of k products: (8 + 2 sqrt(k)) u sum |A||x|
  out, dx      h |out| for the one rounding, plus scale * sum over the rank of |B| times (the error of t, the part of t that the second
               product drops: 2^-16 |t| in bfloat16, 2^-20 max |t| in float16, nothing in float32) and (8 + 2 sqrt(rank)) u of the
               same sum for its additions
  da, db       h |.| plus (8 + 2 sqrt(rows)) u times the sum of the products' sizes, and the error of u for da"""
import math

import numpy as np
import pytest
import torch

from jmodt_amd.ops import adapters as AD
from jmodt_amd.ops import rows as R
from jmodt_amd.ops import rows8 as R8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = [torch.float32, torch.bfloat16, torch.float16]


def acc(n):
    return (8 + 2 * math.sqrt(max(1, n))) * U


def make(m, k, n, r, count, dtype, seed=0, none=0.2, frames=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=g, device="cuda")
    if frames:
        ids = (torch.arange(m, device="cuda") * 7 // max(1, m)) % (count + 1) - 1
    else:
        ids = torch.randint(0, count, (m,), generator=g, device="cuda")
        ids = torch.where(torch.rand(m, generator=g, device="cuda") < none, torch.full_like(ids, -1), ids)
    d = dict(x=rn(m, k), a=rn(count, r, k) / math.sqrt(k), b=rn(count, n, r) * 0.3, base=rn(m, n), dy=rn(m, n), dbase=rn(m, k))
    d = {key: v.to(dtype) for key, v in d.items()}
    d.update(ids=ids.to(torch.int32), scales=0.5 + torch.rand(count, generator=g, device="cuda"))
    return d


def member(d, i):
    return (d["ids"] == i).double()[:, None]


def low(x, w, scales, d, base, dtype, drop=True):
    """base + scales B (A x) with w = (A (count, r, k), B (count, n, r)): (t, tolerance of t, out, tolerance of out)"""
    a, b = w[0].double(), w[1].double()
    x, m = x.double(), x.shape[0]
    t = torch.zeros(m, a.shape[1], dtype=torch.float64, device=x.device)
    tt = torch.zeros_like(t)
    out = base.double().clone()
    tol = torch.zeros_like(out)
    part = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -20}[dtype]
    for i in range(a.shape[0]):
        s, on = scales[i].double(), member(d, i)
        ti = torch.mm(x * on, a[i].t().contiguous())
        te = acc(x.shape[1]) * torch.mm(x.abs() * on, a[i].abs().t().contiguous())
        t, tt = t + ti, tt + te
        size = ti.abs().amax(1, keepdim=True).expand_as(ti) if dtype == torch.float16 else ti.abs()
        bt = b[i].t().contiguous()
        out = out + s * torch.mm(ti, bt)
        tol = tol + s * torch.mm(te + part * size + acc(a.shape[1]) * ti.abs(), bt.abs())
    return t, tt + 1e-38, out, tol + torch.finfo(dtype).eps / 2 * out.abs() * 1.001 + (6e-8 if dtype == torch.float16 else 1e-38) + 2 * U * base.double().abs()


def check(got, want, tol):
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.2f} of the tolerance"


SHAPES = [(1, 1, 1, 1, 1), (1, 64, 64, 16, 3), (8, 512, 512, 16, 8), (15, 33, 70, 3, 2), (17, 130, 66, 17, 5), (100, 200, 31, 33, 7), (257, 96, 129, 64, 4),
          (300, 64, 100, 65, 3), (70, 40, 80, 128, 2), (1500, 131, 197, 9, 40), (5000, 32, 64, 16, 3), (9000, 20, 12, 8, 1023)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n,r,count", SHAPES)
def test_forward(m, k, n, r, count, dtype):
    d = make(m, k, n, r, count, dtype, seed=m + k)
    plan = AD.AdapterPlan(d["ids"], count)
    out, t = AD.adapter_forward(d["base"], d["x"], d["a"], d["b"], d["scales"], plan, want_t=True)
    if count <= 64:
        wt, tt, wo, to = low(d["x"], (d["a"], d["b"]), d["scales"], d, d["base"], dtype)
        check(t, wt, tt)
        check(out, wo, to)
    none = d["ids"] < 0
    assert torch.equal(out[none], d["base"][none]) and not t[none].any()
    assert torch.equal(out, AD.adapter_forward(d["base"], d["x"], d["a"], d["b"], d["scales"], plan))
    zero = AD.adapter_forward(None, d["x"], d["a"], d["b"], d["scales"], plan)
    assert torch.equal(zero, AD.adapter_forward(torch.zeros_like(d["base"]), d["x"], d["a"], d["b"], d["scales"], plan))
    buf = d["base"].clone()
    assert AD.adapter_forward(buf, d["x"], d["a"], d["b"], d["scales"], plan, out=buf) is buf and torch.equal(buf, out)


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n,r,count", SHAPES[:-1])
def test_grad(m, k, n, r, count, dtype, kept):
    d = make(m, k, n, r, count, dtype, seed=m + n, frames=m % 2 == 0)
    plan = AD.AdapterPlan(d["ids"], count)
    x = d["x"]
    t = low(x, (d["a"], d["b"]), d["scales"], d, d["base"], dtype)[0].float()
    if kept:
        x = R8.checkpoint_rows(x)
    xv = (R8.restore_rows(x) if kept else x).double()
    dx, da, db = AD.adapter_grad(d["dy"], x, t, d["a"], d["b"], d["scales"], plan, base=d["dbase"])
    wu, tu, wdx, tdx = low(d["dy"], (d["b"].transpose(1, 2), d["a"].transpose(1, 2)), d["scales"], d, d["dbase"], dtype)
    check(dx, wdx, tdx)
    h = torch.finfo(dtype).eps / 2 * 1.001
    floor = 6e-8 if dtype == torch.float16 else 1e-38
    for i in range(count):
        on, s = member(d, i), d["scales"][i].double()
        rows = int(on.sum().item())
        u, dy = wu * on, d["dy"].double() * on
        wa = s * torch.mm(u.t().contiguous(), xv)
        check(da[i], wa, h * wa.abs() + s * torch.mm((u.abs() * acc(rows) + tu * on).t().contiguous(), xv.abs()) + floor)
        wb = s * torch.mm(dy.t().contiguous(), t.double())
        check(db[i], wb, h * wb.abs() + s * acc(rows) * torch.mm(dy.abs().t().contiguous(), t.double().abs()) + floor)
        if rows == 0:
            assert not da[i].any() and not db[i].any()
    again = AD.adapter_grad(d["dy"], x, t, d["a"], d["b"], d["scales"], plan, base=d["dbase"])
    assert torch.equal(dx, again[0]) and torch.equal(da, again[1]) and torch.equal(db, again[2])
    buf = d["dbase"].clone()
    assert AD.adapter_grad(d["dy"], x, t, d["a"], d["b"], d["scales"], plan, base=buf, out=buf)[0] is buf and torch.equal(buf, dx)


@pytest.mark.parametrize("m,count,kind", [(0, 3, "mixed"), (1, 1, "mixed"), (63, 2, "mixed"), (1024, 5, "mixed"), (4096, 64, "mixed"), (4097, 64, "mixed"),
                                          (30000, 1023, "mixed"), (30000, 4, "runs"), (9000, 7, "none"), (9000, 7, "one"), (5000, 3, "range")])
def test_plan(m, count, kind):
    """order = the stable sort of the rows by adapter (rows without one last); tiles and chunks cover it once, one adapter each"""
    g = np.random.default_rng(m + count)
    ids = g.integers(-1, count, m)
    if kind == "runs":
        ids = np.arange(m) * 9 // max(m, 1) % count
    elif kind == "none":
        ids[:] = -1
    elif kind == "one":
        ids[:] = count - 1
    elif kind == "range":
        ids = g.choice([-2 ** 31, -5, 0, 1, 2, 3, 2 ** 31 - 1], m)
    plan = AD.AdapterPlan(torch.from_numpy(ids.astype(np.int32)).cuda(), count)
    p = plan.data.cpu().numpy()
    bucket = np.where((ids >= 0) & (ids < count), ids, count)
    order = p[4:4 + m]
    assert np.array_equal(order, np.argsort(bucket, kind="stable"))
    at = 4 + (m + 3) // 4 * 4
    pos, last = 0, -1
    for ad, start, n, _ in p[at:at + 4 * p[0]].reshape(-1, 4):
        key = count if ad < 0 else ad
        assert start == pos and n > 0 and key >= last and (bucket[order[start:start + n]] == key).all()
        pos, last = pos + n, key
    assert pos == m


@pytest.mark.parametrize("dtype", DT)
def test_strides_and_alignment(dtype):
    m, k, n, r = 150, 75, 90, 12
    d = make(m, k, n, r, 3, dtype, seed=4)
    plan = AD.AdapterPlan(d["ids"], 3)
    want, t = AD.adapter_forward(d["base"], d["x"], d["a"], d["b"], d["scales"], plan, want_t=True)
    wide = torch.full((2 * m, k + n + 9), 7.0, device="cuda", dtype=dtype)
    x, out = wide[::2, 3:3 + k], wide[::2, 5 + k:5 + k + n]
    x.copy_(d["x"])
    out.copy_(d["base"])
    keep = wide.clone()
    AD.adapter_forward(out, x, d["a"], d["b"], d["scales"], plan, out=out)
    assert torch.equal(out, want)
    keep[::2, 5 + k:5 + k + n] = want
    assert torch.equal(wide, keep)                        # nothing beside it was written
    odd = torch.empty(d["a"].numel() + 1, device="cuda", dtype=dtype)[1:].view_as(d["a"])
    odd.copy_(d["a"])
    assert torch.equal(AD.adapter_forward(d["base"], d["x"], odd, d["b"], d["scales"], plan), want)
    one = AD.adapter_grad(d["dy"], d["x"], t, d["a"], d["b"], d["scales"], plan)
    dys = torch.zeros(m, n + 5, device="cuda", dtype=dtype)[:, 2:2 + n]
    dys.copy_(d["dy"])
    for p, q in zip(AD.adapter_grad(dys, x, t, d["a"], d["b"], d["scales"], plan), one):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", DT)
def test_values_that_are_not_finite_stay_where_they_are(dtype):
    """a NaN row, an adapter of NaNs and an infinite row reach nobody else's rows; rows without an adapter keep base whatever x holds"""
    d = make(120, 50, 60, 10, 4, dtype, seed=6)
    d["ids"][:4] = torch.tensor([0, 1, -1, 2], dtype=torch.int32)
    plan = AD.AdapterPlan(d["ids"], 4)
    want = AD.adapter_forward(d["base"], d["x"], d["a"], d["b"], d["scales"], plan)
    d["x"][0] = float("nan")
    d["x"][2] = float("nan")
    d["x"][1] = float("inf")
    d["a"][3] = float("nan")
    d["b"][3] = float("inf")
    out, t = AD.adapter_forward(d["base"], d["x"], d["a"], d["b"], d["scales"], plan, want_t=True)
    ok = d["ids"] != 3
    ok[0] = ok[1] = False
    assert torch.equal(out[ok], want[ok]) and torch.isnan(out[0]).all() and not torch.isfinite(out[1]).any()
    assert torch.equal(out[2], d["base"][2]) and not t[2].any()
    t = torch.nan_to_num(t, 0.0, 0.0, 0.0)
    dx, da, db = AD.adapter_grad(d["dy"], d["x"], t, d["a"], d["b"], d["scales"], plan)
    assert torch.isfinite(da[2]).all() and torch.isfinite(db[:3]).all() and torch.isnan(da[0]).all()
    assert torch.isfinite(dx[d["ids"] != 3]).all() and not dx[d["ids"] < 0].any()


def test_float16_low_rank_values_beyond_its_range():
    """t larger than float16's largest value, with a B that brings it back, is no overflow"""
    x = torch.full((5, 256), 60.0, device="cuda", dtype=torch.float16)
    a = torch.full((1, 4, 256), 100.0, device="cuda", dtype=torch.float16)
    b = torch.full((1, 8, 4), 2.0 ** -14, device="cuda", dtype=torch.float16)
    plan = AD.AdapterPlan(torch.zeros(5, dtype=torch.int32, device="cuda"), 1)
    out = AD.adapter_forward(None, x, a, b, torch.ones(1, device="cuda"), plan)
    want = 60.0 * 100.0 * 256 * 4 * 2.0 ** -14
    assert (out.double() - want).abs().max() <= want * 2.0 ** -11


def test_graph_replays_with_new_rows_and_adapters():
    d = make(700, 64, 72, 16, 5, torch.float32, seed=8)
    ids = d["ids"].clone()

    def step():
        plan = AD.AdapterPlan(ids, 5)
        out, t = AD.adapter_forward(d["base"], d["x"], d["a"], d["b"], d["scales"], plan, want_t=True)
        return (out,) + AD.adapter_grad(d["dy"], R8.checkpoint_rows(d["x"]), t, d["a"], d["b"], d["scales"], plan)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        n = make(700, 64, 72, 16, 5, torch.float32, seed=30 + i, none=0.1 * i)
        for key in ("x", "dy", "a"):
            d[key].copy_(n[key])
        ids.copy_(n["ids"])
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, step()):
            assert torch.equal(p, q)


def layer_case(seed=0, m=300, k=64, n=48, r=8, count=3):
    d = make(m, k, n, r, count, torch.float32, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
    bias = torch.randn(n, generator=g, device="cuda")
    return d, w, bias, AD.AdapterPlan(d["ids"], count)


def formula(x, w, bias, a, b, scales, ids):
    y = x @ w.t() + bias
    for i in range(a.shape[0]):
        on = (ids == i).to(x.dtype)[:, None]
        y = y + scales[i] * ((x * on) @ a[i].t()) @ b[i].t()
    return y


@pytest.mark.parametrize("keep", ["float32", "e4m3"])
def test_layer_and_its_gradients(keep):
    """adapter_linear = projection + adapters; gradients against autograd of the formula in 64 bits (with e4m3: da and dw as the formula
    gives them for the kept x).  All sums are float32 over at most 300 rows: 1e-5 of a tensor's largest value is over 100 u."""
    d, w, bias, plan = layer_case()
    leaves = [v.clone().requires_grad_() for v in (d["x"], w, bias, d["a"], d["b"])]
    y = AD.adapter_linear(leaves[0], leaves[1], leaves[2], leaves[3], leaves[4], d["scales"], plan, keep=keep)
    y.backward(d["dy"])

    def grads(x):
        ref = [v.detach().double().cpu().requires_grad_() for v in (x, w, bias, d["a"], d["b"])]
        yr = formula(*ref, d["scales"].double().cpu(), d["ids"].cpu())
        return yr.detach(), torch.autograd.grad(yr, ref, d["dy"].double().cpu())
    yr, want = grads(d["x"])
    assert (y.detach().double().cpu() - yr).abs().max() <= 1e-5 * yr.abs().max()
    if keep == "e4m3":
        kept = grads(R8.restore_rows(R8.checkpoint_rows(d["x"])))[1]
        want = (want[0], kept[1], want[2], kept[3], want[4])
    for leaf, g in zip(leaves, want):
        assert (leaf.grad.double().cpu() - g).abs().max() <= 1e-5 * g.abs().max()


def test_layer_gradients_against_differences():
    """d(loss)/d(a, b) along random directions against central differences of the formula in 64 bits: the function is quadratic in (a, b)
    together, so a step of 1e-3 leaves no error but rounding"""
    d, w, bias, plan = layer_case(seed=5)
    a, b = d["a"].clone().requires_grad_(), d["b"].clone().requires_grad_()
    y = AD.adapter_linear(d["x"], w, bias, a, b, d["scales"], plan)
    y.backward(d["dy"])
    da, db = torch.randn_like(a).double().cpu(), torch.randn_like(b).double().cpu()
    args = [v.double().cpu() for v in (d["x"], w, bias)]
    sc, ids, dy = d["scales"].double().cpu(), d["ids"].cpu(), d["dy"].double().cpu()

    def loss(s):
        return (formula(*args, d["a"].double().cpu() + s * da, d["b"].double().cpu() + s * db, sc, ids) * dy).sum().item()
    num = (loss(1e-3) - loss(-1e-3)) / 2e-3
    ana = (a.grad.double().cpu() * da).sum().item() + (b.grad.double().cpu() * db).sum().item()
    size = (a.grad.double().cpu().abs() * da.abs()).sum().item() + (b.grad.double().cpu().abs() * db.abs()).sum().item()
    assert abs(num - ana) <= 1e-6 * size + 1e-6 * abs(num)


def test_two_layers_share_a_plan_and_only_the_adapters_train():
    """frozen projections, two layers, inputs kept in 8 bits: gradients for the adapters only, the same bits in a second run"""
    d, w, bias, plan = layer_case(seed=9, n=64)
    runs = []
    for _ in range(2):
        ps = [d["a"].clone().requires_grad_(), d["b"].clone().requires_grad_(), (d["a"] * 0.5).requires_grad_(), (d["b"] * 0.5).requires_grad_()]
        h = torch.relu(AD.adapter_linear(d["x"], w, bias, ps[0], ps[1], d["scales"], plan, keep="e4m3"))
        y = AD.adapter_linear(h, w, None, ps[2], ps[3], d["scales"], plan, keep="e4m3")
        runs.append(torch.autograd.grad(y.square().sum(), ps))
    for p, q in zip(*runs):
        assert torch.isfinite(p).all() and p.abs().max() > 0 and torch.equal(p, q)


def test_layer_rejects_gradients_it_does_not_make():
    d, w, bias, plan = layer_case()
    with pytest.raises(ValueError):
        AD.adapter_linear(d["x"], w, bias, d["a"], d["b"], d["scales"].requires_grad_(), plan)
    with pytest.raises(ValueError):
        AD.adapter_linear(d["x"], w, bias, d["a"], d["b"], d["scales"].detach(), plan, keep="int8")


def test_refusals():
    d = make(30, 24, 20, 4, 3, torch.float32)
    plan = AD.AdapterPlan(d["ids"], 3)
    ok = dict(base=d["base"], x=d["x"], a=d["a"], b=d["b"], scales=d["scales"], plan=plan)

    def bad(err, **kw):
        with pytest.raises(err):
            AD.adapter_forward(**{**ok, **kw})
    bad(TypeError, x=d["x"].half())
    bad(TypeError, x=d["x"].double())
    bad(RuntimeError, x=d["x"].cpu())
    bad(RuntimeError, x=d["x"].t().contiguous().t())
    bad(ValueError, x=d["x"][:, :20])
    bad(ValueError, x=d["x"][:29])
    bad(ValueError, b=d["b"][:, :, :3].contiguous())
    bad(RuntimeError, a=d["a"].transpose(1, 2))
    bad(ValueError, a=d["a"][:2].contiguous(), b=d["b"][:2].contiguous(), scales=d["scales"][:2].contiguous())
    bad(TypeError, scales=d["scales"].half())
    bad(TypeError, scales=d["scales"][:2])
    bad(TypeError, plan=None)
    bad(ValueError, base=d["base"][:, :19])
    bad(TypeError, base=d["base"].half())
    bad(ValueError, out=d["base"][:, :19])
    square = torch.randn(30, 24, device="cuda")
    with pytest.raises(RuntimeError):                     # out over x
        AD.adapter_forward(None, square, d["a"], torch.randn(3, 24, 4, device="cuda"), d["scales"], plan, out=square)
    shifted = torch.randn(31, 20, device="cuda")
    bad(RuntimeError, base=shifted[:30], out=shifted[1:])  # out over other rows of base
    with pytest.raises(ValueError):
        AD.adapter_forward(None, d["x"], torch.randn(3, 129, 24, device="cuda"), torch.randn(3, 20, 129, device="cuda"), d["scales"], plan)
    for n in (0, 1024):
        with pytest.raises(ValueError):
            AD.AdapterPlan(d["ids"], n)
    for ids in (d["ids"].long(), d["ids"][None], d["ids"].repeat(2)[::2]):
        with pytest.raises(TypeError):
            AD.AdapterPlan(ids, 3)
    with pytest.raises(RuntimeError):
        AD.AdapterPlan(d["ids"].cpu(), 3)
    t = torch.zeros(30, 4, device="cuda")
    good = dict(dy=d["dy"], x=d["x"], t=t, a=d["a"], b=d["b"], scales=d["scales"], plan=plan)
    for err, kw in ((TypeError, dict(t=t[:29])), (TypeError, dict(t=t.half())), (ValueError, dict(x=d["x"][:29])), (TypeError, dict(x=d["x"].half())),
                    (ValueError, dict(x=R8.checkpoint_rows(d["x"][:29]))), (ValueError, dict(dy=d["dy"][:, :19])), (RuntimeError, dict(out=d["x"]))):
        with pytest.raises(err):
            AD.adapter_grad(**{**good, **kw})


def test_beside_the_shared_projection_of_the_row_layers():
    """the way a served batch runs: ops.rows.linear_forward for all rows, the adapters added in place, frames without one untouched"""
    d, w, bias, plan = layer_case(seed=12)
    y = R.linear_forward(d["x"], w, bias)
    plain = y.clone()
    AD.adapter_forward(y, d["x"], d["a"], d["b"], d["scales"], plan, out=y)
    none = d["ids"] < 0
    assert none.any() and torch.equal(y[none], plain[none]) and not torch.equal(y, plain)


@pytest.mark.parametrize("m,count", [(16384, 5), (64 * 4096, 3), (64 * 4096 + 1, 1023), (300001, 2), (2 ** 20 + 4099, 7)])
def test_plan_of_many_rows(m, count):
    """the same for tiles of 32 rows and counting blocks of more rows; chunks too"""
    ids = np.random.default_rng(m).integers(-1, count, m)
    p = AD.AdapterPlan(torch.from_numpy(ids.astype(np.int32)).cuda(), count).data.cpu().numpy()
    bucket = np.where(ids >= 0, ids, count)
    order = p[4:4 + m]
    assert np.array_equal(order, np.argsort(bucket, kind="stable"))
    rows = np.bincount(bucket, minlength=count + 1)
    start = np.concatenate([[0], np.cumsum(rows)])

    def table(width, buckets):
        return np.array([(b if b < count else -1, start[b] + q, min(width, rows[b] - q)) for b in range(buckets) for q in range(0, rows[b], width)])
    at = 4 + (m + 3) // 4 * 4
    tiles, chunks = table(32, count + 1), table(512, count)
    assert p[0] == len(tiles) and p[1] == len(chunks)
    assert np.array_equal(p[at:at + 4 * p[0]].reshape(-1, 4)[:, :3], tiles)
    at += 4 * ((m + 31) // 32 + min(count + 1, m))
    assert np.array_equal(p[at:at + 4 * p[1]].reshape(-1, 4)[:, :3], chunks)
    at += 4 * ((m + 511) // 512 + min(count, m))
    assert np.array_equal(p[at:at + count + 1], np.concatenate([[0], np.cumsum((rows[:count] + 511) // 512)]))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kept", [False, True])
def test_no_rows(dtype, kept):
    d = make(0, 24, 20, 4, 3, dtype)
    plan = AD.AdapterPlan(d["ids"], 3)
    out, t = AD.adapter_forward(d["base"], d["x"], d["a"], d["b"], d["scales"], plan, want_t=True)
    assert out.shape == (0, 20) and t.shape == (0, 4)
    x = R8.checkpoint_rows(d["x"]) if kept else d["x"]
    dx, da, db = AD.adapter_grad(d["dy"], x, t, d["a"], d["b"], d["scales"], plan, base=d["dbase"])
    assert dx.shape == (0, 24) and not da.any() and not db.any()


def test_on_another_stream_and_two_graphs():
    """a side stream; two captured graphs of different sizes, replayed in turn"""
    runs = []
    for seed, m, r in ((1, 900, 16), (2, 200, 40)):
        d = make(m, 64, 72, r, 5, torch.bfloat16, seed=seed)

        def step(d=d):
            plan = AD.AdapterPlan(d["ids"], 5)
            out, t = AD.adapter_forward(d["base"], d["x"], d["a"], d["b"], d["scales"], plan, want_t=True)
            return (out,) + AD.adapter_grad(d["dy"], R8.checkpoint_rows(d["x"]), t, d["a"], d["b"], d["scales"], plan)
        want = step()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = step()
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        runs.append((graph, out, want, d))                # (a graph reads its inputs where they were: they live as long as it does)
    for _ in range(3):
        for _, out, _, _ in runs:
            for v in out:
                v.zero_()
        for graph, _, _, _ in runs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in runs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.parametrize("keep", ["float32", "e4m3"])
def test_layer_captured_forward_and_backward(keep):
    """both directions in one graph, its leaves first used there; new values on every replay"""
    d, w, bias, plan = layer_case(seed=21)
    x = d["x"]

    def step(ps):
        y = AD.adapter_linear(x, ps[0], ps[1], ps[2], ps[3], d["scales"], plan, keep=keep)
        return (y.detach(),) + torch.autograd.grad(y, ps, d["dy"])

    def leaves():
        return [v.detach().clone().requires_grad_() for v in (w, bias, d["a"], d["b"])]
    step(leaves())
    torch.cuda.synchronize()
    ps = leaves()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(ps)
    for i in range(4):
        n = layer_case(seed=40 + i)[0]
        x.copy_(n["x"])
        d["dy"].copy_(n["dy"])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, step(leaves())))


def test_layer_has_no_second_derivative():
    d, w, bias, plan = layer_case(seed=22)
    a = d["a"].clone().requires_grad_()
    y = AD.adapter_linear(d["x"], w, bias, a, d["b"], d["scales"], plan)
    g, = torch.autograd.grad(y.square().sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


MANY = [(16384, 40, 72, 5, 6), (16500, 72, 40, 24, 3), (16384, 33, 50, 50, 2), (17000, 31, 70, 100, 4), (6000, 130, 66, 16, 2), (8200, 40, 30, 33, 1), (16383, 20, 24, 8, 5)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n,r,count", MANY)
def test_forward_of_many_rows(m, k, n, r, count, dtype):
    """tiles of 32 rows and the largest ones of 16"""
    test_forward(m, k, n, r, count, dtype)


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,k,n,r,count", MANY)
def test_grad_of_many_rows(m, k, n, r, count, dtype, kept):
    """the weights transposed first and gathered, chunks of 256 and 512 rows"""
    test_grad(m, k, n, r, count, dtype, kept)


@pytest.mark.parametrize("keep", ["float32", "e4m3"])
def test_layer_of_one_row_and_of_none(keep):
    d, w, bias, plan = layer_case(seed=31, m=1, count=2)
    ps = [v.detach().clone().requires_grad_() for v in (d["x"], w, bias, d["a"], d["b"])]
    y = AD.adapter_linear(*ps, d["scales"], plan, keep=keep)
    want = formula(d["x"].double(), w.double(), bias.double(), d["a"].double(), d["b"].double(), d["scales"].double(), d["ids"])
    assert (y.double() - want).abs().max() <= 1e-5 * want.abs().max()
    assert torch.equal(torch.autograd.grad(y, ps, d["dy"])[2], d["dy"][0])
    none = AD.AdapterPlan(d["ids"][:0], 2)
    with pytest.raises(RuntimeError):                     # the dense layers take at least one row
        AD.adapter_linear(d["x"][:0], w, bias, d["a"], d["b"], d["scales"], none, keep=keep)
