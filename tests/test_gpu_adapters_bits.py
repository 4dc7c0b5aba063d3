"""The low-rank values keep float32's bits through the second product, also in bfloat16 and float16.

base is the rounded negative of the adapter's own part, so that the result is what that rounding left: its own rounding no longer hides the
product's.  Tolerance, u = 2^-24, with no term for bits of t that the product drops: half a step of the result; scale * sum over the rank of |B| times t's
own error (8 + 2 sqrt(k)) u sum |A||x| and (8 + 2 sqrt(rank)) u |t| for the product's additions; 2 u |base| for the last one.  In float16 the pieces of t
are cut relative to the row's largest value: 2^-23 of it."""
import pytest
import torch

from jmodt_amd.ops import adapters as AD
from tests.test_gpu_adapters import U, acc, check, make

pytestmark = pytest.mark.gpu


def parts(x, a, b, d, dtype):
    """(the adapter's part of the result, its tolerance) in float64"""
    x = x.double()
    part, tol = torch.zeros(x.shape[0], b.shape[1], dtype=torch.float64, device=x.device), 0.0
    for i in range(a.shape[0]):
        on, s, ai, bt = (d["ids"] == i).double()[:, None], d["scales"][i].double(), a[i].double(), b[i].double().t().contiguous()
        t = torch.mm(x * on, ai.t().contiguous())
        te = acc(x.shape[1]) * torch.mm(x.abs() * on, ai.abs().t().contiguous()) + acc(ai.shape[0]) * t.abs()
        if dtype == torch.float16:
            te = te + 2.0 ** -23 * t.abs().amax(1, keepdim=True)
        part, tol = part + s * torch.mm(t, bt), tol + s * torch.mm(te, bt.abs())
    return part, tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,r,count", [(1, 64, 64, 1, 1), (40, 33, 70, 7, 2), (300, 64, 100, 16, 3), (300, 64, 100, 17, 3), (200, 96, 129, 64, 4), (70, 40, 80, 128, 2),
                                           (16400, 40, 72, 16, 3), (16400, 40, 72, 40, 3), (16400, 24, 40, 128, 2)])
def test_what_cancellation_leaves(m, k, n, r, count, dtype):
    d = make(m, k, n, r, count, dtype, seed=m + r, none=0.0)
    plan, h = AD.AdapterPlan(d["ids"], count), torch.finfo(dtype).eps / 2 * 1.001
    floor = 6e-8 if dtype == torch.float16 else 1e-38
    part, tol = parts(d["x"], d["a"], d["b"], d, dtype)
    base = (-part).to(dtype)
    want = base.double() + part
    check(AD.adapter_forward(base, d["x"], d["a"], d["b"], d["scales"], plan), want, tol + h * want.abs() + 2 * U * base.double().abs() + floor)
    at, bt = d["b"].transpose(1, 2), d["a"].transpose(1, 2)
    part, tol = parts(d["dy"], at, bt, d, dtype)
    base = (-part).to(dtype)
    want = base.double() + part
    dx = AD.adapter_grad(d["dy"], None, None, d["a"], d["b"], d["scales"], plan, base=base, need=(True, False, False))[0]
    check(dx, want, tol + h * want.abs() + 2 * U * base.double().abs() + floor)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 40, 16400])
@pytest.mark.parametrize("r", [2, 16, 17, 40, 64, 100, 128])
def test_low_rank_values_that_cancel(r, m, dtype):
    """t = (1 + 2^-9 + 2^-19, 1 + 2^-9) in two places of the rank, taken with 1 and -1: what is left is 2^-19, and every step of it is exact
    in float32"""
    k, n = 40, 24
    p, q = r // 2, r - 1
    if p == q:
        p = 0
    x = torch.zeros(m, k, device="cuda")
    x[:, 3], x[:, 17], x[:, 38] = 1.0, 2.0 ** -9, 2.0 ** -19
    a, b = torch.zeros(2, r, k, device="cuda"), torch.zeros(2, n, r, device="cuda")
    a[:, p, [3, 17, 38]], a[:, q, [3, 17]] = 1.0, 1.0
    b[:, :, p], b[:, :, q] = 1.0, -1.0
    x, a, b = x.to(dtype), a.to(dtype), b.to(dtype)
    plan, one = AD.AdapterPlan((torch.arange(m, device="cuda") % 2).int(), 2), torch.ones(2, device="cuda")
    assert (AD.adapter_forward(None, x, a, b, one, plan).double() == 2.0 ** -19).all()
    dx = AD.adapter_grad(x, None, None, b.transpose(1, 2).contiguous(), a.transpose(1, 2).contiguous(), one, plan, need=(True, False, False))[0]
    assert dx.shape == (m, n) and (dx.double() == 2.0 ** -19).all()
