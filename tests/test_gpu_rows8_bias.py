"""The bias sums of linear_wgrad8: few additions one behind the other.

One 1 and many values just below half a step of 1: an addition of one of them to the sum is lost, and costs up to u = 2^-24 of it, so the error counts
the additions one behind the other.  512 rows, one split: 3 within eight rows, 2 steps a wave group, 7 + 2 over the 32 row groups: 14.  With the
rows added one by one it was 15 + 31."""
import pytest
import torch

from jmodt_amd.ops import rows8 as R8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("first", [0, 1, 7, 8, 130, 511])
def test_additions_one_behind_the_other(first):
    m, n, k = 512, 512, 512
    dy = torch.full((m, n), U * (1 - 2.0 ** -10), device="cuda")
    dy[first] = 1.0
    db = R8.linear_wgrad8(dy, R8.checkpoint_rows(torch.ones(m, k, device="cuda")))[1]
    want = dy.double().sum(0)
    assert ((db.double() - want).abs() <= 14 * U * want).all(), float((db.double() - want).abs().max() / U)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(8, 64, 64), (100, 70, 40), (512, 512, 512), (20000, 130, 256), (16400, 512, 512)])
def test_sums(m, n, k, dtype):
    """integers: every order of addition is exact"""
    g = torch.Generator(device="cuda").manual_seed(m)
    dy = torch.randint(-8, 9, (m, n), generator=g, device="cuda").to(dtype)
    x8 = R8.checkpoint_rows(torch.randint(0, 9, (m, k), generator=g, device="cuda").float())
    dw, db = R8.linear_wgrad8(dy, x8)
    assert torch.equal(db.double(), dy.double().sum(0))
    assert torch.equal(dw.double(), torch.mm(dy.double().t().contiguous(), R8.restore_rows(x8).double()))
