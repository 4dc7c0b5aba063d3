"""linear_wgrad8 from 16-bit gradient rows of an odd number of columns in a wider tensor of an even row stride: the last group of four
columns starts at an odd column, 2 bytes off a word.  Tolerance as in test_gpu_rows8.py: (8 + 2 sqrt(m)) 2^-24 of the products' sizes."""
import pytest
import torch

from jmodt_amd.ops import rows8 as R8
from tests.test_gpu_rows8 import wgrad_case, wgrad_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 5, 4), (40, 7, 16), (300, 67, 40), (1000, 131, 64), (130, 65, 33), (4097, 129, 130), (16400, 257, 512), (9000, 503, 520)])
def test_odd_columns_in_rows_of_even_stride(m, n, k, dtype):
    dy, x8 = wgrad_case(m, n, k, dtype, m + n)
    want = R8.linear_wgrad8(dy, x8)
    wgrad_check(dy, x8, want)
    for lead, behind in ((0, 1), (2, 3), (4, 1)):
        wide = torch.full((m, lead + n + behind), float("nan"), device="cuda", dtype=dtype)
        part = wide[:, lead:lead + n]
        part.copy_(dy)
        assert part.stride(0) % 2 == 0 or m == 1
        got = R8.linear_wgrad8(part, x8)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (lead, behind)
