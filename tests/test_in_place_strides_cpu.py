"""The C entries that may work in place refuse the same address with two row strides (rows would be read after others were written there)."""
import pytest

from jmodt_amd import _lib as L
from tests.test_adapters_cpu import EINVAL, EWORKSPACE, PTR


def test_relu_mask():
    lib = L.load()
    assert lib.jm_rows8_relu_mask(2, 8, PTR, 8, PTR, 16, PTR, 9, None) == EINVAL and b"in place" in lib.jm_last_error()


def test_adapter_forward():
    lib = L.load()
    args = [2, 8, 4, 2, 3, 0, PTR, 8, PTR, PTR, PTR, PTR, PTR, 5, PTR, 4, None, None]
    assert lib.jm_adapter_forward(*args) == EINVAL and b"in place" in lib.jm_last_error()


@pytest.mark.parametrize("m,results,ldb,want", [(2, 7, 9, EINVAL), (2, 1, 9, EINVAL), (2, 6, 9, EWORKSPACE), (1, 7, 9, EWORKSPACE), (2, 7, 8, EWORKSPACE)])
def test_adapter_grad(m, results, ldb, want):
    """(what passes the check only lacks its workspace)"""
    assert L.load().jm_adapter_grad_select(results, m, 8, 4, 2, 3, 0, PTR, 4, PTR, 8, None, 0, None, 0, PTR, PTR, PTR, PTR, PTR, PTR, ldb, PTR, 8, PTR, PTR, None, 0, None) == want
