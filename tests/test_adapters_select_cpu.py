"""The C entry of single adapter gradients: what each choice of results needs, and refusals, without a GPU."""
import pytest

from jmodt_amd import _lib as L
from tests.test_adapters_cpu import EINVAL, EWORKSPACE, PTR

DX, DA, DB = 1, 2, 4


def call(results, **kw):
    a = dict(m=2, k=8, n=4, rank=2, adapters=3, type=0, dy=PTR, lddy=4, x=PTR, ldx=8, codes=None, ldc=0, exps=None, lde=0, t=PTR, a=PTR, b=PTR, scales=PTR, plan=PTR,
             base=None, ldb=0, dx=PTR, lddx=8, da=PTR, db=PTR, ws=None, ws_bytes=0)
    a.update(kw)
    return L.load().jm_adapter_grad_select(results, *a.values(), None)


@pytest.mark.parametrize("results", [-1, 8])
def test_other_results_are_refused(results):
    assert call(results) == EINVAL


@pytest.mark.parametrize("results", range(8))
@pytest.mark.parametrize("kw,belongs", [(dict(x=None), DA), (dict(ldx=7), DA), (dict(x=None, codes=PTR, ldc=8, exps=PTR, lde=16), DA), (dict(da=None), DA), (dict(t=None), DB),
                                        (dict(db=None), DB), (dict(dx=None), DX), (dict(lddx=7), DX), (dict(base=PTR, ldb=7), DX), (dict(dy=None), 7), (dict(a=None), 7),
                                        (dict(lddy=3), 7)])
def test_what_a_result_needs(results, kw, belongs):
    """an argument of a result that is not wanted is not looked at (the call then only lacks its workspace)"""
    needed = belongs == 7 or results & belongs
    assert call(results, **kw) == (EINVAL if needed else EWORKSPACE)
