"""Refusals of the fine-tuning operators that need no GPU: the C entries' argument checks and the Python checks of host tensors."""
import ctypes

import pytest
import torch

from jmodt_amd import _lib as L
from jmodt_amd.ops import adapters as AD
from jmodt_amd.ops import rows8 as R8

EINVAL, EWORKSPACE = 1, 3
BUF = ctypes.create_string_buffer(4096)
PTR = (ctypes.addressof(BUF) + 63) // 64 * 64


def test_host_tensors_are_refused():
    x = torch.randn(4, 8)
    with pytest.raises(RuntimeError):
        R8.checkpoint_rows(x)
    k = R8.Rows8.from_codes(torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))
    assert k.shape == (4, 8) and k.nbytes() == 80
    for call in (lambda: R8.restore_rows(k), lambda: R8.linear_wgrad8(x, k), lambda: R8.relu_mask8(x, k), lambda: AD.AdapterPlan(torch.zeros(4, dtype=torch.int32), 2)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("args", [dict(m=-1), dict(c=0), dict(type=3), dict(ldc=24), dict(ldc=0), dict(ldx=7), dict(x=None), dict(codes=None),
                                  dict(codes=PTR + 4), dict(exps=None), dict(lde=1), dict(lde=24)])
def test_pack_refuses(args):
    a = dict(m=2, c=8, type=0, x=PTR, ldx=8, codes=PTR, ldc=16, exps=PTR, lde=16)
    a.update(args)
    lib = L.load()
    assert lib.jm_rows8_pack(a["m"], a["c"], a["type"], a["x"], a["ldx"], a["codes"], a["ldc"], a["exps"], a["lde"], None) == EINVAL
    assert lib.jm_rows8_restore(a["m"], a["c"], a["type"], a["codes"], a["ldc"], a["exps"], a["lde"], a["x"], a["ldx"], None) == EINVAL
    assert b"rows8" in lib.jm_last_error()


@pytest.mark.parametrize("args,code", [(dict(m=-1), EINVAL), (dict(n=0), EINVAL), (dict(k=0), EINVAL), (dict(type=-1), EINVAL), (dict(dw=None), EINVAL),
                                       (dict(lddy=3), EINVAL), (dict(ldc=40), EINVAL), (dict(lddw=4), EINVAL), (dict(codes=PTR + 8), EINVAL), (dict(lde=8), EINVAL), (dict(lddy=1 << 23), EINVAL),
                                       (dict(m=100000, ws=None), EWORKSPACE), (dict(m=100000, ws_bytes=8), EWORKSPACE)])
def test_wgrad_refuses(args, code):
    a = dict(m=4, n=4, k=8, type=0, dy=PTR, lddy=4, codes=PTR, ldc=16, exps=PTR, lde=1 << 20, dw=PTR, lddw=8, db=PTR, ws=PTR, ws_bytes=0)
    a.update(args)
    assert L.load().jm_rows8_linear_wgrad(a["m"], a["n"], a["k"], a["type"], a["dy"], a["lddy"], a["codes"], a["ldc"], a["exps"], a["lde"], a["dw"], a["lddw"], a["db"],
                                          a["ws"], a["ws_bytes"], None) == code


@pytest.mark.parametrize("args", [dict(m=-1), dict(m=2 ** 31 - 1), dict(k=0), dict(k=2 ** 21), dict(n=0), dict(type=3), dict(rank=0), dict(rank=129), dict(adapters=0),
                                  dict(adapters=1024), dict(ldx=7), dict(ldo=3), dict(ldb=3), dict(x=None), dict(a=None), dict(b=None), dict(scales=None),
                                  dict(plan=None), dict(out=None)])
def test_adapter_forward_refuses(args):
    a = dict(m=2, k=8, n=4, rank=2, adapters=3, type=0, x=PTR, ldx=8, a=PTR, b=PTR, scales=PTR, plan=PTR, base=PTR, ldb=4, out=PTR, ldo=4, t=None)
    a.update(args)
    assert L.load().jm_adapter_forward(*[a[key] for key in ("m", "k", "n", "rank", "adapters", "type", "x", "ldx", "a", "b", "scales", "plan", "base", "ldb", "out",
                                                            "ldo", "t")], None) == EINVAL


@pytest.mark.parametrize("args,code", [(dict(rank=129), EINVAL), (dict(adapters=1024), EINVAL), (dict(lddy=3), EINVAL), (dict(lddx=7), EINVAL), (dict(ldx=7), EINVAL),
                                       (dict(x=None, codes=None), EINVAL), (dict(x=None, ldc=8), EINVAL), (dict(x=None, lde=1), EINVAL), (dict(t=None), EINVAL), (dict(da=None), EINVAL),
                                       (dict(ws=None), EWORKSPACE), (dict(ws_bytes=16), EWORKSPACE)])
def test_adapter_grad_refuses(args, code):
    a = dict(m=2, k=8, n=4, rank=2, adapters=3, type=0, dy=PTR, lddy=4, x=PTR, ldx=8, codes=PTR, ldc=16, exps=PTR, lde=16, t=PTR, a=PTR, b=PTR, scales=PTR, plan=PTR,
             base=PTR, ldb=8, dx=PTR, lddx=8, da=PTR, db=PTR, ws=PTR, ws_bytes=100)
    a.update(args)
    assert L.load().jm_adapter_grad(*a.values(), None) == code


def test_plan_and_workspace_sizes():
    lib = L.load()
    assert lib.jm_adapter_plan_elems(-1, 4) == 0 and lib.jm_adapter_plan_elems(10, 0) == 0 and lib.jm_adapter_plan_elems(10, 1024) == 0
    assert lib.jm_adapter_plan_elems(0, 1) > 0 and lib.jm_adapter_plan_elems(100000, 8) > 100000
    assert lib.jm_adapter_plan(4, 2000, PTR, PTR, None) == EINVAL and lib.jm_adapter_plan(4, 2, None, PTR, None) == EINVAL
    assert lib.jm_adapter_plan(4, 2, PTR, PTR + 4, None) == EINVAL
    assert lib.jm_adapter_grad_workspace_bytes(10, 8, 4, 200, 3, 0) == 0
    big = lib.jm_adapter_grad_workspace_bytes(1 << 28, 1024, 1024, 128, 1023, 0)
    assert big > (1 << 28) * 128 * 4                      # (beyond 32 bits)


@pytest.mark.parametrize("args", [dict(m=-1), dict(c=0), dict(ldd=7), dict(ldo=7), dict(ldc=24), dict(ldc=0), dict(dy=None), dict(codes=None), dict(codes=PTR + 8),
                                  dict(out=None), dict(m=2 ** 31 - 1), dict(c=2 ** 23, ldc=2 ** 23, ldd=2 ** 23, ldo=2 ** 23)])
def test_relu_mask_refuses(args):
    a = dict(m=2, c=8, dy=PTR, ldd=8, codes=PTR, ldc=16, out=PTR, ldo=8)
    a.update(args)
    assert L.load().jm_rows8_relu_mask(*a.values(), None) == EINVAL


def test_sizes_beyond_the_counters_are_refused():
    lib = L.load()
    many, wide = 2 ** 30 + 16, 2 ** 22 + 32
    for m, c in ((many, 8), (2, wide)):
        lde, ldc = (m + 15) // 16 * 16, (c + 15) // 16 * 16
        assert lib.jm_rows8_pack(m, c, 0, PTR, c, PTR, ldc, PTR, lde, None) == EINVAL
        assert lib.jm_rows8_restore(m, c, 0, PTR, ldc, PTR, lde, PTR, c, None) == EINVAL
        assert lib.jm_rows8_linear_wgrad(m, c, 8, 0, PTR, c, PTR, 16, PTR, lde, PTR, 8, None, PTR, 1 << 40, None) == EINVAL
        assert lib.jm_rows8_wgrad_workspace_bytes(m, c, 8) == 0
        with pytest.raises(ValueError):
            R8.Rows8(torch.empty(16, dtype=torch.uint8), m, c)
    assert lib.jm_rows8_linear_wgrad(2, 8, wide, 0, PTR, 8, PTR, wide, PTR, 16, PTR, wide, None, PTR, 1 << 40, None) == EINVAL
    assert lib.jm_adapter_plan(2 ** 28 + 1, 2, PTR, PTR, None) == EINVAL and lib.jm_adapter_plan_elems(2 ** 28 + 1, 2) == 0
