"""Adapters of which only some gradients are asked for: the others are not computed, and what only they need is not kept."""
import itertools

import pytest
import torch

from jmodt_amd.ops import adapters as AD
from jmodt_amd.ops import rows8 as R8
from tests.test_gpu_adapters import make

pytestmark = pytest.mark.gpu
M = 640


@pytest.mark.parametrize("keep", ["float32", "e4m3"])
def test_adapter_layer_with_frozen_parts(keep):
    """each of x, w, bias, a, b alone: the gradient of the run in which all train; x is kept only for w, a"""
    g = torch.Generator(device="cuda").manual_seed(2)
    shapes = dict(x=(M, 32), w=(48, 32), bias=(48,), a=(3, 8, 32), b=(3, 48, 8))
    base = {n: torch.randn(*sh, generator=g, device="cuda") * 0.3 for n, sh in shapes.items()}
    plan = AD.AdapterPlan(torch.randint(-1, 3, (M,), generator=g, device="cuda").to(torch.int32), 3)
    dy, scales = torch.randn(M, 48, generator=g, device="cuda"), torch.rand(3, generator=g, device="cuda")

    def run(train):
        d = {n: v.clone().requires_grad_(n in train) for n, v in base.items()}
        y = AD.adapter_linear(*d.values(), scales, plan, keep=keep)
        return dict(zip(train, torch.autograd.grad(y, [d[n] for n in train], dy)))
    every = run(list(shapes))
    for train in [[n] for n in shapes] + [["x", "w"], ["a", "b"], ["w", "bias"], ["bias", "b"], ["x", "a"]]:
        got = run(train)
        for n in train:
            if n == "bias" and "w" not in train:              # (summed on its own: another order)
                size = dy.abs().sum(0).max()
                assert (got[n] - every[n]).abs().max() <= 2 * (8 + 2 * M ** 0.5) * 2.0 ** -24 * size
            else:
                assert torch.equal(got[n], every[n]), (train, n)


@pytest.mark.parametrize("keep", ["float32", "e4m3"])
def test_nothing_is_held_where_nothing_trains(keep):
    d = make(M, 32, 48, 8, 2, torch.float32)
    plan, w = AD.AdapterPlan(d["ids"], 2), torch.randn(48, 32, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = AD.adapter_linear(d["x"], w, None, d["a"], d["b"], d["scales"], plan, keep=keep)
    assert torch.cuda.memory_allocated() - before <= y.numel() * 4 + 2048


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,r,count", [(1, 3, 5, 2, 2), (100, 40, 70, 16, 3), (512, 130, 66, 40, 4), (700, 64, 72, 17, 5), (17000, 40, 36, 70, 3), (0, 8, 12, 4, 2)])
def test_any_of_the_three_gradients(m, k, n, r, count, dtype, kept):
    """every choice of (dx, da, db): the bits of the call that makes all three, None in the other places; what is not needed may be missing"""
    d = make(m, k, n, r, count, dtype, seed=m)
    plan = AD.AdapterPlan(d["ids"], count)
    t = torch.randn(m, r, device="cuda")
    x = R8.checkpoint_rows(d["x"]) if kept else d["x"]
    args = (d["a"], d["b"], d["scales"], plan)
    every = AD.adapter_grad(d["dy"], x, t, *args, base=d["dbase"])
    for need in itertools.product((False, True), repeat=3):
        got = AD.adapter_grad(d["dy"], x if need[1] else None, t if need[2] else None, *args, base=d["dbase"] if need[0] else None, need=need)
        for on, p, q in zip(need, got, every):
            assert torch.equal(p, q) if on else p is None, need
        out = torch.empty_like(every[0])
        if need[0]:
            assert AD.adapter_grad(d["dy"], x, t, *args, base=d["dbase"], out=out, need=need)[0] is out and torch.equal(out, every[0])


def test_refusals():
    d = make(30, 24, 20, 4, 3, torch.float32)
    plan, t = AD.AdapterPlan(d["ids"], 3), torch.zeros(30, 4, device="cuda")
    good = dict(dy=d["dy"], x=d["x"], t=t, a=d["a"], b=d["b"], scales=d["scales"], plan=plan)
    for kw in (dict(x=None), dict(t=None), dict(x=None, need=(False, True, False)), dict(t=None, need=(False, False, True))):
        with pytest.raises(TypeError):
            AD.adapter_grad(**{**good, **kw})
    for kw in (dict(need=(True, True)), dict(need=(False, True, True), out=d["dbase"]), dict(need=(False, True, True), base=d["dbase"])):
        with pytest.raises(ValueError):
            AD.adapter_grad(**{**good, **kw})
