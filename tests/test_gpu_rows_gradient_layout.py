"""Incoming gradients in every layout that autograd may hand in: contiguous but off a 16-byte address, one row for all, transposed."""
import pytest
import torch

from jmodt_amd.ops import adapters as AD
from jmodt_amd.ops import rows as R

pytestmark = pytest.mark.gpu
M, K, N = 37, 16, 12


def layouts(g):
    """the same values, or one row of them for all rows"""
    dy = torch.randn(M, N, generator=g, device="cuda")
    off = torch.empty(M * N + 1, device="cuda")[1:].view(M, N)
    wide = torch.empty(M, N + 4, device="cuda")[:, 1:1 + N]
    for t in (off, wide):
        t.copy_(dy)
    return {"off": (off, dy), "wide": (wide, dy), "transposed": (dy.t().contiguous().t(), dy), "one row": (dy[:1].expand(M, N), dy[:1].repeat(M, 1)),
            "one column": (dy[:, :1].expand(M, N), dy[:, :1].repeat(1, N))}


@pytest.mark.parametrize("acts", [(1, 0), (0, 1)])
@pytest.mark.parametrize("keep", ["float32", "e4m3"])
@pytest.mark.parametrize("kind", ["off", "wide", "transposed", "one row", "one column"])
def test_chain(kind, keep, acts):
    g = torch.Generator(device="cuda").manual_seed(3)
    ps = [torch.randn(*s, generator=g, device="cuda").requires_grad_() for s in ((M, K), (20, K), (20,), (N, 20), (N,))]
    dy, same = layouts(g)[kind]
    y = R.rows_mlp(ps[0], [(ps[1], ps[2]), (ps[3], ps[4])], acts, keep=keep)
    got = torch.autograd.grad(y, ps, dy, retain_graph=True)
    for p, q in zip(got, torch.autograd.grad(y, ps, same)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("keep", ["float32", "e4m3"])
@pytest.mark.parametrize("kind", ["off", "wide", "transposed", "one row", "one column"])
def test_adapters(kind, keep):
    g = torch.Generator(device="cuda").manual_seed(4)
    ps = [torch.randn(*s, generator=g, device="cuda").requires_grad_() for s in ((M, K), (N, K), (N,), (3, 5, K), (3, N, 5))]
    plan = AD.AdapterPlan((torch.arange(M, device="cuda") % 4 - 1).to(torch.int32), 3)
    dy, same = layouts(g)[kind]
    y = AD.adapter_linear(*ps, torch.ones(3, device="cuda"), plan, keep=keep)
    got = torch.autograd.grad(y, ps, dy, retain_graph=True)
    for p, q in zip(got, torch.autograd.grad(y, ps, same)):
        assert torch.equal(p, q)
