"""The ReLU's mask from a kept output where the output is infinite: the float32 route's mask is y > 0, so its gradient passes."""
import pytest
import torch

from jmodt_amd.ops import rows as R
from jmodt_amd.ops import rows8 as R8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,c", [(1, 1), (3, 8), (40, 45), (300, 130)])
def test_infinite_outputs_pass_their_gradient(m, c):
    g = torch.Generator(device="cuda").manual_seed(m)
    y = torch.randn(m, c, generator=g, device="cuda").clamp(min=0)
    y[torch.rand(m, c, generator=g, device="cuda") < 0.1] = float("inf")
    y[0, 0] = float("inf")
    dy = torch.randn(m, c, generator=g, device="cuda")
    assert torch.equal(R8.relu_mask8(dy, R8.checkpoint_rows(y)), torch.where(y > 0, dy, torch.zeros_like(dy)))


def test_chain_with_an_activation_that_overflows():
    """a hidden activation and an output beyond float32's range: masks and data gradients of both routes are the same"""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(64, 16, generator=g, device="cuda").abs()
    x[5] = 3e38
    layers = [(torch.rand(24, 16, generator=g, device="cuda") + 0.1, torch.zeros(24, device="cuda")), (torch.rand(8, 24, generator=g, device="cuda") + 0.1, None)]
    dy = torch.randn(64, 8, generator=g, device="cuda")
    grads = []
    for keep in ("float32", "e4m3"):
        leaf = x.clone().requires_grad_()
        y = R.rows_mlp(leaf, layers, [1, 1], keep=keep)
        assert torch.isinf(y[5]).all() and torch.isfinite(y[:5]).all()
        grads.append(torch.autograd.grad(y, leaf, dy)[0])
    assert torch.equal(grads[0], grads[1]) and grads[1][5].abs().max() > 0
