"""Only what a gradient needs is kept and computed: frozen layers, frozen inputs, nothing that trains."""
import itertools

import pytest
import torch

from jmodt_amd.ops import rows as R
from jmodt_amd.ops import rows8 as R8

pytestmark = pytest.mark.gpu
M, WIDTHS = 640, (48, 32, 16)


def chain(train, acts, two=True, seed=0):
    """train: names of the leaves that require a gradient, of x1, x2, w0, b0, w1, ..."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    k1, k2 = 32, 64 if two else 0
    d = {"x1": torch.randn(M, k1, generator=g, device="cuda")}
    if two:
        d["x2"] = torch.randn(M, k2, generator=g, device="cuda")
    k = k1 + k2
    for l, n in enumerate(WIDTHS[:len(acts)]):
        d[f"w{l}"] = torch.randn(n, k, generator=g, device="cuda") / k ** 0.5
        d[f"b{l}"] = torch.randn(n, generator=g, device="cuda")
        k = n
    for name in train:
        d[name].requires_grad_()
    layers = [(d[f"w{l}"], d[f"b{l}"]) for l in range(len(acts))]
    return d, layers, torch.randn(M, k, generator=g, device="cuda")


def run(train, acts, two=True):
    d, layers, dy = chain(train, acts, two)
    y = R.rows_mlp(d["x1"], layers, acts, x2=d.get("x2"), keep="e4m3")
    return dict(zip(train, torch.autograd.grad(y, [d[n] for n in train], dy)))


def sizes(acts):
    """per layer the sum over the rows of |d(pre-activation)|, in float64"""
    d, layers, dy = chain([], acts)
    cur, cur2, ys = d["x1"], d["x2"], []
    for (W, b), act in zip(layers, acts):
        cur, cur2 = R.linear_forward(cur, W, b, act, x2=cur2), None
        ys.append(cur)
    g, out = dy.double(), [None] * len(acts)
    for l in range(len(acts) - 1, -1, -1):
        g = g * (ys[l] > 0) if acts[l] else g
        out[l] = g.abs().sum(0)
        g = torch.mm(g, layers[l][0].double())
    return out


@pytest.mark.parametrize("acts", [(1, 1, 1), (0, 1, 0), (1, 0, 1)])
def test_gradients_of_every_subset_of_layers(acts):
    """any subset of the weights, biases and inputs: the gradients of the run in which everything trains, bit for bit — but for the bias of a
    frozen weight, which is summed in another order: both sums are within (8 + 2 sqrt(m)) 2^-24 of the sum of the sizes"""
    names = ["x1", "x2"] + [f"{p}{l}" for l in range(3) for p in "wb"]
    every, size = run(names, acts), sizes(acts)
    for train in itertools.chain(([n] for n in names), (["w0", "b2"], ["w1", "b1"], ["x2", "w2"], ["b0", "b1"], ["w2", "b2"], ["x1", "x2"])):
        got = run(train, acts)
        for n in train:
            if n[0] == "b" and "w" + n[1] not in train:
                tol = 2.01 * (8 + 2 * M ** 0.5) * 2.0 ** -24 * size[int(n[1])]
                assert ((got[n] - every[n]).abs() <= tol).all(), (train, n)
            else:
                assert torch.equal(got[n], every[n]), (train, n)


def held(fn):
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = fn()
    torch.cuda.synchronize()
    return torch.cuda.memory_allocated() - before - y.numel() * y.element_size()


def test_what_is_kept(monkeypatch):
    """how many tensors each combination keeps"""
    packed = []
    pack = R8.checkpoint_rows
    monkeypatch.setattr(R8, "checkpoint_rows", lambda x: packed.append(tuple(x.shape)) or pack(x))
    for train, acts, want in ((["w0"], (1, 1, 1), 5), (["w2"], (1, 1, 1), 2), (["b2"], (1, 1, 1), 1), (["b2"], (1, 1, 0), 0), (["w2"], (1, 1, 0), 1), (["x1"], (1, 1, 1), 3),
                              (["x1"], (0, 0, 0), 0), (["x1"], (0, 1, 0), 1), (["w1"], (0, 1, 0), 2), (["w0"], (0, 0, 0), 2), (["b0", "w1"], (1, 1, 0), 2), ([], (1, 1, 1), 0)):
        d, layers, _ = chain(train, acts)
        del packed[:]
        R.rows_mlp(d["x1"], layers, acts, x2=d["x2"], keep="e4m3")
        assert len(packed) == want, (train, acts, packed)


def test_nothing_is_held_where_nothing_trains():
    """gradients enabled, but no leaf that requires one: the result is all that stays allocated"""
    d, layers, _ = chain([], (1, 1, 1))
    for keep in ("float32", "e4m3"):
        assert held(lambda: R.rows_mlp(d["x1"], layers, (1, 1, 1), x2=d["x2"], keep=keep)) <= 2048, keep
