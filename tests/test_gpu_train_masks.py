"""Both training routes at the benchmarked widths against their OWN ReLU masks, in float64.

Two correct runs can differ by more than any fixed bound: a gradient depends on the forward through the signs of the pre-activations, and one
that lies within the routes' rounding of zero (1.4e-6 between them; the library convolutions of the image branch are not bit-reproducible)
falls on either side.  Of the 65536 pooled pre-activations of the last level's first scale on the kitti cloud one is -1.2e-7, and its sign alone
moves that layer's bias gradient by 1.15e-2 of its largest entry.  What holds whatever the signs are: the bias gradient of a level's last
layer is the sum over the groups of d(out) where the pooled output is positive.  Sums of G float32 values: (8 + 2 sqrt(G)) 2^-24 of the
sum of their sizes."""
import numpy as np
import pytest
import torch

from jmodt_amd import synth

pytestmark = pytest.mark.gpu
DEV, K = "cuda:0", 64


def T(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


@pytest.fixture(scope="module")
def engine():
    from jmodt_amd.detector import DetectorConfig
    from tests.test_gpu_detector import make_engine
    eng = make_engine(seed=5, cfg=DetectorConfig.survey()).to(DEV).eval()
    for p in eng.parameters():
        p.requires_grad_(True)
    return eng


class Levels:
    """a level's pooled output and the gradient that reaches it"""

    def __init__(self):
        self.seen = []

    def add(self, out):
        entry = [out.detach().clone(), None]
        self.seen.append(entry)
        out.register_hook(lambda g: entry.__setitem__(1, g.detach().clone()))


def check(eng, seen, what):
    grads = {k: v.grad.detach().clone() for k, v in eng.named_parameters() if v.grad is not None}
    eng.zero_grad(set_to_none=True)
    levels = eng.rpn.backbone_net.SA_modules
    assert len(seen) == len(levels)
    for lev, ((out, d), sa) in enumerate(zip(seen, levels)):
        c0 = 0
        for k in range(len(sa.mlps)):
            name = [n for n in grads if n.startswith(f"rpn.backbone_net.SA_modules.{lev}.mlps.{k}.") and n.endswith("bn.bn.bias")][-1]
            got = grads[name].double()
            part = d[:, c0:c0 + got.numel()].double() * (out[:, c0:c0 + got.numel()] > 0)
            tol = (8 + 2 * out.shape[0] ** 0.5) * 2.0 ** -24 * part.abs().sum(0)
            assert part.abs().sum() > 0
            assert ((got - part.sum(0)).abs() <= tol + 1e-30).all(), (what, name)
            c0 += got.numel()
        assert c0 == out.shape[1]


@pytest.mark.parametrize("kind", ["uniform", "kitti", "packed"])
def test_bias_gradients_follow_from_the_runs_own_masks(engine, kind, monkeypatch):
    from jmodt_amd import train_joint, train_rows
    eng = engine
    xyz_h, img_h, xy_h = synth.frames(2, 16384, 4321, kind=kind, H=96, W=320, native=(94, 310))
    xy_h = np.random.default_rng(5).uniform(-0.98, 0.98, size=xy_h.shape).astype(np.float32)
    xyz, img, xy = T(xyz_h), T(img_h), T(xy_h)
    g = torch.Generator(device=DEV).manual_seed(7)
    levels = Levels()
    plain = train_rows._sa_level_rows

    def level(*a, **kw):
        out = plain(*a, **kw)
        levels.add(out)
        return out
    monkeypatch.setattr(train_rows, "_sa_level_rows", level)
    out = train_rows.rpn_forward_rows(eng, xyz, img, xy, train_rows.BnFold(eng.rpn))
    d = [torch.randn(v.shape, generator=g, device=DEV) for v in (out["rpn_cls"], out["rpn_reg"])]
    torch.autograd.backward([out["rpn_cls"], out["rpn_reg"]], d)
    torch.cuda.synchronize()
    check(eng, levels.seen, "rows")
    del out
    levels = Levels()
    hooks = [m.register_forward_hook(lambda mod, a, o: levels.add(o[1])) for m in eng.rpn.backbone_net.SA_modules]
    feats = train_joint.backbone_forward(eng.rpn.backbone_net, xyz, img, xy)
    torch.autograd.backward([eng.rpn.rpn_cls_layer(feats).transpose(1, 2), eng.rpn.rpn_reg_layer(feats).transpose(1, 2)], d)
    torch.cuda.synchronize()
    for h in hooks:
        h.remove()
    check(eng, [[o.transpose(1, 2).reshape(-1, o.shape[1]), q.transpose(1, 2).reshape(-1, q.shape[1])] for o, q in levels.seen], "operators")
