"""Dense-layer chains with their activations kept in 8 bits (ops.rows.rows_mlp(keep="e4m3")) and the training routes that take them.

The forward and the data gradients are the float32 route's; a weight gradient is the float64 product with the kept activations, to the
float32 sums' (8 + 2 sqrt(m)) u of the products' sizes plus what the chain's own data gradient is off (float32 products of up to 96
terms a layer: the same bound again, three layers deep)."""
import math

import numpy as np
import pytest
import torch

from jmodt_amd import synth
from jmodt_amd.ops import rows as R
from jmodt_amd.ops import rows8 as R8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def chain(m, k1, k2, widths, acts, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x1 = torch.randn(m, k1, generator=g, device="cuda").requires_grad_()
    x2 = torch.randn(m, k2, generator=g, device="cuda").requires_grad_() if k2 else None
    layers, k = [], k1 + k2
    for n in widths:
        layers.append((torch.randn(n, k, generator=g, device="cuda").div_(math.sqrt(k)).requires_grad_(),
                       torch.randn(n, generator=g, device="cuda").requires_grad_() if bias else None))
        k = n
    return x1, x2, layers, list(acts), torch.randn(m, widths[-1], generator=g, device="cuda")


def leaves(x1, x2, layers):
    return [x1] + ([x2] if x2 is not None else []) + [t for W, b in layers for t in (W, b) if t is not None]


@pytest.mark.parametrize("m,k1,k2,widths,acts,bias", [(300, 64, 0, (96, 32), (1, 0), True), (1, 4, 4, (4,), (1,), True), (1000, 32, 64, (48, 96, 64), (1, 1, 1), True),
                                                       (777, 20, 0, (36, 12, 8), (0, 1, 0), False), (50, 8, 0, (4,), (0,), True)])
def test_chain(m, k1, k2, widths, acts, bias):
    x1, x2, layers, acts, dy = chain(m, k1, k2, widths, acts, seed=m, bias=bias)
    ps = leaves(x1, x2, layers)
    y = R.rows_mlp(x1, layers, acts, x2=x2)
    want = torch.autograd.grad(y, ps, dy)
    y8 = R.rows_mlp(x1, layers, acts, x2=x2, keep="e4m3")
    got = torch.autograd.grad(y8, ps, dy)
    assert torch.equal(y8, y)
    # the formula in float64 on the kept activations, masks from the float32 values
    with torch.no_grad():
        acts_in, cur, cur2, ys = [], x1, x2, []
        for l, (W, b) in enumerate(layers):
            kept = R8.restore_rows(R8.checkpoint_rows(cur)).double()
            if cur2 is not None:
                kept = torch.cat([kept, R8.restore_rows(R8.checkpoint_rows(cur2)).double()], dim=1)
            acts_in.append(kept)
            cur, cur2 = R.linear_forward(cur, W, b, acts[l], x2=cur2), None
            ys.append(cur)
        d = dy.double()
        i = len(ps)
        tol = 4 * (8 + 2 * math.sqrt(max(m, 128))) * U
        for l in range(len(layers) - 1, -1, -1):
            W, b = layers[l]
            if acts[l] == 1:
                d = d * (ys[l] > 0)
            if b is not None:
                i -= 1
                assert ((got[i].double() - d.sum(0)).abs() <= tol * d.abs().sum(0) + 1e-30).all()
            i -= 1
            size = torch.mm(d.abs().t().contiguous(), acts_in[l].abs()) + d.abs().sum(0)[:, None] * acts_in[l].abs().amax()
            assert ((got[i].double() - torch.mm(d.t().contiguous(), acts_in[l])).abs() <= tol * size + 1e-30).all()
            d = torch.mm(d, W.double())
    n_in = 1 if x2 is None else 2
    for p, q in zip(got[:n_in], want[:n_in]):             # data gradients: the float32 route's own
        assert torch.equal(p, q)


def test_memory_of_a_chain():
    """what the backward holds: 1.03 bytes an activation (and the weights) instead of 4"""
    x1, _, layers, acts, dy = chain(40960, 128, 0, (128, 128, 128), (1, 1, 1))
    x1 = x1.detach()

    def held(keep):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = R.rows_mlp(x1, layers, acts, keep=keep)
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated() - before - y.numel() * y.element_size()
    full, kept = held("float32"), held("e4m3")
    per = 40960 * 128
    assert full >= 2 * per * 4 and kept <= 4 * per * (1 + 1 / 32) + (1 << 20)          # float32: two hidden (x1, y exist anyway); e4m3: all four


def test_refusals():
    x1, _, layers, acts, _ = chain(8, 8, 0, (4,), (1,))
    with pytest.raises(ValueError):
        R.rows_mlp(x1, layers, [2], keep="e4m3")
    with pytest.raises(ValueError):
        R.rows_mlp(x1, layers, acts, keep="int8")
    k = R8.checkpoint_rows(x1.detach())
    with pytest.raises(ValueError):
        R8.linear_wgrad8(torch.zeros(8, 4, device="cuda"), k, out=torch.zeros(4, 8, device="cuda"), col0=4)
    with pytest.raises(ValueError):
        R8.relu_mask8(torch.zeros(8, 8, device="cuda"), k, out=torch.zeros(8, 4, device="cuda"))
    from jmodt_amd import train_joint
    with pytest.raises(ValueError):
        train_joint.joint_step(_engine()[0], *_engine()[1:], None, torch.optim.SGD(_engine()[0].parameters(), lr=0.0), route="operators", keep="e4m3")


_cache = []


def _engine():
    if not _cache:
        from jmodt_amd.detector import DetectorConfig
        from tests.test_gpu_detector import make_engine
        eng = make_engine(seed=3, cfg=DetectorConfig.tiny()).to("cuda:0").eval()
        xyz, img, xy = synth.frames(2, 2048, 77, H=96, W=320, native=(94, 310))
        xy = np.random.default_rng(5).uniform(-0.98, 0.98, size=xy.shape).astype(np.float32)
        _cache.append([eng] + [torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0") for a in (xyz, img, xy)])
    return _cache[0]


def test_joint_forward_with_kept_activations():
    """the whole detector: same outputs, and every parameter's gradient as near to the float32 route's as the rounding of the kept
    activations allows — 2^-4 of each product, so 2^-4 of a tensor's norm where products do not cancel; 0.1 leaves room for a tenth of cancellation"""
    from jmodt_amd import train_joint
    from jmodt_amd.train_rows import joint_forward_rows
    eng, xyz, img, xy = _engine()
    K = eng.cfg.rpn_post_nms_top_n
    tids = torch.randint(0, 6, (2, K), generator=torch.Generator().manual_seed(4)).float().to("cuda:0")

    def run(keep):
        eng.zero_grad(set_to_none=True)
        out = joint_forward_rows(eng, xyz, img, xy, rois_per_frame=K, keep=keep)
        train_joint.thin_loss(eng, out, tids).backward()
        torch.cuda.synchronize()
        grads = {k: None if v.grad is None else v.grad.double() for k, v in eng.named_parameters()}
        eng.zero_grad(set_to_none=True)
        return {k: out[k].detach() for k in ("rpn_cls", "rpn_reg", "rcnn_cls", "rcnn_reg")}, grads
    (o32, g32), (o8, g8) = run("float32"), run("e4m3")
    for k in o32:
        assert (o8[k] - o32[k]).abs().max() <= 1e-4 * max(1.0, float(o32[k].abs().max())), k
    top = max(float(g.norm()) for g in g32.values() if g is not None)
    differ = 0
    for k, g in g32.items():
        assert (g is None) == (g8[k] is None), k
        if g is None or float(g.norm()) < 1e-5 * top:
            continue
        err = float((g8[k] - g).norm() / g.norm())
        assert err <= 0.1, (k, err)
        differ += err > 1e-4
    assert differ > 10                                    # (the kept layers do see their rounding)


def test_joint_step_with_kept_activations():
    from jmodt_amd import train_joint
    eng, xyz, img, xy = _engine()
    K = eng.cfg.rpn_post_nms_top_n
    tids = torch.randint(0, 6, (2, K), generator=torch.Generator().manual_seed(4)).float().to("cuda:0")
    opt = torch.optim.SGD([p for p in eng.parameters() if p.requires_grad], lr=0.0)
    a = train_joint.joint_step(eng, xyz, img, xy, tids, opt, rois_per_frame=K, route="rows")
    b = train_joint.joint_step(eng, xyz, img, xy, tids, opt, rois_per_frame=K, route="rows", keep="e4m3")
    assert torch.isfinite(b) and abs(float(a) - float(b)) <= 1e-4 * max(1.0, abs(float(a)))


def test_nothing_is_kept_without_a_backward():
    """under no_grad the same values, and nothing but the result stays allocated"""
    from jmodt_amd.ops import adapters as AD
    x1, x2, layers, acts, _ = chain(4000, 64, 0, (96, 32), (1, 0), seed=3)
    y = R.rows_mlp(x1, layers, acts, keep="e4m3").detach()
    ids = torch.arange(4000, device="cuda", dtype=torch.int32) % 3
    a, b = torch.randn(3, 8, 64, device="cuda"), torch.randn(3, 96, 8, device="cuda")
    plan, scales = AD.AdapterPlan(ids, 3), torch.ones(3, device="cuda")
    w, bias = layers[0]
    z = AD.adapter_linear(x1, w.detach(), bias.detach(), a, b, scales, plan, keep="e4m3").detach()
    with torch.no_grad():
        before = torch.cuda.memory_allocated()
        y2 = R.rows_mlp(x1, layers, acts, keep="e4m3")
        z2 = AD.adapter_linear(x1, w, bias, a, b, scales, plan, keep="e4m3")
        assert torch.cuda.memory_allocated() - before <= y.numel() * 4 + z.numel() * 4 + 2048
    assert torch.equal(y, y2) and torch.equal(z, z2) and not y2.requires_grad and not z2.requires_grad
