"""keep="e4m3" beside float32 users of the same tensors: an 8-bit copy of a tensor that stays in float32 anyway is not made, chains share
a kept tensor, and the detector's graph holds less than with float32 — every block of it."""
import pytest
import torch

from jmodt_amd.ops import rows as R
from jmodt_amd.ops import rows8 as R8
from tests.test_gpu_rows8_chain import _engine

pytestmark = pytest.mark.gpu


def leaves(g, m=500, k1=32, k2=64, widths=(48, 16)):
    x1, x2 = torch.randn(m, k1, generator=g, device="cuda"), torch.randn(m, k2, generator=g, device="cuda")
    layers, k = [], k1 + k2
    for n in widths:
        layers.append([torch.randn(n, k, generator=g, device="cuda") / k ** 0.5, torch.randn(n, generator=g, device="cuda")])
        k = n
    ps = [x1, x2] + [t for layer in layers for t in layer]
    for p in ps:
        p.requires_grad_()
    return x1, x2, layers, ps, torch.randn(m, k, generator=g, device="cuda")


@pytest.mark.parametrize("acts", [(1, 1), (0, 1), (1, 0)])
@pytest.mark.parametrize("held", [(), ("x1",), ("x2",), ("y",), ("x1", "x2"), ("x1", "x2", "y")])
def test_gradients_with_held_tensors(held, acts):
    """the held operand's columns of dW are the float32 route's own, the others' those of the kept form; everything else is as it was.
    (float32 columns: the same kernel on the same operand; db comes with the first operand's kernel, within (8 + 2 sqrt(m)) 2^-24 of the sizes)"""
    x1, x2, layers, ps, dy = leaves(torch.Generator(device="cuda").manual_seed(1))
    f32 = torch.autograd.grad(R.rows_mlp(x1, layers, acts, x2=x2), ps, dy)
    e43 = torch.autograd.grad(R.rows_mlp(x1, layers, acts, x2=x2, keep="e4m3"), ps, dy)
    y = R.rows_mlp(x1, layers, acts, x2=x2, keep="e4m3", held=held)
    got = torch.autograd.grad(y, ps, dy)
    assert torch.equal(y, R.rows_mlp(x1, layers, acts, x2=x2))
    assert torch.equal(got[0], f32[0]) and torch.equal(got[1], f32[1])
    assert torch.equal(got[2][:, :32], (f32 if "x1" in held else e43)[2][:, :32])
    assert torch.equal(got[2][:, 32:], (f32 if "x2" in held else e43)[2][:, 32:])
    assert torch.equal(got[3], (f32 if "x1" in held else e43)[3])
    assert torch.equal(got[4], e43[4]) and torch.equal(got[5], e43[5])


def test_two_chains_share_a_kept_tensor(monkeypatch):
    g = torch.Generator(device="cuda").manual_seed(2)
    x1, x2, layers, ps, _ = leaves(g, widths=(64, 32))
    _, x4, more, ps2, dy = leaves(g, widths=(16,))
    packed = []
    pack = R8.checkpoint_rows
    monkeypatch.setattr(R8, "checkpoint_rows", lambda x: packed.append(x) or pack(x))

    def run(share):
        del packed[:]
        h, kept = R.rows_mlp(x1, layers, (1, 1), x2=x2, keep="e4m3", want_kept=True)
        y = R.rows_mlp(h, more, (1,), x2=x4, keep="e4m3", kept=kept if share else None)
        return len(packed), torch.autograd.grad(y, ps + ps2[1:], dy)
    (n1, one), (n2, two) = run(True), run(False)
    assert n1 == 6 and n2 == 7
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    h, kept = R.rows_mlp(x1, layers, (1, 0), x2=x2, keep="e4m3", want_kept=True)       # (no mask: nothing was kept of it)
    assert kept is None
    with torch.no_grad():
        assert R.rows_mlp(x1, layers, (1, 1), x2=x2, keep="e4m3", want_kept=True)[1] is None
    assert R.rows_mlp(x1, layers, (1, 1), x2=x2, want_kept=True)[1] is None
    for bad in (dict(held=("x3",)), dict(kept=x1), dict(kept=R8.checkpoint_rows(x2.detach()))):
        with pytest.raises(ValueError):
            R.rows_mlp(x1, layers, (1, 1), x2=x2, keep="e4m3", **bad)


def test_no_tensor_of_the_detector_is_kept_twice(monkeypatch):
    """the whole joint forward: nothing that the graph saves in float32 and nothing that it returns is packed, and nothing is packed twice"""
    from jmodt_amd.train_rows import joint_forward_rows
    eng, xyz, img, xy = _engine()
    packed, saved = [], []
    pack = R8.checkpoint_rows
    monkeypatch.setattr(R8, "checkpoint_rows", lambda x: packed.append(x) or pack(x))

    def save(t):
        saved.append(t)
        return t
    with torch.autograd.graph.saved_tensors_hooks(save, lambda t: t):
        out = joint_forward_rows(eng, xyz, img, xy, rois_per_frame=eng.cfg.rpn_post_nms_top_n, keep="e4m3")
    at = [x.data_ptr() for x in packed]                    # (all of them are alive: no address is another's)
    assert len(at) > 20 and len(set(at)) == len(at)
    others = {t.data_ptr() for t in saved if t.dtype == torch.float32} | {t.data_ptr() for t in out.values()}
    assert not others & set(at)


def held_bytes(fn):
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    keep_alive = fn()
    torch.cuda.synchronize()
    return torch.cuda.memory_allocated() - before, keep_alive


@pytest.mark.parametrize("last", [False, True])
def test_memory_of_an_attention_block(last):
    """the block itself, its result read by a node that keeps it in float32 (or not): the kept form saves the gated image features' (and the
    result's) float32 copy, and adds nothing else"""
    from jmodt_amd.train_rows import BnFold, _attention_rows
    eng = _engine()[0]
    mod = eng.rpn.backbone_net.Fusion_Conv[0]
    m, pc, ic, oc = 20000, mod.IA_Layer.fc2.weight.shape[1], mod.IA_Layer.fc1.weight.shape[1], mod.conv1.weight.shape[0]
    point, img = torch.randn(m, pc, device="cuda", requires_grad=True), torch.randn(m, ic, device="cuda", requires_grad=True)

    def run(keep):
        def fn():
            out = _attention_rows(BnFold(eng.rpn, keep=keep), mod, point, img, out_held=not last)
            return (out if last else out.square()).sum()              # (a sum keeps nothing, a square its input)
        return held_bytes(fn)[0]
    run("float32")
    full, kept = run("float32"), run("e4m3")
    wi = mod.IA_Layer.conv1[0].weight.shape[0]
    less = m * (4 * wi - (wi + 15) // 16 * 16 - (wi + 31) // 32)
    if last:
        less += m * (4 * oc - (oc + 15) // 16 * 16 - (oc + 31) // 32)
    assert full - kept >= less - 8192


def test_memory_of_the_detector():
    from jmodt_amd.train_rows import joint_forward_rows
    eng, xyz, img, xy = _engine()

    def run(keep):
        return held_bytes(lambda: joint_forward_rows(eng, xyz, img, xy, rois_per_frame=eng.cfg.rpn_post_nms_top_n, keep=keep))[0]
    run("float32"), run("e4m3")
    full, kept = run("float32"), run("e4m3")
    print("held by the graph: float32", full, "e4m3", kept)
    assert kept < full
