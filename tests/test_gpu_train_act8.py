"""The training path that keeps its activations in 8 bits (MVSNet.train_act8, act8= of the layers), and the matching loss of FeatureNet."""
import math

import numpy as np
import pytest
import torch

from mvs_amd import ops, parallel, synth, train_ops
from mvs_amd.models import MVSNet, feature_matching_loss, matching_cells, mvsnet_loss

pytestmark = pytest.mark.gpu


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def same_up_to_atomics(a, b):
    """The weight-gradient kernels end in floating-point atomics: a sum of n float32 terms in another order."""
    return float((a - b).norm()) <= 1e-5 * float(b.norm())


@pytest.mark.parametrize("ci,co,transposed,stride", [(8, 16, False, 2), (16, 16, False, 1), (16, 8, True, 2), (8, 1, False, 1)])
def test_conv3d_act8_gradients_are_those_of_the_rounded_input(ci, co, transposed, stride):
    w0 = randn(*((ci, co) if transposed else (co, ci)), 3, 3, 3, seed=1) * 0.2
    x0 = randn(1, 8, 16, 24, ci, seed=2)
    rounded = ops.act8_dequantize(ops.act8_quantize(x0))
    res = []
    for x, act8 in ((x0, True), (x0, False), (rounded, False)):
        x, w = x.clone().requires_grad_(), w0.clone().requires_grad_()
        y = train_ops.conv3d_cl(x, w, transposed, stride, act8=act8)
        res.append((y.detach(), *torch.autograd.grad(y, (x, w), randn(*y.shape, seed=3))))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])      # the output and the input gradient do not change
    assert same_up_to_atomics(res[0][2], res[2][2])


@pytest.mark.parametrize("ci,co,k,stride", [(8, 8, 3, 1), (8, 16, 5, 2), (32, 32, 3, 1)])
def test_conv2d_act8_gradients_are_those_of_the_rounded_input(ci, co, k, stride):
    w0, x0 = randn(co, ci, k, k, seed=1) * 0.2, randn(2, 24, 40, ci, seed=2)
    rounded = ops.act8_dequantize(ops.act8_quantize(x0))
    res = []
    for x, act8 in ((x0, True), (x0, False), (rounded, False)):
        x, w = x.clone().requires_grad_(), w0.clone().requires_grad_()
        y = train_ops.conv2d_cl(x, w, stride, act8=act8)
        res.append((y.detach(), *torch.autograd.grad(y, (x, w), randn(*y.shape, seed=3))))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])
    assert same_up_to_atomics(res[0][2], res[2][2])


def _scene(H=128, W=160, V=3, D=16, B=1):
    rng = np.random.default_rng(5)
    h, w = H // 4, W // 4
    imgs = torch.from_numpy(synth.images(rng, B, V, H, W)).cuda()
    proj = torch.from_numpy(synth.proj_matrices(V, h, w)).cuda().expand(B, -1, -1, -1).contiguous()
    dvals = torch.from_numpy(synth.depth_values(D)).cuda().expand(B, -1).contiguous()
    gt = torch.from_numpy((synth.DTU_TARGET_Z + 20 * rng.standard_normal((B, h, w))).astype(np.float32)).cuda()
    return imgs, proj, dvals, gt


def _kept_and_grads(act8, batched=True):
    torch.manual_seed(3)
    model = MVSNet(refine=False).cuda().train()
    model.train_act8, model.train_feature_batched = act8, batched
    imgs, proj, dvals, gt = _scene()
    kept = {}
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.__setitem__(t.data_ptr(), t.numel() * t.element_size()) or t, lambda t: t):
        depth = model(imgs, proj, dvals)["depth"]
        loss = mvsnet_loss(depth, gt, torch.ones_like(gt))
    loss.backward()
    return sum(kept.values()), depth.detach(), {k: p.grad for k, p in model.named_parameters()}, dict(model.named_buffers())


@pytest.mark.parametrize("batched", [True, False])
def test_train_act8_step(batched):
    full, depth, grads, buffers = _kept_and_grads(False, batched)
    less, depth8, grads8, buffers8 = _kept_and_grads(True, batched)
    # the forward pass is the same; what it keeps is about a third (images, features and the cost volume stay float32)
    assert torch.equal(depth, depth8) and less < 0.45 * full, (less, full)
    for k in buffers:
        assert torch.equal(buffers[k], buffers8[k]), k
    # the gradients are those of activations off by at most 1 / 254 of their block's largest: a relative error of a per cent or so
    # per layer, eleven layers deep at most
    for k in grads:
        a, b = grads8[k].double().flatten(), grads[k].double().flatten()
        assert torch.isfinite(a).all()
        assert float((a - b).norm()) <= 0.2 * float(b.norm()) + 1e-6, (k, float((a - b).norm() / b.norm()))


def test_train_act8_step_as_graph_replays():
    torch.manual_seed(3)
    model = MVSNet(refine=False).cuda().train()
    model.train_act8 = True
    imgs, proj, dvals, gt = _scene()
    opt = torch.optim.SGD(model.parameters(), lr=1e-4)
    g = parallel.GraphedTrainStep(model.parameters(), opt, lambda: mvsnet_loss(model(imgs, proj, dvals)["depth"], gt, torch.ones_like(gt)), warmup=2)
    losses = [float(g.replay().detach()) for _ in range(4)]
    assert all(math.isfinite(v) for v in losses) and len(set(losses)) == 4


def test_matching_cells_of_a_plane():
    """Identical cameras: every cell falls on itself; without depth, behind the camera or masked: on none."""
    h, w = 12, 20
    proj = torch.from_numpy(synth.proj_matrices(2, h, w)).cuda()
    depth = torch.full((1, h, w), 600.0, device="cuda")
    depth[0, 0, 0], depth[0, 0, 1], depth[0, 0, 2] = 0.0, -5.0, float("nan")
    mask = torch.ones_like(depth)
    mask[0, 3] = 0
    cells = matching_cells(depth, proj[:, 0], proj[:, 0], mask)[0]
    want = torch.arange(h * w, device="cuda")
    want[:3] = -1
    want[3 * w:4 * w] = -1
    assert torch.equal(cells, want)
    # against the projection in 64 bits, away from a cell's edge
    depth = torch.full((1, h, w), 650.0, device="cuda")
    cells = matching_cells(depth, proj[:, 1], proj[:, 0])[0].cpu().numpy()
    P = proj[0].double().cpu().numpy()
    y, x = np.mgrid[0:h, 0:w].reshape(2, -1).astype(float)
    p = (P[1] @ np.linalg.inv(P[0])) @ np.stack([x * 650, y * 650, np.full_like(x, 650), np.ones_like(x)])
    u, v = p[0] / p[2], p[1] / p[2]
    clear = (np.abs(u - np.floor(u) - 0.5) > 1e-3) & (np.abs(v - np.floor(v) - 0.5) > 1e-3)
    ok = (np.rint(u) >= 0) & (np.rint(u) < w) & (np.rint(v) >= 0) & (np.rint(v) < h)
    want = np.where(ok, np.rint(v) * w + np.rint(u), -1).astype(int)
    assert ok.any() and np.array_equal(cells[clear], want[clear])


def test_feature_matching_loss_against_64_bits():
    B, C, h, w, P = 2, 32, 10, 14, 60
    ref, src = (randn(B, C, h, w, seed=s).requires_grad_() for s in (1, 2))
    gen = torch.Generator(device="cuda").manual_seed(3)
    ref_cells, src_cells = (torch.randint(-1, h * w, (B, P), generator=gen, device="cuda") for _ in range(2))
    ref_cells[:, ::4] = 7                       # several points in one cell
    loss = feature_matching_loss(ref, src, ref_cells, src_cells, temperature=0.5)
    grads = torch.autograd.grad(loss, (ref, src))
    rd, sd = ref.detach().double().requires_grad_(), src.detach().double().requires_grad_()
    total, count = 0.0, 0
    for b in range(B):
        a, k = rd[b].reshape(C, -1).t(), sd[b].reshape(C, -1).t()
        ok = (ref_cells[b] >= 0) & (src_cells[b] >= 0)
        total = total + torch.nn.functional.cross_entropy(a[ref_cells[b][ok]] @ k.t() / 0.5, src_cells[b][ok], reduction="sum")
        count += int(ok.sum())
    want = total / count
    wants = torch.autograd.grad(want, (rd, sd))
    # logits of up to 60: (C + 4) 2^-24 of the sum of their terms' magnitudes (about 120) moves a probability by 3e-4 at worst,
    # in the norm over 140 cells by far less
    assert abs(float(loss) - float(want)) <= 1e-4 * float(want)
    for g, r in zip(grads, wants):
        assert float((g.double() - r).norm()) <= 1e-4 * float(r.norm())


def test_model_matching_loss_trains_featurenet_only():
    imgs, proj, dvals, gt = _scene(B=2)
    res = []
    for act8 in (False, True):
        torch.manual_seed(3)
        model = MVSNet(refine=False).cuda().train()
        model.train_act8 = act8
        loss = model.matching_loss(imgs, proj, gt)
        loss.backward()
        res.append(float(loss))
        for k, p in model.named_parameters():
            assert (p.grad is not None) == k.startswith("feature."), k
            assert p.grad is None or (torch.isfinite(p.grad).all() and float(p.grad.abs().max()) > 0), k
    assert res[0] == res[1] and math.isfinite(res[0])
    with pytest.raises(ops.MvsHipError, match="matching_loss"):
        model.eval().matching_loss(imgs, proj, gt)


def test_matching_loss_refuses_another_grid_and_shows_cells_beyond_a_map():
    model = MVSNet(refine=False).cuda().train()
    imgs, proj, _, gt = _scene()
    mask = torch.ones_like(gt)
    before = model.feature.conv0.bn.running_mean.clone()
    with pytest.raises(ops.MvsHipError, match="depth"):
        model.matching_loss(imgs, proj, gt[:, :-1])
    with pytest.raises(ops.MvsHipError, match="mask"):
        model.matching_loss(imgs, proj, gt, mask[:, :, :-1])
    assert torch.equal(model.feature.conv0.bn.running_mean, before)
    fea = torch.randn(1, 32, 6, 7, device="cuda")
    cells = torch.arange(5, device="cuda").unsqueeze(0)
    assert math.isfinite(float(feature_matching_loss(fea, fea, cells, cells)))
    for r, c in ((42, 3), (3, 42)):
        ref, src = cells.clone(), cells.clone()
        ref[0, 2], src[0, 2] = r, c
        assert math.isnan(float(feature_matching_loss(fea, fea, ref, src)))
