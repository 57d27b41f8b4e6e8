"""Corners of the training operators that keep no large tensor, on the GPU."""
import math

import numpy as np
import pytest
import torch

from mvs_amd import ops, synth
from mvs_amd.models import MVSNet, feature_matching_loss
from product_pieces import LOW_PIECES, PAIRS, SCALE, gradient_bound, gradient_case, gradient_errors, logit_case

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("upstream", [float("inf"), float("nan"), 0.0])
@pytest.mark.parametrize("n,C", [(1, 40), (20, 40), (300, 40), (1, 200), (3, 200), (20, 200), (300, 200), (700, 136)])
def test_linear_cross_entropy_without_a_kept_row_has_no_gradient(n, C, upstream, dtype):
    """... whatever comes from above: a loss divided by the number of rows kept hands down 1 / 0."""
    x, w = randn(n, C, seed=1).to(dtype).requires_grad_(), randn(150, C, seed=2).to(dtype).requires_grad_()
    t = torch.full((n,), -100, device="cuda")
    for reduction in ("sum", "mean", "none"):
        loss = ops.linear_cross_entropy(x, w, t, reduction=reduction)
        gx, gw = torch.autograd.grad(loss, (x, w), torch.full_like(loss, upstream))
        assert (gx == 0).all() and (gw == 0).all(), reduction
        assert math.isnan(float(loss.detach())) if reduction == "mean" else (loss == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("C", [40, 200, 1024, 2056])
def test_linear_cross_entropy_of_a_single_ignored_row_whatever_the_table_holds(C, bad, dtype):
    x, w = randn(1, C, seed=1).to(dtype), randn(150, C, seed=2).to(dtype)
    w[7], w[149, 3] = bad, bad
    x, w = x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, torch.tensor([-100], device="cuda"), reduction="sum")
    gx, gw = torch.autograd.grad(loss, (x, w))
    assert float(loss.detach()) == 0 and (gx == 0).all() and (gw == 0).all()


def _scene(V=3, seed=5, H=128, W=160):
    rng = np.random.default_rng(seed)
    imgs = torch.from_numpy(synth.images(rng, 1, V, H, W)).cuda()
    proj = torch.from_numpy(synth.proj_matrices(V, H // 4, W // 4)).cuda().expand(1, -1, -1, -1).contiguous()
    gt = torch.from_numpy((synth.DTU_TARGET_Z + 20 * rng.standard_normal((1, H // 4, W // 4))).astype(np.float32)).cuda()
    return imgs, proj, gt


def _matching_step(imgs, proj, gt, mask=None):
    torch.manual_seed(3)
    model = MVSNet(refine=False).cuda().train()
    loss = model.matching_loss(imgs, proj, gt, mask)
    loss.backward()
    return float(loss.detach()), {k: p.grad for k, p in model.feature.named_parameters()}


@pytest.mark.parametrize("without", [1, 2])
def test_matching_loss_leaves_out_a_view_without_a_pair(without):
    """Every point behind that view's camera: the loss and the gradients are those of the other views."""
    imgs, proj, gt = _scene()
    proj[:, without, 2] *= -1
    loss, grads = _matching_step(imgs, proj, gt)
    rest = [v for v in range(3) if v != without]
    want, wants = _matching_step(imgs[:, rest].contiguous(), proj[:, rest].contiguous(), gt)
    # FeatureNet normalises each view by itself; its statistics may be rounded another way in a batch of three: logits of a few hundred
    # move by their last bits, 1e-4 at most, and a probability by that part of it
    assert math.isfinite(loss) and abs(loss - want) <= 1e-4 * want
    for k in grads:
        assert torch.isfinite(grads[k]).all() and float((grads[k] - wants[k]).norm()) <= 1e-3 * float(wants[k].norm()) + 1e-12, k


def test_matching_loss_without_any_pair_is_zero():
    imgs, proj, gt = _scene()
    loss, grads = _matching_step(imgs, proj, gt, torch.zeros_like(gt))
    assert loss == 0
    for k in grads:
        assert (grads[k] == 0).all(), k
    # ... and the loss of a single pair of maps is 0 / 0, with gradients of zero
    a, b = randn(1, 32, 8, 9, seed=1).requires_grad_(), randn(1, 32, 8, 9, seed=2).requires_grad_()
    none = torch.full((1, 5), -1, device="cuda")
    loss = feature_matching_loss(a, b, none, none)
    assert math.isnan(float(loss.detach()))
    for g in torch.autograd.grad(loss, (a, b)):
        assert (g == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [2, 4])
def test_linear_cross_entropy_few_16_bit_rows_in_pieces(n, dtype):
    """The rows that the one-pass kernel takes, against a table of more than 2^26 / n rows: a second piece, a short one, whose sums are
    added to the first's."""
    V, C = (1 << 26) // n + 777, 136
    w = torch.empty(V, C, device="cuda", dtype=dtype)
    spans = [slice(v, min(v + (1 << 22), V)) for v in range(0, V, 1 << 22)]
    for s in spans:
        w[s] = randn(s.stop - s.start, C, seed=s.start) * 0.1
    t = torch.tensor([V - 1, (1 << 26) // n, 5, -100], device="cuda")[-n:]      # (n = 2: one row, of the second piece, and an ignored one)
    t[0] = V - 1
    x = (randn(n, C, seed=2) + 8 * w[t.clamp(min=0)].float()).to(dtype)
    x[t < 0] = float("nan")
    leaves = [x.requires_grad_(), w.requires_grad_()]
    loss = ops.linear_cross_entropy(*leaves, t, reduction="sum")
    gx, gw = torch.autograd.grad(loss, leaves)
    keep = t >= 0
    k, xd = int(keep.sum()), x.detach()[keep].double()
    logits = torch.cat([xd @ w.detach()[s].double().t() for s in spans], 1)
    lse = torch.logsumexp(logits, 1)
    # A logit is off by `most` = (C + 4) u |x| |w|; a row's sum of exponentials by twice that part of it and one rounding for each of the
    # terms that are added one after the other (a tile's, and every sixteenth tile); a probability by `rel` in all.  dl is rounded to
    # the type (h; float16 carries it times 2^14: down to 2^-39), and so is each result.
    u = 2.0 ** -24
    most = (C + 4) * u * float(xd.abs().sum(1).max()) * float(w.detach().abs().max())
    rel = math.expm1(2 * most) + (V / 128 / 16 + 300) * u
    assert abs(float(loss.detach()) - float((lse - logits.gather(1, t[keep].unsqueeze(1)).squeeze(1)).sum())) <= k * (rel + 2 * u * float(lse.max()))
    h, least = torch.finfo(dtype).eps / 2, 2.0 ** -39 if dtype == torch.float16 else 0.0
    p = torch.exp(logits - lse.unsqueeze(1))
    p[torch.arange(k, device="cuda"), t[keep]] -= 1
    want = sum(p[:, s] @ w.detach()[s].double() for s in spans)
    off = sum((p[:, s].abs() * (h + rel) + least) @ w.detach()[s].double().abs() for s in spans)
    assert ((gx[keep].double() - want).abs() <= off + h * (want.abs() + off)).all() and (gx[~keep] == 0).all()
    smallest = torch.finfo(dtype).smallest_normal
    for s in (slice(0, 100), slice((1 << 26) // n // 256 * 256 - 300, V)):
        want = p[:, s].t() @ xd
        off = (p[:, s].abs() * (h + rel) + least).t() @ xd.abs()
        assert ((gw[s].double() - want).abs() <= off + h * (want.abs() + off) + smallest).all()


@pytest.mark.parametrize("route", ["f16", "f32 weight gradient", "bf16"])
def test_variance_conv0_act8_gradients_are_those_of_the_rounded_volume(route, monkeypatch):
    """The variance volume held in 8 bits: conv0's weight gradient is that of the volume read back, nothing else changes."""
    if route != "f16":
        monkeypatch.setenv("MVS_WGRAD_F16" if route == "f32 weight gradient" else "MVS_CONV0_F16", "0")
    V, h, w, D = 3, 32, 40, 16
    f0, w0 = randn(V, 1, 2, h, w, 16, seed=3) * 0.5, randn(8, 32, 3, 3, 3, seed=4) / 30
    rts = ops.rot_trans_all(torch.from_numpy(synth.proj_matrices(V, h, w)).cuda(), "device")
    dv = torch.from_numpy(synth.depth_values(D, interval=synth.sweep_interval(D))).cuda()
    go = randn(1, D, h, w, 8, seed=5)
    res = []
    for act8 in (True, False):
        f, k = f0.clone().requires_grad_(), w0.clone().requires_grad_()
        y = ops.variance_conv0_autograd(f[0], f[1:], rts, dv, k, act8=act8)
        res.append((y.detach(), *torch.autograd.grad(y, (f, k), go)))
    (y8, gf8, gw8), (y, gf, gw) = res
    # (the variance's backward pass ends in floating-point atomics: a sum of float32 terms in another order)
    assert torch.equal(y8, y) and float((gf8 - gf).norm()) <= 1e-5 * float(gf.norm())
    with torch.no_grad():
        var = ops.costvol_variance_c16(f0[0].contiguous(), f0[1:].contiguous(), rts, dv, False, out_c8=True,
                                       absmax_out=ops.absmax_block(f0.device) if route != "bf16" else None)
        back = ops.act8_dequantize(ops.act8_quantize(var))
    blocks = torch.nn.functional.pad(var.reshape(-1), (0, -var.numel() % 32)).view(-1, 32)
    off = torch.nn.functional.pad((back - var).reshape(-1), (0, -var.numel() % 32)).view(-1, 32)
    assert (off.abs() <= blocks.abs().amax(1, keepdim=True) / 127).all()      # half a step of its block's scale

    def weight_gradient(volume):      # [B, D, H, C / 8, W, 8], in 64 bits on the CPU
        x = volume.double().cpu().permute(0, 3, 5, 1, 2, 4).reshape(1, 32, D, h, w)
        return torch.nn.grad.conv3d_weight(x, (8, 32, 3, 3, 3), go.double().cpu().permute(0, 4, 1, 2, 3), padding=1)
    rounded, full = weight_gradient(back), weight_gradient(var)
    # two-piece and float32 products of D h w terms: below 1e-5 of the norm, where the volume's rounding moves it by far more
    for got, want in ((gw8, rounded), (gw, full)):
        assert float((got.double().cpu() - want).norm()) <= 1e-5 * float(want.norm())
    assert float((rounded - full).norm()) > 1e-4 * float(full.norm())


# (the last three: 256 x 256 tiles in the logits', in dW's and in dx's product)
@pytest.mark.parametrize("n,V,C", LOW_PIECES + [(200, 119, 130), (5000, 12004, 130), (600, 48016, 768), (9001, 811, 1000)])
def test_linear_cross_entropy_float32_logits_of_the_low_pieces(n, V, C):
    """tests/test_training_corners.py: any of the low pieces' products left out moves a logit by more than 1."""
    for which in PAIRS[:3]:
        x, w, logits = (t.cuda() for t in logit_case(which, n, V, C))
        t = torch.arange(n, device="cuda") * 7 % V
        loss = ops.linear_cross_entropy(x, w, t, scale=SCALE, reduction="none")
        logits = SCALE * logits[0].double()
        want = torch.logsumexp(logits, 0) - logits[t]
        # exact products; a logit of at most 9, rounded once or twice, and the sum of V exponentials
        assert float((loss.double() - want).abs().max()) <= 4 * 9 * 2.0 ** -24 + (V / 128 + 160) * 2.0 ** -24 + 4 * 16 * 2.0 ** -24, which


@pytest.mark.parametrize("n,V,C", LOW_PIECES + [(200, 119, 130), (5000, 12004, 130), (600, 48016, 768), (9001, 811, 1000)])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_linear_cross_entropy_float32_gradients_keep_24_bits(reduction, n, V, C):
    x, w, of_x, of_w = gradient_case(n, V, C)
    t = torch.full((n,), V - 1)
    leaves = [x.cuda().requires_grad_(), w.cuda().requires_grad_()]
    loss = ops.linear_cross_entropy(*leaves, t.cuda(), reduction=reduction)
    gx, gw = torch.autograd.grad(loss, leaves, torch.full_like(loss, float(n) if reduction == "mean" else 1.0))
    assert gradient_errors(V, gx.cpu(), gw.cpu(), t, of_x, of_w) <= gradient_bound(V)


def _poison(value):
    """What the allocator hands out next has held `value`."""
    blocks = [torch.full((n,), value, device="cuda") for n in (1 << 26, 1 << 22, 1 << 18, 1 << 14, 1 << 10, 64) for _ in range(4)]
    torch.cuda.synchronize()
    del blocks


@pytest.mark.parametrize("dtype", TYPES)
def test_training_operators_give_equal_bits_whatever_memory_held_and_on_two_streams(dtype):
    cases = []
    for n, V, C in ((1, 700, 200), (4, 700, 200), (16, 300, 136), (100, 700, 200), (300, 5001, 200), (1000, 700, 48)):
        x, w = randn(n, C, seed=n).to(dtype).requires_grad_(), randn(V, C, seed=n + 1).to(dtype).requires_grad_()
        t = torch.arange(n, device="cuda") * 7 % V
        t[1::3] = -100

        def loss(x=x, w=w, t=t):
            value = ops.linear_cross_entropy(x, w, t, scale=0.3)
            return (value.detach(), *torch.autograd.grad(value, (x, w)))
        cases.append(loss)
    for n, rows, C in ((50, 1000, 33), (9000, 70, 64), (40000, 5000, 8)):
        table, index = randn(rows, C, seed=n).to(dtype).requires_grad_(), (torch.rand(n, device="cuda") ** 3 * rows).long()
        g = randn(n, C, seed=n + 1).to(dtype)
        cases.append(lambda table=table, index=index, g=g: torch.autograd.grad(ops.lookup_rows(table, index, 0.7), table, g))
    a = randn(777, 33, seed=1).to(dtype)
    cases.append(lambda: (ops.act8_dequantize(ops.act8_quantize(a)),))
    side = torch.cuda.Stream()
    for i, case in enumerate(cases):
        want = case()
        for value in (float("nan"), 3e38):
            _poison(value)
            assert all(torch.equal(p, q) for p, q in zip(case(), want)), (i, value)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            there = [case() for _ in range(3)]
        here = [case() for _ in range(3)]
        torch.cuda.synchronize()
        for got in there + here:
            assert all(torch.equal(p, q) for p, q in zip(got, want)), i


def test_matching_loss_captured_and_replayed():
    """... with another number of pairs each time, a view without any among them."""
    bufs = [*_scene(H=256, W=320), torch.ones(1, 64, 80, device="cuda")]
    torch.manual_seed(3)
    model = MVSNet(refine=False).cuda().train()
    weights = list(model.feature.parameters())

    def step():
        loss = model.matching_loss(*bufs)
        return [loss.detach(), *torch.autograd.grad(loss, weights)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="relaxed"):
        out = step()
    for seed in range(6, 12):
        imgs, proj, gt = _scene(seed=seed, H=256, W=320)
        if seed % 3 == 1:
            proj[:, 1, 2] *= -1
        mask = (torch.rand(gt.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") < 0.3 * (seed % 4)).float()
        for b, v in zip(bufs, (imgs, proj, gt, mask)):
            b.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and (float(want[0]) == 0) == (seed % 4 == 0), seed
        for g, w in zip(got[1:], want[1:]):      # (the convolutions' weight gradients end in floating-point atomics)
            assert torch.isfinite(w).all() and float((g - w).norm()) <= 1e-5 * float(w.norm()), seed


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,V,C", [(300, 300, 8), (1021, 511, 8), (50, 200, 33), (400, 300, 128), (130, 511, 100), (2, 300, 130), (3, 511, 1024), (4, 301, 257)])
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_linear_cross_entropy_of_narrow_or_few_16_bit_rows_keeps_the_logits_gradient(reduction, n, V, C, dtype):
    """A table around a common value: what a row's gradients of the logits, which sum to 0, make of it cancels, and what they are rounded
    to would show.  Sixteenths throughout, so that a logit is a sum of exact products without a rounding."""
    x, w = (torch.round(4 * randn(n, C, seed=n)) / 16).to(dtype), (2 + torch.round(4 * randn(V, C, seed=n + 1)) / 16).to(dtype)
    t = torch.arange(n, device="cuda") * 7 % V
    t[1::5] = -100
    leaves = [x.requires_grad_(), w.requires_grad_()]
    loss = ops.linear_cross_entropy(*leaves, t, reduction=reduction)
    g = 0.5 + torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") if reduction == "none" else torch.ones((), device="cuda")
    gx, gw = torch.autograd.grad(loss, leaves, g)
    kept = (t >= 0).nonzero().squeeze(1)
    xd, wd = x.detach()[kept].double(), w.detach().double()
    l = xd @ wd.t()
    p = torch.exp(l - torch.logsumexp(l, 1, keepdim=True))
    dl = p.clone()
    dl[torch.arange(len(kept), device="cuda"), t[kept]] -= 1
    factor = (g.double()[kept] if reduction == "none" else torch.ones(len(kept), dtype=torch.float64, device="cuda")).unsqueeze(1)
    # A logit is rounded with its scale and again as an exponent, 4 u of it; a probability is off by twice the largest of a row's and its
    # sum's roundings, (V / 128 + 160) u.  Each logit's gradient keeps 16 bits at the least (float16: down to 2^-39; with factors of its own a
    # row's come to the largest one's before that).  Sums of V or n float32 products, and the result rounded once.
    u, h = 2.0 ** -24, torch.finfo(dtype).eps / 2
    off_l = 4 * u * l.abs().amax(1, keepdim=True)
    off = p * (2 * off_l + 2 * (V / 128 + 160) * u) + 2.0 ** -16 * dl.abs() + (2.0 ** -38 if dtype == torch.float16 else 0.0)
    least = torch.finfo(dtype).smallest_normal * h
    dx, off_x = (dl * factor) @ wd, ((off + (V + 8) * u * dl.abs()) * factor) @ wd.abs()
    dw, off_w = (dl * factor).t() @ xd, ((off + (n + 8) * u * dl.abs()) * factor).t() @ xd.abs()
    over_x = ((gx[kept].double() - dx).abs() / (off_x + h * (dx.abs() + off_x) + least)).max()
    over_w = ((gw.double() - dw).abs() / (off_w + h * (dw.abs() + off_w) + least)).max()
    assert float(over_x) <= 1 and float(over_w) <= 1, (float(over_x), float(over_w))
    assert (gx[t < 0] == 0).all()
