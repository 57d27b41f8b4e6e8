"""The training operators that keep no large tensor, on the GPU, against plain implementations in 64 bits.

Tolerances are error bounds: u = 2^-24 (float32 rounding), h = half a unit in the last place of the operand type (finfo.eps / 2)."""
import math

import numpy as np
import pytest
import torch

from mvs_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed), device="cuda")


# ------------------------------------------------------------------ activations in 8 bits
def act8_by_definition(x):
    """(codes, scales) from the definition, in 64 bits on the host."""
    v = x.detach().double().cpu().numpy().reshape(-1)
    n = v.size
    v = np.concatenate([v, np.zeros(-n % 32)]).reshape(-1, 32)
    codes, scales = np.zeros(v.shape, np.int8), np.zeros(len(v), np.uint8)
    for b, row in enumerate(v):
        if not np.isfinite(row).all():
            scales[b] = 255
            continue
        most, k = np.abs(row).max(), -126
        if most > 0:
            k = max(-126, int(math.floor(math.log2(most))) - 8)
        while np.rint(most * 2.0 ** -k) > 127:
            k += 1
        codes[b], scales[b] = np.rint(row * 2.0 ** -k), k + 127
    return codes.reshape(-1)[:n], scales


def values_of(codes, scales, shape):
    step = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return torch.from_numpy(codes.astype(np.float64) * np.repeat(step, 32)[:codes.size]).reshape(shape)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (31,), (32,), (33,), (64, 8), (5, 77), (3, 1024), (2, 5, 7, 16), (65, 1031)])
def test_act8_is_its_definition_bit_for_bit(shape, dtype):
    x = (randn(*shape, seed=len(shape)) * torch.exp(2 * randn(*shape, seed=3))).to(dtype)
    held = ops.act8_quantize(x)
    codes, scales = act8_by_definition(x)
    assert np.array_equal(held.codes.cpu().numpy(), codes) and np.array_equal(held.scales.cpu().numpy(), scales)
    back = ops.act8_dequantize(held)
    assert back.dtype == dtype and back.shape == x.shape and held.nbytes == x.numel() + -(-x.numel() // 32)
    assert torch.equal(back.cpu(), values_of(codes, scales, shape).to(dtype))
    for other in TYPES:
        assert torch.equal(ops.act8_dequantize(held, other).cpu().double().clamp(-1e30, 1e30),
                           values_of(codes, scales, shape).clamp(-torch.finfo(other).max, torch.finfo(other).max).to(other).double().clamp(-1e30, 1e30))


def test_act8_extreme_values():
    big = torch.finfo(torch.float32).max
    rows = [[0.0] * 32, [big] * 32, [-big] + [1.0] * 31, [1e-45] * 32, [1e-38, -3e-39] * 16, [127.0, 127.49, -127.49, 0.5, 1.5, 2.5, -0.5, -1.5] * 4,
            [127.5, 0.5] * 16, [255.0 / 128, 1.0] * 16, [2.0 ** -120] * 32, [-0.0] * 32]
    x = torch.tensor(rows, device="cuda")
    held = ops.act8_quantize(x)
    codes, scales = act8_by_definition(x)
    assert np.array_equal(held.codes.cpu().numpy(), codes) and np.array_equal(held.scales.cpu().numpy(), scales)
    back = ops.act8_dequantize(held)
    assert torch.isfinite(back).all() and float(back[1, 0]) == big
    h = torch.full((64,), 65504.0, device="cuda", dtype=torch.float16)
    assert torch.equal(ops.act8_dequantize(ops.act8_quantize(h)), h)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", TYPES)
def test_act8_a_poisoned_block_reads_back_as_nan_and_no_other(bad, dtype):
    x = randn(100, seed=1).to(dtype)
    x[40] = bad
    x[99] = bad
    back = ops.act8_dequantize(ops.act8_quantize(x))
    assert torch.isnan(back[32:64]).all() and torch.isnan(back[96:]).all() and torch.isfinite(back[:32]).all() and torch.isfinite(back[64:96]).all()


def test_act8_strides_offsets_and_empty_tensors():
    x = randn(64, 40, seed=5)
    for view in (x.t(), x[:, ::2], x[1:, 1:], x.reshape(-1)[3:], x.half().reshape(-1)[1:]):
        a, b = ops.act8_quantize(view), ops.act8_quantize(view.clone(memory_format=torch.contiguous_format))
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        assert torch.equal(ops.act8_dequantize(a), ops.act8_dequantize(b))
    empty = ops.act8_quantize(torch.empty(0, 8, device="cuda"))
    assert ops.act8_dequantize(empty).shape == (0, 8) and empty.nbytes == 0


def bn_by_formula(x, held, gy, w, b, skip, relu, groups, eps):
    """y and the gradients in 64 bits; x [G, N, C]; the backward sees `held` (the values of the 8-bit form) and the forward's mask."""
    x, gy, w, b = x.double(), gy.double(), w.double(), b.double()
    mean, var = x.mean(1, keepdim=True), x.var(1, keepdim=True, unbiased=False)
    inv = 1 / torch.sqrt(var + eps)
    z = (x - mean) * inv * w + b
    y = torch.relu(z) if relu else z
    dz = gy * (z > 0) if relu else gy
    hat = (held.double() - mean) * inv
    dx = w * inv * (dz - dz.mean(1, keepdim=True) - hat * (dz * hat).mean(1, keepdim=True))
    return y + (skip.double() if skip is not None else 0), dx, (dz * hat).sum((0, 1)), dz.sum((0, 1)), z, (dz, hat, inv, w)


@pytest.mark.parametrize("relu", [True, False])
@pytest.mark.parametrize("C,N,groups,skip", [(8, 1, 1, False), (8, 7, 3, True), (8, 1000, 1, True), (16, 333, 2, False), (32, 65, 5, True), (64, 129, 1, False),
                                            (8, 5003, 3, True)])
def test_bn_act8_against_the_formula(C, N, groups, skip, relu):
    x = randn(groups, N, C, seed=1) * 2 + randn(C, seed=2)
    bn, plain = torch.nn.BatchNorm2d(C).cuda().train(), torch.nn.BatchNorm2d(C).cuda().train()
    with torch.no_grad():
        bn.weight.copy_(1 + 0.3 * randn(C, seed=3))
        bn.bias.copy_(0.5 * randn(C, seed=4))
    plain.load_state_dict(bn.state_dict())
    with torch.no_grad():      # off the ReLU's corner, where either gradient is right
        mean, var = x.double().mean(1, keepdim=True), x.double().var(1, keepdim=True, unbiased=False)
        z = (x - mean) / torch.sqrt(var + bn.eps) * bn.weight + bn.bias
        x = x + 0.05 * (z.abs() < 1e-4).float()
    sk = randn(groups, N, C, seed=6) if skip else None
    gy = randn(groups, N, C, seed=7)
    leaves = [x.clone().requires_grad_(), bn.weight, bn.bias] + ([sk.clone().requires_grad_()] if skip else [])
    y = ops.bn_relu_cl(leaves[0], bn, relu=relu, skip=leaves[3] if skip else None, groups=groups, act8=True)
    grads = torch.autograd.grad(y, leaves, gy)
    # the output and the running statistics are those of the block that keeps float32
    assert torch.equal(y, ops.bn_relu_cl(x, plain, relu=relu, skip=sk, groups=groups))
    assert torch.equal(bn.running_mean, plain.running_mean) and torch.equal(bn.running_var, plain.running_var)
    assert int(bn.num_batches_tracked) == groups
    held = ops.act8_dequantize(ops.act8_quantize(x))
    want_y, want_dx, want_dw, want_db, _, (dz, hat, inv, w) = bn_by_formula(x, held, gy, bn.weight.detach(), bn.bias.detach(), sk, relu, groups, bn.eps)
    if skip:
        assert torch.equal(grads[3], gy)
    if N == 1:
        # one row: the variance is 0, x - mean a rounding of 0 and 1 / sqrt(eps) = 316 multiplies whatever the codes are off by
        # -- the formula's dx is 0 only for held == x; what is asserted is that dL/dbias does not depend on it
        assert torch.allclose(grads[2].double(), want_db, atol=4 * U * float(gy.abs().sum()))
        return
    # dx = inv w (dz - k2 - xm k1): about ten float32 roundings of terms of these magnitudes, mean and inv rounded once each (the
    # mean's rounding moves hat by u |mean| inv)
    n = dz.shape[1]
    shift = x.double().abs().amax() * inv
    scale = w.abs() * inv * (dz.abs() + dz.abs().mean(1, keepdim=True) + (hat.abs() + shift) * (dz * hat).abs().mean(1, keepdim=True)
                             + hat.abs() * (dz.abs() * shift).mean(1, keepdim=True))
    assert ((grads[0].double() - want_dx).abs() <= 16 * U * scale).all()
    assert ((grads[1].double() - want_dw).abs() <= 16 * U * (dz.abs() * (hat.abs() + shift)).sum((0, 1))).all()
    assert ((grads[2].double() - want_db).abs() <= 4 * U * dz.abs().sum((0, 1))).all()


def test_bn_act8_keeps_a_third_of_the_memory():
    x = randn(1, 200_000, 8, seed=1).requires_grad_()
    bn = torch.nn.BatchNorm2d(8).cuda().train()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.numel() * t.element_size()) or t, lambda t: t):
        ops.bn_relu_cl(x, bn, act8=True)
    assert sum(kept) < 1.2 * x.numel()


# ------------------------------------------------------------------ rows by index
def lookup_bound(table, index, g, scale):
    """The gradient in 64 bits, and the error bound of a float32 sum of a row's k terms, rounded to the type once."""
    ok = (index >= 0) & (index < table.shape[0])
    at = torch.where(ok, index, 0)
    g = torch.where(ok.unsqueeze(-1), g.double(), torch.zeros((), dtype=torch.float64, device=g.device))
    C = table.shape[1]
    want, mag = (torch.zeros(table.shape, dtype=torch.float64, device="cuda").index_put_((at.reshape(-1),), t.reshape(-1, C), accumulate=True)
                 for t in (g, g.abs()))
    count = torch.zeros(table.shape[0], dtype=torch.float64, device="cuda").index_put_((at.reshape(-1),), ok.double().reshape(-1), accumulate=True)
    bound = abs(scale) * mag * (count.unsqueeze(1) + 2) * U + half_ulp(table.dtype) * abs(scale) * mag + torch.finfo(table.dtype).smallest_normal
    return want * scale, bound


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C,n", [(1, 1, 1), (1, 8, 50), (5, 3, 17), (100, 8, 1), (64, 32, 64), (65, 33, 200), (1000, 257, 333), (20480, 32, 1021),
                                      (300, 2048, 129), (7, 64, 9000), (5000, 16, 20011), (40000, 40, 8193)])
def test_lookup_rows_and_its_gradient(rows, C, n, dtype):
    table = randn(rows, C, seed=rows).to(dtype).requires_grad_()
    index = torch.randint(rows, (n,), generator=gen(n), device="cuda")
    index[::3] = int(index[0])                                  # one index makes up a third: its run spans many pieces
    if n > 4:
        index[1], index[3] = -1, rows                       # these name no row
    scale = 1.7
    out = ops.lookup_rows(table, index, scale)
    ok = (index >= 0) & (index < rows)
    # The product of a float32 scale and a 16-bit value takes up to 35 bits.  A multiplication in float32 and one rounding to the type
    # give (1 + u)(1 + h) at worst, a multiply-and-round instruction (float16 has one) 1 + h: both are within h + u + h u of the
    # exact product, plus half the spacing of the type's subnormal numbers
    want = table.detach()[torch.where(ok, index, 0)].double() * float(np.float32(scale)) * ok.unsqueeze(1)
    h = half_ulp(dtype)
    assert ((out.double() - want).abs() <= (h + U + h * U) * want.abs() + torch.finfo(dtype).smallest_normal * h).all()
    assert (out[~ok] == 0).all()
    g = randn(n, C, seed=2).to(dtype)
    grad, = torch.autograd.grad(out, table, g, retain_graph=True)
    want, bound = lookup_bound(table, index, g, scale)
    assert ((grad.double() - want).abs() <= bound).all()
    untouched = torch.ones(rows, dtype=torch.bool, device="cuda")
    untouched[index[ok]] = False
    assert (grad[untouched] == 0).all()
    again, = torch.autograd.grad(out, table, g)
    assert torch.equal(grad, again)


@pytest.mark.parametrize("n", [8191, 8192, 8193, 30000])
def test_lookup_rows_gradient_order_is_the_indices_order(n):
    """Equal keys are summed in their order: with terms 2^24, 1, ..., 1, -2^24 any other order gives another float32 sum."""
    index = torch.full((n,), 3, device="cuda")
    index[:16] = torch.tensor([3, 1] * 8, device="cuda")
    table = torch.zeros(5, 4, device="cuda", requires_grad=True)
    g = torch.zeros(n, 4, device="cuda")
    g[1], g[3:15:2], g[15] = 2.0 ** 24, 1.0, -2.0 ** 24      # index 1's eight terms: 2^24 + 1 + ... (each lost) - 2^24 = 0
    grad, = torch.autograd.grad(ops.lookup_rows(table, index), table, g)
    assert (grad[1] == 0).all() and (grad[[0, 2, 4]] == 0).all()


def test_lookup_rows_shapes_strides_and_empty():
    table = randn(50, 16, seed=1)
    index = torch.randint(50, (4, 6), generator=gen(2), device="cuda")
    for t in (table, randn(16, 50, seed=3).t(), randn(50, 32, seed=4)[:, ::2], randn(51, 16, seed=5)[1:], randn(50, 17, seed=6)[:, 1:]):
        for i in (index, index.t(), index.to(torch.int32), index[:, :1]):
            leaf = t.detach().requires_grad_()
            out = ops.lookup_rows(leaf, i, 0.5)
            assert torch.equal(out, t[i.long()] * 0.5)
            grad, = torch.autograd.grad(out, leaf, torch.ones_like(out))
            assert torch.equal(grad[:, 0], 0.5 * torch.bincount(i.long().reshape(-1), minlength=50).float())
    leaf = table.clone().requires_grad_()
    out = ops.lookup_rows(leaf, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert out.shape == (0, 16)
    grad, = torch.autograd.grad(out, leaf, torch.empty(0, 16, device="cuda"))
    assert (grad == 0).all()


@pytest.mark.parametrize("n", [16384, 16385, 40000, (1 << 18) + 1, (1 << 22) + 3])
@pytest.mark.parametrize("spread", ["flat", "steep", "one"])
def test_lookup_rows_gradient_pieces_of_every_length(n, spread):
    """Runs of equal indices that end on, before and behind the ends of the pieces that the sorted terms are cut into."""
    rows, C = 1000, 8
    if spread == "flat":
        index = torch.randint(-1, rows + 1, (n,), generator=gen(1), device="cuda")
    elif spread == "steep":
        index = (rows * torch.rand(n, generator=gen(1), device="cuda", dtype=torch.float64) ** 8).long()
    else:
        index = torch.full((n,), 7, device="cuda")
        index[::3001] = 11
    g = randn(n, C, seed=2)
    leaf = torch.zeros(rows, C, device="cuda").requires_grad_()
    grad, = torch.autograd.grad(ops.lookup_rows(leaf, index, 0.5), leaf, g)
    named = (index >= 0) & (index < rows)
    at, terms = index[named].cpu(), g[named].double().cpu()      # (in order, on the CPU: a card's float64 atomics on one row queue for minutes)
    zero = torch.zeros(rows, C, dtype=torch.float64)
    want, mag = zero.index_add(0, at, terms) * 0.5, zero.index_add(0, at, terms.abs()) * 0.5
    count = torch.bincount(at, minlength=rows).unsqueeze(1)
    assert ((grad.cpu().double() - want).abs() <= (count + 2) * U * mag).all()
    assert torch.equal(grad, torch.autograd.grad(ops.lookup_rows(leaf, index, 0.5), leaf, g)[0])

# ------------------------------------------------------------------ cross entropy against a large table
def ce_case(n, V, C, dtype, ignored=0.2, sharp=1.0, seed=0):
    w = randn(V, C, seed=seed + 1) / math.sqrt(C)
    t = torch.randint(V, (n,), generator=gen(seed + 2), device="cuda")
    x = (randn(n, C, seed=seed + 3) + w[t] * 2).to(dtype)
    t[torch.rand(n, generator=gen(seed + 4), device="cuda") < ignored] = -100
    return x, w.to(dtype), t, sharp


def ce_bounds(x, w, t, scale, ignore, g_row):
    """Row losses and gradients in 64 bits (g_row: dL/dloss_n) with bounds of the kernels' error.
    A logit: C products summed in float32, in any order, and the scale: (C + 4) u scale |x||w|^T =: d (base-2 scaling included).
    A row's lse moves by at most the largest d of the row, its terms are summed in float32 (a tile's 128 terms, then tiles):
    e = max d + (V / 128 + 160) u.  p: relative error 2 e + 8 u.  dl rounded to the type (h), its unit's smallest normal number
    for float16.  The products: one float32 sum over V (or n) terms.  The result rounded once."""
    dtype = x.dtype
    xd, wd = x.double(), w.double()
    kept = t != ignore
    xd = torch.where(kept.unsqueeze(1), xd, torch.zeros((), dtype=torch.float64, device=x.device))
    at = torch.where(kept, t, 0)
    n, V, C = x.shape[0], w.shape[0], x.shape[1]
    l = scale * (xd @ wd.t())
    d = (C + 4) * U * abs(scale) * (xd.abs() @ wd.abs().t()) + 4 * U * l.abs()
    e = d.amax(1, keepdim=True) + (V / 128 + 160) * U
    lse = torch.logsumexp(l, 1, keepdim=True)
    own = l.gather(1, at.unsqueeze(1))
    loss = torch.where(kept, (lse - own).squeeze(1), torch.zeros((), dtype=torch.float64, device=x.device))
    loss_bound = (2 * e + 4 * U * (lse.abs() + own.abs())).squeeze(1)
    p = torch.exp(l - lse)
    dl = p.clone()
    dl[torch.arange(n, device=x.device), at] -= 1
    h = half_ulp(dtype) if dtype != torch.float32 else U
    tiny = 2.0 ** -25 / 16384 if dtype == torch.float16 else 0.0
    dl_err = p * (2 * e + 8 * U) + 2 * h * dl.abs() + tiny
    grow = (torch.where(kept, g_row.double(), torch.zeros((), dtype=torch.float64, device=x.device)) * scale).unsqueeze(1)
    small = torch.finfo(dtype).smallest_normal * (2.0 ** -10 if dtype == torch.float16 else 1)
    dx, dw = (dl * grow) @ wd, (dl * grow).t() @ xd
    dx_bound = (dl_err * grow.abs()) @ wd.abs() + (V + 8) * U * (dl.abs() * grow.abs()) @ wd.abs()
    dw_bound = (dl_err * grow.abs()).t() @ xd.abs() + (n + 8) * U * (dl.abs() * grow.abs()).t() @ xd.abs()
    return loss, loss_bound, dx, dx_bound + half_ulp(dtype) * (dx.abs() + dx_bound) + small, dw, dw_bound + half_ulp(dtype) * (dw.abs() + dw_bound) + small


def ce_check(x, w, t, scale, ignore=-100, reduction="mean", seed=9):
    leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
    loss = ops.linear_cross_entropy(*leaves, t, scale=scale, ignore_index=ignore, reduction=reduction)
    n, kept = x.shape[0], int((t != ignore).sum())
    g = randn(n, seed=seed) if reduction == "none" else torch.tensor(0.7, device="cuda")
    g_row = g if reduction == "none" else (g / kept if reduction == "mean" and kept else g).expand(n)
    want, bound, dx, dx_bound, dw, dw_bound = ce_bounds(x, w, t, scale, ignore, g_row)
    got_dx, got_dw = torch.autograd.grad(loss, leaves, g)
    assert loss.dtype == torch.float32 and got_dx.dtype == x.dtype and got_dw.dtype == w.dtype
    if reduction == "none":
        assert ((loss.double() - want).abs() <= bound).all()
    elif reduction == "sum":
        assert abs(float(loss) - float(want.sum())) <= float(bound.sum()) + U * float(want.sum())
    elif kept:
        assert abs(float(loss) - float(want.sum() / kept)) <= float(bound.max()) + 2 * U * float(want.sum() / kept)
    else:
        assert math.isnan(float(loss))
    assert ((got_dx.double() - dx).abs() <= dx_bound).all(), float(((got_dx.double() - dx).abs() / dx_bound).max())
    assert ((got_dw.double() - dw).abs() <= dw_bound).all(), float(((got_dw.double() - dw).abs() / dw_bound).max())
    assert (got_dx[t == ignore] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,C", [(1, 1, 1), (1, 2, 3), (2, 129, 8), (1, 1000, 64), (17, 130, 32), (64, 128, 33), (100, 257, 100), (129, 2000, 64),
                                   (130, 511, 200), (33, 5000, 320), (300, 300, 16), (1, 3, 130), (2, 1000, 257), (129, 129, 129), (70, 300, 1000),
                                   (257, 400, 128), (1, 5000, 512), (1500, 10, 32), (2000, 1000, 160)])
def test_linear_cross_entropy(n, V, C, dtype):
    x, w, t, _ = ce_case(n, V, C, dtype, seed=n)
    t[0] = min(t.clamp(min=0).max(), V - 1)
    ce_check(x, w, t, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_linear_cross_entropy_reductions_and_scales(reduction, dtype):
    x, w, t, _ = ce_case(150, 700, 48, dtype, seed=5)
    for scale in (1.0, 8.0, 0.125, -2.0):
        ce_check(x, w, t, scale, reduction=reduction)
    ce_check(x, w, t.clamp(min=3), 1.0, ignore=3, reduction=reduction)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [8, 130])
def test_linear_cross_entropy_in_pieces_of_the_table(dtype, C):
    """n V beyond 2^26: the backward pass walks the table in more than one piece (wide rows), the last of them a ragged one."""
    x, w, t, _ = ce_case(1025, 70001, C, dtype, seed=6)
    ce_check(x, w, t, 2.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_cross_entropy_no_row_kept(dtype):
    x, w, t, _ = ce_case(20, 50, 16, dtype, ignored=2.0)
    for reduction in ("mean", "sum", "none"):
        ce_check(x, w, t, 1.0, reduction=reduction)
    x = torch.empty(0, 16, device="cuda", dtype=dtype, requires_grad=True)
    w = w.detach().requires_grad_()
    empty = torch.empty(0, dtype=torch.int64, device="cuda")
    assert math.isnan(float(ops.linear_cross_entropy(x, w, empty)))
    loss = ops.linear_cross_entropy(x, w, empty, reduction="sum")
    gx, gw = torch.autograd.grad(loss, (x, w))
    assert float(loss) == 0 and gx.shape == (0, 16) and (gw == 0).all()
    assert ops.linear_cross_entropy(x, w, empty, reduction="none").shape == (0,)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_linear_cross_entropy_what_an_ignored_row_holds_leaves_no_trace(bad, dtype):
    x, w, t, _ = ce_case(70, 200, 40, dtype, seed=7)
    t[3] = t[50] = -100
    clean = x.clone()
    clean[[3, 50]] = 0
    x[3], x[50, 5] = bad, bad
    res = []
    for rows in (x, clean):
        leaves = [rows.detach().requires_grad_(), w.detach().requires_grad_()]
        loss = ops.linear_cross_entropy(*leaves, t)
        res.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    for a, b in zip(*res):
        assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_cross_entropy_poisoned_rows_show(dtype):
    x, w, t, _ = ce_case(10, 200, 40, dtype, ignored=0.0, seed=8)
    for bad_t in (-1, 200, 2 ** 40):
        t2 = t.clone()
        t2[4] = bad_t
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        loss = ops.linear_cross_entropy(*leaves, t2, reduction="none")
        assert torch.isnan(loss[4]) and torch.isfinite(loss[[0, 1, 2, 3, 5, 6, 7, 8, 9]]).all()
        gx, gw = torch.autograd.grad(loss.sum(), leaves)
        assert torch.isnan(gx[4]).all() and torch.isfinite(gx[:4]).all() and torch.isnan(gw).all()
    x2 = x.clone()
    x2[2, 3] = float("nan")
    loss = ops.linear_cross_entropy(x2, w, t, reduction="none")
    assert torch.isnan(loss[2]) and torch.isfinite(loss[3:]).all()
    # a table row of the type's lowest value: its logit is a large number of either sign or -Inf / Inf, as in torch
    low = w.clone()
    low[7] = torch.finfo(dtype).min
    want = torch.nn.functional.cross_entropy((x.float().abs() @ low.float().t()), t.clamp(min=8), reduction="none")
    got = ops.linear_cross_entropy(x.abs(), low, t.clamp(min=8), reduction="none")
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)) and torch.allclose(got, want, rtol=1e-3, atol=1e-3)


def test_linear_cross_entropy_one_gradient_at_a_time_and_shapes():
    x, w, t, _ = ce_case(60, 300, 64, torch.bfloat16, seed=10)
    both = torch.autograd.grad(ops.linear_cross_entropy(a := x.detach().requires_grad_(), b := w.detach().requires_grad_(), t), (a, b))
    gx, = torch.autograd.grad(ops.linear_cross_entropy(a := x.detach().requires_grad_(), w, t), (a,))
    gw, = torch.autograd.grad(ops.linear_cross_entropy(x, b := w.detach().requires_grad_(), t), (b,))
    assert torch.equal(gx, both[0]) and torch.equal(gw, both[1])
    flat = ops.linear_cross_entropy(x, w, t, reduction="none")
    assert torch.equal(ops.linear_cross_entropy(x.view(6, 10, 64), w, t.view(6, 10), reduction="none"), flat.view(6, 10))
    assert torch.equal(ops.linear_cross_entropy(x[0], w, t[0], reduction="none"), flat[0])
    wide = torch.zeros(60, 130, device="cuda", dtype=x.dtype)
    wide[:, 1:65] = x
    assert torch.equal(ops.linear_cross_entropy(wide[:, 1:65], w, t.to(torch.int32), reduction="none"), flat)
    assert torch.equal(ops.linear_cross_entropy(x, w.t().contiguous().t(), t, reduction="none"), flat)


# rows longer than the narrow kernels take: few of them, those of one tile, and those that are moved together
WIDE = [10, 70, 200]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", WIDE)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_linear_cross_entropy_wide_rows_reductions_and_scales(reduction, n, dtype):
    x, w, t, _ = ce_case(n, 701, 200, dtype, seed=n)
    for scale in (1.0, 4.0, 0.125, -2.0, 0.0):
        ce_check(x, w, t, scale, reduction=reduction)
    ce_check(x, w, t.clamp(min=3), 1.0, ignore=3, reduction=reduction)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", WIDE)
def test_linear_cross_entropy_wide_rows_without_a_kept_one(n, dtype):
    x, w, t, _ = ce_case(n, 150, 136, dtype, ignored=2.0)
    for reduction in ("mean", "sum", "none"):
        ce_check(x, w, t, 1.0, reduction=reduction)
    t[n // 2] = 149      # ... and with one
    for reduction in ("mean", "sum", "none"):
        ce_check(x, w, t, 1.0, reduction=reduction)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", WIDE)
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_linear_cross_entropy_wide_rows_ignored_and_poisoned(reduction, n, dtype):
    x, w, t, _ = ce_case(n, 333, 200, dtype, seed=7)
    t[3], t[n - 1], t[1], t[n - 2] = -100, -100, 0, 332
    clean = x.clone()
    clean[[3, n - 1]] = 0
    x[3], x[n - 1, 5] = float("nan"), float("inf")
    res = []
    for rows in (x, clean):
        leaves = [rows.detach().requires_grad_(), w.detach().requires_grad_()]
        loss = ops.linear_cross_entropy(*leaves, t, reduction=reduction)
        res.append([loss.detach(), *torch.autograd.grad(loss.sum(), leaves)])
    for a, b in zip(*res):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    # the last kept row holds a NaN, or names no class: it shows in its own gradient and in the table's, and nowhere else
    for target in (332, 333):
        bad = clean.clone()
        t[n - 2] = target
        if target == 332:
            bad[n - 2, 9] = float("nan")
        leaves = [bad.requires_grad_(), w.detach().requires_grad_()]
        loss = ops.linear_cross_entropy(*leaves, t, reduction=reduction)
        gx, gw = torch.autograd.grad(loss.sum(), leaves)
        assert torch.isnan(gx[n - 2]).all() and torch.isfinite(gx[:n - 2]).all() and (gx[[3, n - 1]] == 0).all() and torch.isnan(gw).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", WIDE)
def test_linear_cross_entropy_wide_rows_one_gradient_at_a_time(n, dtype):
    x, w, t, _ = ce_case(n, 500, 140, dtype, seed=10)
    both = torch.autograd.grad(ops.linear_cross_entropy(a := x.detach().requires_grad_(), b := w.detach().requires_grad_(), t), (a, b))
    again = torch.autograd.grad(ops.linear_cross_entropy(a, b, t), (a, b))
    gx, = torch.autograd.grad(ops.linear_cross_entropy(a := x.detach().requires_grad_(), w, t), (a,))
    gw, = torch.autograd.grad(ops.linear_cross_entropy(x, b := w.detach().requires_grad_(), t), (b,))
    assert torch.equal(gx, both[0]) and torch.equal(gw, both[1]) and torch.equal(again[0], gx) and torch.equal(again[1], gw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [65, 129, 200, 500, 1000, 1024, 1025, 2048, 2050, 3000])
def test_linear_cross_entropy_of_a_single_row(C, dtype):
    """Rows that a workgroup holds whole, and longer ones; the target in the table's first, last and other rows, or ignored."""
    V = 331
    x, w, t, _ = ce_case(1, V, C, dtype, ignored=0.0, seed=C)
    for target in (0, 63, 64, V - 1, -100):
        t[0] = target
        for scale in (1.0, -0.5, 0.0):
            ce_check(x, w, t, scale, reduction="sum")
    x[0, C - 1] = float("nan")
    leaves = [x.requires_grad_(), w.requires_grad_()]
    for target, wrong in ((-100, False), (5, True)):
        t[0] = target
        loss = ops.linear_cross_entropy(*leaves, t, reduction="sum")
        gx, gw = torch.autograd.grad(loss, leaves)
        assert math.isnan(float(loss.detach())) == wrong and bool(torch.isnan(gx).all()) == wrong and bool(torch.isnan(gw).all()) == wrong
        assert wrong or ((gx == 0).all() and (gw == 0).all())
    leaves[0] = torch.full_like(x, float("inf")).detach().requires_grad_()
    t[0] = 5
    gx, gw = torch.autograd.grad(ops.linear_cross_entropy(*leaves, t, reduction="sum"), leaves)
    assert not torch.isfinite(gx).any() and not torch.isfinite(gw).any()

@pytest.mark.parametrize("n,V,C", [(257, 100, 65), (300, 3001, 130), (1100, 777, 513), (2500, 6000, 700)])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_linear_cross_entropy_of_many_wide_float32_rows(reduction, n, V, C):
    """float32 rows in three pieces, forward and backward (reduction 'none': its backward pass in float32)."""
    x, w, t, _ = ce_case(n, V, C, torch.float32, seed=n)
    for scale in (1.0, -3.0):
        ce_check(x, w, t, scale, reduction=reduction)


@pytest.mark.parametrize("n,V,C", [(257, 100, 65), (300, 3001, 130), (1100, 777, 513), (2500, 6000, 700)])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_linear_cross_entropy_float32_pieces_at_the_ends_of_the_range(reduction, n, V, C):
    """Values that bfloat16 rounds to infinity, and ones whose last bits are below its least: a value is carried to within half of
    2^-133, so a logit of x = 2^128 (1 - 2^-24) and w < 2^-127 is off by at most 2^128 2^-134 = 2^-6, in either pass; a loss by two of
    those, an exponential by a factor of e^(2 2^-6).  (dW, some 2^128 times a probability, has sums that no float32 holds.)"""
    _, _, t, _ = ce_case(n, V, C, torch.float32, seed=n)
    big = torch.finfo(torch.float32).max
    x = torch.zeros(n, C, device="cuda")
    x[:, 0], x[:, 1] = big, 1e-30
    w = torch.zeros(V, C, device="cuda")
    w[:, 0], w[:, 1] = torch.arange(V, device="cuda") / V / big, 1e30
    leaf = x.requires_grad_()
    loss = ops.linear_cross_entropy(leaf, w, t, reduction=reduction)
    gx, = torch.autograd.grad(loss.sum(), leaf)
    kept = t >= 0
    logits = x.detach().double() @ w.double().t()
    lse = torch.logsumexp(logits, 1, keepdim=True)
    want = torch.where(kept, (lse - logits.gather(1, t.clamp(min=0).unsqueeze(1))).squeeze(1), 0.0)
    off = 2 * 2.0 ** -6 + 1e-4
    if reduction == "none":
        assert ((loss.detach().double() - want).abs() <= off).all()
    else:
        total, count = float(want.sum()), int(kept.sum())
        assert abs(float(loss.detach()) - (total if reduction == "sum" else total / count)) <= off * (count if reduction == "sum" else 1)
    p = torch.exp(logits - lse)
    dl = p.clone()
    dl[torch.arange(n, device="cuda"), t.clamp(min=0)] -= 1
    g = kept.double().unsqueeze(1) / (int(kept.sum()) if reduction == "mean" else 1)
    bound = (math.expm1(2 * 2.0 ** -6) + 1e-4) * (p * g) @ w.double().abs() + V * U * (dl.abs() * g) @ w.double().abs() + 2.0 ** -126
    assert ((gx.double() - (dl * g) @ w.double()).abs() <= bound).all()


def test_linear_cross_entropy_of_wide_float32_rows_in_pieces_of_the_table():
    x, w, t, _ = ce_case(1025, (1 << 17) + 301, 100, torch.float32, seed=6)
    ce_check(x, w, t, 2.0)
    x[5, 7] = float("nan")
    t[5] = -100
    leaves = [x.requires_grad_(), w.requires_grad_()]
    gx, gw = torch.autograd.grad(ops.linear_cross_entropy(*leaves, t), leaves)
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all() and (gx[5] == 0).all()

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,V,C", [(600, 40001, 768), (9001, 700, 1000), (3000, 5000, 1096)])
def test_linear_cross_entropy_on_large_tiles(n, V, C, dtype):
    """Sizes at which the 256 x 256 tiles are taken, with ragged edges on every side: by dW's product, by dx's, by the logits'."""
    x, w, t, _ = ce_case(n, V, C, dtype, seed=3)
    ce_check(x, w, t, 1.0)


def test_linear_cross_entropy_against_differences():
    x, w, t, _ = ce_case(12, 40, 8, torch.float32, seed=11)
    leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
    grads = torch.autograd.grad(ops.linear_cross_entropy(*leaves, t, scale=1.5, reduction="sum"), leaves)
    step = 2.0 ** -6
    for which, g in enumerate(grads):
        for seed in range(3):
            d = randn(*g.shape, seed=seed)
            d /= d.norm()
            ends = [float(ops.linear_cross_entropy(x + s * step * d if which == 0 else x, w + s * step * d if which else w, t, scale=1.5, reduction="sum"))
                    for s in (1, -1)]
            # second-order differences: the third derivative of the summed loss along a unit direction is below 12 * (1.5 |.|)^3
            # with |.| <= 5 the largest row norm; float32 losses of about 50 are off by 2^-18
            bound = 12 * (1.5 * 5) ** 3 * step ** 2 / 6 + 2.0 ** -17 / step
            assert abs((ends[0] - ends[1]) / (2 * step) - float((g * d).sum())) <= bound


# ------------------------------------------------------------------ together, other streams, graphs
def _step(features, keys, points, cells, bn, act8=True):
    """A training step as it uses them together: a BatchNorm block kept in 8 bits, the points' rows of its output, their loss
    against every cell of the other view."""
    f = ops.bn_relu_cl(features, bn, act8=act8)
    rows = ops.lookup_rows(f.reshape(-1, f.shape[-1]), points)
    loss = ops.linear_cross_entropy(rows, keys, cells, scale=4.0)
    return loss, torch.autograd.grad(loss, (features, keys, bn.weight, bn.bias))


def _step_inputs(seed):
    f = randn(1, 40, 50, 32, seed=seed).requires_grad_()
    keys = randn(2000, 32, seed=seed + 1).requires_grad_()
    points = torch.randint(2000, (333,), generator=gen(seed + 2), device="cuda")
    cells = torch.randint(2000, (333,), generator=gen(seed + 3), device="cuda")
    cells[::7] = -100
    return f, keys, points, cells


def test_the_operators_together_follow_autograd_in_64_bits():
    f, keys, points, cells = _step_inputs(1)
    bn = torch.nn.BatchNorm2d(32).cuda().train()
    loss, grads = _step(f, keys, points, cells, bn)
    fd, kd = f.detach().double().requires_grad_(), keys.detach().double().requires_grad_()
    wd, bd = bn.weight.detach().double().requires_grad_(), bn.bias.detach().double().requires_grad_()
    y = torch.relu(torch.nn.functional.batch_norm(fd.reshape(-1, 32), None, None, wd, bd, True, 0.0, bn.eps))
    want = torch.nn.functional.cross_entropy(4.0 * (y[points] @ kd.t()), cells)
    wants = torch.autograd.grad(want, (fd, kd, wd, bd))
    assert abs(float(loss) - float(want)) < 1e-5
    # float32 products of 32 terms and a softmax at scale 4: 1e-5; the 8-bit block enters through the normalised input only, within
    # half a step of its block's scale (1 / 254 of its largest magnitude, at most 5 standard deviations here): 2 % of the terms it is in
    for got, ref, tol in zip(grads, wants, (5e-3, 1e-5, 2e-2, 1e-5)):
        assert float((got.double() - ref).norm() / ref.norm()) < tol


def test_another_stream():
    side = torch.cuda.Stream()
    f, keys, points, cells = _step_inputs(2)
    bn = torch.nn.BatchNorm2d(32).cuda().train()
    want = _step(f, keys, points, cells, bn)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = _step(f, keys, points, cells, bn)
    side.synchronize()
    for a, b in zip((want[0], *want[1]), (got[0], *got[1])):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    bufs = _step_inputs(3)
    bn = torch.nn.BatchNorm2d(32).cuda().train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(*bufs, bn)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(*bufs, bn)
    for seed in (4, 8, 12, 16):
        new = _step_inputs(seed)
        with torch.no_grad():
            for b, v in zip(bufs, new):
                b.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(*new, bn)
        for a, b in zip((want[0], *want[1]), (out[0], *out[1])):
            assert torch.equal(a, b), seed


def test_double_backward_is_refused():
    x, w, t, _ = ce_case(5, 20, 8, torch.float32, ignored=0.0)
    leaf = x.detach().requires_grad_()
    g, = torch.autograd.grad(ops.linear_cross_entropy(leaf, w, t), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,C", [(1000, 300, 32), (1000, 300, 200), (5000, 100, 16), (129, 50, 160), (300, 70000, 40)])
@pytest.mark.parametrize("kept", ["first", "last", "one", "half", "none", "all"])
def test_linear_cross_entropy_kept_rows_anywhere(n, V, C, dtype, kept):
    """More than a tile of rows: the kept ones are moved together, wherever they are and however few."""
    x, w, t, _ = ce_case(n, V, C, dtype, ignored=0.0, seed=12)
    keep = torch.zeros(n, dtype=torch.bool, device="cuda")
    {"first": lambda: keep[:70].fill_(True), "last": lambda: keep[-70:].fill_(True), "one": lambda: keep[n // 2:n // 2 + 1].fill_(True),
     "half": lambda: keep[::2].fill_(True), "none": lambda: None, "all": lambda: keep.fill_(True)}[kept]()
    t = torch.where(keep, t, -100)
    x[~keep] = float("nan")
    ce_check(x, w, t, 1.5, reduction="mean")
    ce_check(x, w, t, 1.5, reduction="none")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,C", [(1, 40, 129), (2, 63, 257), (3, 64, 512), (4, 65, 1000), (5, 700, 130), (8, 1000, 2048), (9, 129, 2056), (15, 3000, 300),
                                   (16, 200, 4100), (17, 200, 300), (1, 20000, 1024)])
def test_linear_cross_entropy_few_rows(n, V, C, dtype):
    """One row to a few (and one more): both gradients in one pass over the table."""
    x, w, t, _ = ce_case(n, V, C, dtype, ignored=0.3 if n > 1 else 0.0, seed=13)
    x[t == -100] = float("nan")
    ce_check(x, w, t, 1.0)
    ce_check(x, w, t, 1.0, reduction="none")


# ------------------------------------------------------------------ offsets beyond 32 bits
def test_act8_beyond_2_to_31_values():
    n = (1 << 31) + 100
    x = torch.empty(n, device="cuda", dtype=torch.bfloat16)
    x[:100], x[100:-200], x[-200:] = randn(100, seed=1), 0.0, randn(200, seed=2)
    held = ops.act8_quantize(x)
    back = ops.act8_dequantize(held)
    small = torch.cat([x[:128], x[-228:]])      # whole blocks of the head; the last blocks (2^31 is a multiple of 32: -228 begins one)
    want = ops.act8_dequantize(ops.act8_quantize(small))
    assert torch.equal(back[:128], want[:128]) and torch.equal(back[-228:], want[128:])
    assert int(torch.count_nonzero(back[128:-228])) == 0


def test_lookup_rows_in_a_table_beyond_2_to_31_elements():
    rows, C, n = 1_100_000, 2048, 300
    table = torch.zeros(rows, C, device="cuda", dtype=torch.bfloat16)
    index = torch.randint(rows, (n,), generator=gen(1), device="cuda")
    index[:3] = rows - 1
    table[index] = randn(n, C, seed=2).to(table.dtype)
    leaf = table.requires_grad_()
    out = ops.lookup_rows(leaf, index)
    assert torch.equal(out, table.detach()[index])
    g = randn(n, C, seed=3).to(table.dtype)
    grad, = torch.autograd.grad(out, leaf, g)
    for row in (int(index[0]), int(index[10])):
        want = g[index == row].double().sum(0)
        assert ((grad[row].double() - want).abs() <= 4 * half_ulp(table.dtype) * g[index == row].double().abs().sum(0)).all()
    untouched = torch.ones(rows, dtype=torch.bool, device="cuda")
    untouched[index] = False
    assert int(torch.count_nonzero(grad.view(torch.int16).amax(1)[untouched])) == 0


@pytest.mark.parametrize("n", [3, 70])
def test_linear_cross_entropy_with_a_table_beyond_2_to_31_elements(n):
    V, C = 1_100_000, 2048
    w = torch.empty(V, C, device="cuda", dtype=torch.bfloat16)
    for v in range(0, V, 100_000):
        w[v:v + 100_000] = randn(min(100_000, V - v), C, seed=v) / math.sqrt(C)
    t = torch.randint(V, (n,), generator=gen(1), device="cuda")
    t[0], t[1] = V - 1, V - 2
    x = (randn(n, C, seed=2) + 4 * w[t].float()).to(torch.bfloat16)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    loss = ops.linear_cross_entropy(*leaves, t)
    gx, gw = torch.autograd.grad(loss, leaves)
    logits = torch.cat([x.detach().double() @ w.detach()[v:v + 100_000].double().t() for v in range(0, V, 100_000)], 1)
    lse = torch.logsumexp(logits, 1)
    want = (lse - logits.gather(1, t.unsqueeze(1)).squeeze(1)).mean()
    assert abs(float(loss.detach()) - float(want)) < 1e-4
    p = torch.exp(logits - lse.unsqueeze(1)) / n
    p[torch.arange(n, device="cuda"), t] -= 1 / n
    want_x = sum(p[:, v:v + 100_000] @ w.detach()[v:v + 100_000].double() for v in range(0, V, 100_000))
    assert float((gx.double() - want_x).norm() / want_x.norm()) < 2 * half_ulp(torch.bfloat16)
    for v in (0, V // 2, V - 100):      # dW = p^T x: h for dl, h for the result, relative to the terms
        mine, want_w = gw[v:v + 100].double(), p[:, v:v + 100].t() @ x.detach().double()
        mag = p[:, v:v + 100].abs().t() @ x.detach().double().abs()
        assert ((mine - want_w).abs() <= 3 * half_ulp(torch.bfloat16) * mag).all()


def test_act8_off_alignment_beyond_2_to_32_values():
    n = (1 << 32) + 100      # one lane a value: more threads than a grid's row has
    x = torch.zeros(n + 1, device="cuda")[1:]
    x[:100], x[-200:] = randn(100, seed=1), randn(200, seed=2)
    held = ops.act8_quantize(x)
    small = ops.act8_quantize(torch.cat([x[:128], x[-228:]]))
    assert torch.equal(held.codes[:128], small.codes[:128]) and torch.equal(held.codes[-228:], small.codes[128:])
    assert int(torch.count_nonzero(held.codes[128:-228])) == 0
    del x
    back = ops.act8_dequantize(held)
    want = ops.act8_dequantize(small)
    assert torch.equal(back[:128], want[:128]) and torch.equal(back[-228:], want[128:])


def test_lookup_rows_of_more_than_2_to_32_threads():
    rows, C, n = 11, 129, (1 << 26) + 5      # 64 lanes a row of odd length
    table = randn(rows, C, seed=1).to(torch.float16)
    index = torch.arange(n, device="cuda") % (rows + 1)      # (every twelfth names no row)
    out = ops.lookup_rows(table, index)
    padded = torch.cat([table, torch.zeros(1, C, device="cuda", dtype=table.dtype)])
    for at in (0, n // 2, n - 4096):
        assert torch.equal(out[at:at + 4096], padded[index[at:at + 4096]])


def test_lookup_rows_gradient_of_more_than_2_to_30_rows():
    rows, n = (1 << 30) + 77, 50
    leaf = torch.zeros(rows, 1, device="cuda", dtype=torch.bfloat16).requires_grad_()
    index = torch.randint(rows, (n,), generator=gen(1), device="cuda")
    index[0], index[1] = rows - 1, 0
    g = randn(n, 1, seed=2).to(torch.bfloat16)
    grad, = torch.autograd.grad(ops.lookup_rows(leaf, index), leaf, g)
    assert torch.equal(grad[index], g)
    grad[index] = 0
    assert int(torch.count_nonzero(grad)) == 0


def test_linear_cross_entropy_of_more_than_2_to_32_threads():
    """Half a million rows against a million: a forward pass of 2^23 tiles of 512 threads."""
    n, V, C = (1 << 19) + 3, (1 << 20) + 5, 136
    x, w = randn(n, C, seed=1).to(torch.bfloat16), (randn(V, C, seed=2) * 0.1).to(torch.bfloat16)
    t = torch.randint(V, (n,), generator=gen(3), device="cuda")
    loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    for at in (0, n // 2, n - 40):
        logits = x[at:at + 40].double() @ w.double().t()
        want = torch.logsumexp(logits, 1) - logits.gather(1, t[at:at + 40].unsqueeze(1)).squeeze(1)
        assert float((loss[at:at + 40].double() - want).abs().max()) < 1e-4

def test_linear_cross_entropy_few_rows_in_pieces():
    """16 rows against a table of more than 2^26 / 16 rows: the one-pass kernel adds the second piece's sums to the first's."""
    n, V, C = 16, (1 << 22) + 777, 136
    w = randn(V, C, seed=1).to(torch.float16) * 0.1
    t = torch.randint(V, (n,), generator=gen(1), device="cuda")
    t[0], t[1] = V - 1, -100
    x = (randn(n, C, seed=2) + 8 * w[t.clamp(min=0)].float()).to(torch.float16)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    loss = ops.linear_cross_entropy(*leaves, t)
    gx, gw = torch.autograd.grad(loss, leaves)
    keep = t >= 0
    logits = x.detach()[keep].double() @ w.detach().double().t()
    lse = torch.logsumexp(logits, 1)
    k = int(keep.sum())
    assert abs(float(loss.detach()) - float((lse - logits.gather(1, t[keep].unsqueeze(1)).squeeze(1)).mean())) < 1e-4
    p = torch.exp(logits - lse.unsqueeze(1)) / k
    p[torch.arange(k, device="cuda"), t[keep]] -= 1 / k
    want = p @ w.detach().double()
    assert float((gx[keep].double() - want).norm() / want.norm()) < 2 * half_ulp(torch.float16) and (gx[~keep] == 0).all()
    for rows in (slice(0, 100), slice(V - 800, V)):
        want = p[:, rows].t() @ x.detach()[keep].double()
        mag = p[:, rows].abs().t() @ x.detach()[keep].double().abs()
        assert ((gw[rows].double() - want).abs() <= 3 * half_ulp(torch.float16) * mag + 2.0 ** -25).all()



@pytest.mark.parametrize("n,V,C", [(16, (1 << 22) + 777, 66), (1, (1 << 26) + 77, 66)])
def test_linear_cross_entropy_few_float32_rows_in_pieces(n, V, C):
    w = randn(V, C, seed=1) * 0.1
    t = torch.randint(V, (n,), generator=gen(1), device="cuda")
    t[0] = V - 1
    x = randn(n, C, seed=2)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    loss = ops.linear_cross_entropy(*leaves, t, reduction="sum")
    gx, gw = torch.autograd.grad(loss, leaves)
    spans = [slice(v, min(v + (1 << 22), V)) for v in range(0, V, 1 << 22)]
    logits = torch.cat([x.detach().double() @ w.detach()[s].double().t() for s in spans], 1)
    lse = torch.logsumexp(logits, 1)
    assert abs(float(loss.detach()) - float((lse - logits.gather(1, t.unsqueeze(1)).squeeze(1)).sum())) < 1e-4 * n
    p = torch.exp(logits - lse.unsqueeze(1))
    p[torch.arange(n, device="cuda"), t] -= 1
    want = sum(p[:, s] @ w.detach()[s].double() for s in spans)
    # p: a logit is off by at most (C + 4) u |x||w| < 1e-5, its exponential by that part of it; V terms of either sign in float32
    assert float((gx.double() - want).norm() / want.norm()) < 1e-4
    for rows in (slice(0, 100), slice(V - 800, V)):
        want = p[:, rows].t() @ x.detach().double()
        mag = p[:, rows].abs().t() @ x.detach().double().abs()
        assert ((gw[rows].double() - want).abs() <= 4e-5 * mag).all()

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,C", [(300, 200), (5, 200)])
def test_linear_cross_entropy_wide_rows_captured_and_replayed(n, C, dtype):
    x, w, t, _ = ce_case(n, 900, C, dtype, seed=20)
    leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]

    def step(a, b, target):
        loss = ops.linear_cross_entropy(a, b, target)
        return [loss, *torch.autograd.grad(loss, (a, b))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves, t)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*leaves, t)
    for seed in (21, 22, 23):      # another number of kept rows each time
        x2, w2, t2, _ = ce_case(n, 900, C, dtype, ignored=0.1 * (seed - 20), seed=seed)
        with torch.no_grad():
            leaves[0].copy_(x2), leaves[1].copy_(w2), t.copy_(t2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(x2.requires_grad_(), w2.requires_grad_(), t2)):
            assert torch.equal(a, b), seed


def test_act8_dequantize_refuses_what_does_not_fit():
    held = ops.act8_quantize(randn(100, seed=1))
    for bad in (ops.Act8(held.codes, held.scales, (101,), torch.float32), ops.Act8(held.codes, held.scales[:3], (100,), torch.float32),
                ops.Act8(held.codes.float(), held.scales, (100,), torch.float32), ops.Act8(held.codes[::2], held.scales, (50,), torch.float32)):
        with pytest.raises(ops.MvsHipError, match="act8_dequantize"):
            ops.act8_dequantize(bad)
