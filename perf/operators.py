"""The training operators that keep no large tensor: what is measured of them, in their plain form and on the kernels.

Three operators, one case each time:
  checkpoint  an activation held in 8 bits for the backward pass (ops.act8_quantize / act8_dequantize), and the BatchNorm + ReLU
              (+ skip) block of the training path that keeps its input so (ops.bn_relu_cl(..., act8=True))
  loss        softmax cross entropy of rows against every row of a large table, without the logits, with both gradients
              (ops.linear_cross_entropy): a language model's head, or points of one view matched against all cells of another
  lookup      rows of a table by index, scaled, and the table's gradient by sorted indices (ops.lookup_rows)

The 8-bit form: blocks of 32 consecutive values share one power of two 2^k, the smallest with round(max|x| / 2^k) <= 127
(k >= -126); a value is round-to-nearest-even(x / 2^k), read back as that whole number times 2^k, at most the type's largest.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
IGNORE = -100


def listed():
    return [
        # one view's feature map of the 640x512 training configuration (32 channels at a quarter of the size)
        dict(name="ckpt-map", op="checkpoint", form="copy", shape="1x128x160x32", type="float32"),
        # an odd number of 16-bit values, the last block a ragged one: a long sequence's hidden states
        dict(name="ckpt-long-bf16", op="checkpoint", form="copy", shape="16385x1031", type="bfloat16"),
        # FeatureNet's full-resolution layers: three views of 640x512, 8 channels, each view with its own statistics
        dict(name="ckpt-bn-views", op="checkpoint", form="block", rows=3 * 512 * 640, channels=8, groups=3, relu=True, skip=False),
        # CostRegNet's full-resolution decoder layer at 640x512 and 192 depth planes, with its skip
        dict(name="ckpt-bn-volume", op="checkpoint", form="block", rows=192 * 128 * 160, channels=8, groups=1, relu=True, skip=True),
        # a single token against a vocabulary: latency, and the table's bytes
        dict(name="loss-one", op="loss", rows=1, classes=32000, width=1024, type="bfloat16", ignored=0.0, sharp=1.0),
        # sparse points of one view against every cell of another view's feature map
        dict(name="loss-points", op="loss", rows=1021, classes=128 * 160, width=32, type="float32", ignored=0.1, sharp=4.0),
        # every cell against every cell: dense matching
        dict(name="loss-dense", op="loss", rows=128 * 160, classes=128 * 160, width=32, type="float32", ignored=0.3, sharp=4.0),
        # an odd vocabulary, a ragged batch
        dict(name="loss-ragged-f16", op="loss", rows=777, classes=49999, width=768, type="float16", ignored=0.25, sharp=1.0),
        # a batch of long sequences against a large vocabulary
        dict(name="loss-large-bf16", op="loss", rows=8192, classes=128000, width=2048, type="bfloat16", ignored=0.05, sharp=1.0),
        # the points' rows of a feature map; several points share a cell
        dict(name="lookup-points", op="lookup", rows=1021, table=128 * 160, width=32, type="float32", spread="flat"),
        # tokens: a few indices make up most of the batch
        dict(name="lookup-tokens", op="lookup", rows=8191, table=32000, width=1024, type="bfloat16", spread="steep"),
        dict(name="lookup-large", op="lookup", rows=65536, table=128000, width=2048, type="bfloat16", spread="steep"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["checkpoint", "checkpoint", "loss", "loss", "lookup"])
    if op == "checkpoint" and rng.random() < 0.5:
        width = rng.choice([8, 32, 64, 1000, 1031, 1024, 4096])
        return dict(op=op, form="copy", shape="%dx%d" % (_log(rng, 1, 33_000_000 // width), width), type=rng.choice(sorted(TYPES)))
    if op == "checkpoint":
        channels, groups = rng.choice([8, 16, 32, 64]), rng.choice([1, 1, 2, 3, 5])
        return dict(op=op, form="block", rows=groups * _log(rng, 64, 31_000_000 // channels // groups), channels=channels, groups=groups,
                    relu=rng.random() < 0.8, skip=rng.random() < 0.5)
    if op == "loss":
        width = rng.choice([8, 32, 33, 64, 100, 256, 512, 768, 1000, 1024, 2048])
        rows, classes = _log(rng, 1, 16384), _log(rng, 16, 131072)
        while rows * classes > 1 << 29:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, classes=classes, width=width, type=rng.choice(sorted(TYPES)), ignored=rng.choice([0.0, 0.1, 0.5]),
                    sharp=rng.choice([1.0, 4.0]))
    width = rng.choice([8, 32, 33, 64, 257, 768, 1024, 2048])
    return dict(op=op, rows=_log(rng, 1, 65536), table=_log(rng, 16, 128000), width=width, type=rng.choice(sorted(TYPES)),
                spread=rng.choice(["flat", "steep"]))


# ------------------------------------------------------------------ inputs
def _dims(case):
    return [int(n) for n in case["shape"].split("x")]


def _off_corner(x, weight, bias, eps):
    """Values whose normalised form lies within rounding of ReLU's corner have either gradient: they are moved off it."""
    var, mean = torch.var_mean(x.double(), 1, correction=0, keepdim=True)
    z = (x - mean) * (weight / torch.sqrt(var + eps)) + bias
    return x + 0.02 * (z.abs() < 2e-5).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    if case["op"] == "checkpoint" and case["form"] == "copy":
        # activations: most near zero, single channels far larger
        shape = _dims(case)
        x = normal(*shape) * torch.exp(normal(shape[-1]))
        return dict(case=case, x=x.to(TYPES[case["type"]]))
    if case["op"] == "checkpoint":
        c, groups = case["channels"], case["groups"]
        bn = torch.nn.BatchNorm2d(c, momentum=1.0).cuda().train()      # (the running statistics are then the last group's own)
        with torch.no_grad():
            bn.weight.copy_(1 + 0.2 * normal(c))
            bn.bias.copy_(0.3 * normal(c))
        x = normal(case["rows"], c) * (0.5 + torch.rand(c, generator=gen, device="cuda")) + normal(c)
        x = x.view(groups, -1, c)
        if case["relu"]:
            x = _off_corner(x, bn.weight.detach().double(), bn.bias.detach().double(), bn.eps)
        skip = normal(*x.shape) if case["skip"] else None
        return dict(case=case, x=x, bn=bn, skip=skip, grad=normal(*x.shape))
    if case["op"] == "loss":
        # rows that lean towards their class's row, as after some training; a share of them carries no target, the first does
        n, v, c = case["rows"], case["classes"], case["width"]
        weight = normal(v, c) / math.sqrt(c)
        target = torch.randint(v, (n,), generator=gen, device="cuda")
        x = (normal(n, c) + weight[target] * (0.6 * math.log(v) / case["sharp"])).to(TYPES[case["type"]])
        target[1:][torch.rand(n, generator=gen, device="cuda")[1:] < case["ignored"]] = IGNORE
        return dict(case=case, x=x, weight=weight.to(TYPES[case["type"]]), target=target, scale=case["sharp"])
    n, v, c = case["rows"], case["table"], case["width"]
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    # flat: every row alike; steep: the i-th most frequent index comes about 1 / i as often as the first
    rank = (u * v).long() if case["spread"] == "flat" else (torch.exp(u * math.log(v + 1)) - 1).long()
    order = torch.randperm(v, generator=gen, device="cuda")
    index = order[rank.clamp(0, v - 1)]
    kind = TYPES[case["type"]]
    return dict(case=case, table=normal(v, c).to(kind), index=index, grad=normal(n, c).to(kind), scale=math.sqrt(c))


# ------------------------------------------------------------------ the plain forms
def _read_back(x):
    """x through the 8-bit form, in 32 bits."""
    flat = x.reshape(-1).float()
    n = flat.numel()
    blocks = torch.zeros((n + 31) // 32 * 32, device=flat.device)
    blocks[:n] = flat
    blocks = blocks.view(-1, 32)
    most = blocks.abs().amax(1, keepdim=True)
    _, exponent = torch.frexp(most)                                    # max|x| = m 2^exponent, m in [0.5, 1)
    power = lambda k: ((k + 127) << 23).view(torch.float32)  # noqa: E731    (2^k, by its bits)
    k = (exponent - 7).clamp(min=-126)
    k = k + (torch.round(most * power(-k)) > 127).int()
    return (torch.round(blocks * power(-k)) * power(k)).view(-1)[:n].view(x.shape)


def _plain_copy(s):
    x = s["x"]
    most = torch.finfo(x.dtype).max
    return _read_back(x).clamp(-most, most).to(x.dtype)


def _plain_block(s):
    x, bn, grad, skip, relu = s["x"], s["bn"], s["grad"], s["skip"], s["case"]["relu"]
    w, b = bn.weight.detach().view(1, 1, -1), bn.bias.detach().view(1, 1, -1)
    n = x.shape[1]
    mean = x.sum(1, keepdim=True, dtype=torch.float64) / n
    var = (x.double() - mean).square().sum(1, keepdim=True) / n
    inv = 1 / torch.sqrt(var + bn.eps)
    z = ((x.double() - mean) * inv * w + b).float()
    y = z.clamp(min=0) if relu else z
    y = y + skip if skip is not None else y
    dz = grad * (z > 0) if relu else grad
    hat = ((_read_back(x).double() - mean) * inv).float()              # the backward pass has the checkpoint only
    db = dz.sum(1, keepdim=True, dtype=torch.float64)
    dw = (dz * hat).sum(1, keepdim=True, dtype=torch.float64)
    dx = ((w * inv).float() * (dz - (db / n).float() - hat * (dw / n).float()))
    out = dict(y=y, dx=dx, dw=dw.sum((0, 1)).float(), db=db.sum((0, 1)).float(), mean=mean[-1, 0].float(), var=(var[-1, 0] * n / max(1, n - 1)).float())
    if skip is not None:
        out["dskip"] = grad
    return out


def _plain_loss(s):
    x, w, t = s["x"].float(), s["weight"].float(), s["target"]
    keep = t != IGNORE
    count = keep.sum()
    at = torch.where(keep, t, 0).unsqueeze(1)
    logits = (x @ w.t()).mul_(s["scale"])
    top = logits.amax(1, keepdim=True)
    own_logit = logits.gather(1, at)
    logits.sub_(top).exp_()
    total = logits.sum(1, keepdim=True)
    row = (torch.log(total) + top - own_logit).squeeze(1)
    loss = (row * keep).sum() / count
    logits.div_(total)
    logits.scatter_add_(1, at, torch.full_like(top, -1.0))
    logits.mul_((keep * (s["scale"] / count.clamp(min=1))).unsqueeze(1))
    return dict(loss=loss, dx=(logits @ w).to(s["x"].dtype), dweight=(logits.t() @ x).to(s["weight"].dtype))


def _plain_lookup(s):
    table, index, grad = s["table"], s["index"], s["grad"]
    rows = (table[index].float() * s["scale"]).to(table.dtype)
    total = torch.zeros(table.shape, device=table.device)
    total.index_add_(0, index, grad.float())
    return dict(rows=rows, dtable=(total * s["scale"]).to(table.dtype))


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "checkpoint":
            return _plain_copy(state) if case["form"] == "copy" else _plain_block(state)
        return _plain_loss(state) if case["op"] == "loss" else _plain_lookup(state)

    from mvs_amd import ops
    if case["op"] == "checkpoint" and case["form"] == "copy":
        return ops.act8_dequantize(ops.act8_quantize(state["x"]))
    if case["op"] == "checkpoint":
        bn, skip = state["bn"], state["skip"]
        leaves = [state["x"].detach().requires_grad_(), bn.weight, bn.bias] + ([skip.detach().requires_grad_()] if skip is not None else [])
        y = ops.bn_relu_cl(leaves[0], bn, relu=case["relu"], skip=leaves[3] if skip is not None else None, groups=case["groups"], act8=True)
        grads = torch.autograd.grad(y, leaves, state["grad"])
        out = dict(y=y.detach(), dx=grads[0], dw=grads[1], db=grads[2], mean=bn.running_mean.clone(), var=bn.running_var.clone())
        if skip is not None:
            out["dskip"] = grads[3]
        return out
    if case["op"] == "loss":
        x, w = state["x"].detach().requires_grad_(), state["weight"].detach().requires_grad_()
        loss = ops.linear_cross_entropy(x, w, state["target"], scale=state["scale"], ignore_index=IGNORE)
        dx, dw = torch.autograd.grad(loss, (x, w))
        return dict(loss=loss.detach(), dx=dx, dweight=dw)
    table = state["table"].detach().requires_grad_()
    rows = ops.lookup_rows(table, state["index"], scale=state["scale"])
    dtable, = torch.autograd.grad(rows, table, state["grad"])
    return dict(rows=rows.detach(), dtable=dtable)


def work(case):
    size = lambda kind: 4 if kind == "float32" else 2  # noqa: E731
    if case["op"] == "checkpoint" and case["form"] == "copy":
        n, e = math.prod(_dims(case)), size(case["type"])
        return dict(bytes=n * (2 * e + 2 + 2 / 32), flops=4 * n)                  # x in, codes out and in, x out
    if case["op"] == "checkpoint":
        n = case["rows"] * case["channels"]
        held = 1 + 1 / 32 + (1 / 8 if case["relu"] else 0)
        # forward: x in, y and the checkpoint out (skip in); backward: dy and the checkpoint in, dx out
        return dict(bytes=n * (8 + 4 * case["skip"] + 8 + 2 * held), flops=30 * n)
    if case["op"] == "loss":
        n, v, c, e = case["rows"], case["classes"], case["width"], size(case["type"])
        return dict(bytes=2 * e * c * (n + v) + 8 * n, flops=6 * max(1, round(n * (1 - case["ignored"]))) * v * c)
    n, v, c, e = case["rows"], case["table"], case["width"], size(case["type"])
    return dict(bytes=e * c * (2 * n + min(n, v) + v) + 16 * n, flops=2 * n * c)


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_read_back(x):
    import numpy as np
    v = x.detach().double().cpu().numpy().reshape(-1)
    n = v.size
    v = np.concatenate([v, np.zeros(-n % 32)]).reshape(-1, 32)
    most = np.abs(v).max(1)
    k = np.full(most.shape, -126.0)
    seen = most > 0
    k[seen] = np.maximum(-126.0, np.ceil(np.log2(most[seen] / 127.5)) - 1)      # at most one too small, or two: raised
    k += np.rint(most / 2.0 ** k) > 127
    k += np.rint(most / 2.0 ** k) > 127
    back = np.rint(v / 2.0 ** k[:, None]) * 2.0 ** k[:, None]
    return torch.from_numpy(back.reshape(-1)[:n]).view(x.shape).to(x.device)


def _exact_block(s):
    bn, x, gy, skip = s["bn"], s["x"].double(), s["grad"].double(), s["skip"]
    w, b, n = bn.weight.detach().double(), bn.bias.detach().double(), s["x"].shape[1]
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    sigma = torch.sqrt(var + bn.eps)
    z = w * (x - mean) / sigma + b
    gz = torch.where(z > 0, gy, torch.zeros_like(gy)) if s["case"]["relu"] else gy
    y = torch.relu(z) if s["case"]["relu"] else z
    hat = (_exact_read_back(s["x"]) - mean) / sigma
    dx = w / sigma * (gz - gz.mean(1, keepdim=True) - hat * (gz * hat).mean(1, keepdim=True))
    out = dict(y=y if skip is None else y + skip.double(), dx=dx, dw=(gz * hat).sum((0, 1)), db=gz.sum((0, 1)), mean=mean[-1, 0], var=var[-1, 0] * n / max(1, n - 1))
    return out if skip is None else dict(out, dskip=gy)


def _exact_loss(s):
    kept = (s["target"] != IGNORE).nonzero().squeeze(1)
    x, w, t = s["x"][kept].double(), s["weight"].double(), s["target"][kept]
    logp = torch.log_softmax(s["scale"] * (x @ w.t()), 1)
    at = torch.arange(len(kept), device=x.device)
    loss = -logp[at, t].sum() / len(kept)
    g = logp.exp_()
    g[at, t] -= 1
    g *= s["scale"] / max(1, len(kept))
    dx = torch.zeros(s["x"].shape, dtype=torch.float64, device=x.device)
    dx[kept] = g @ w
    return dict(loss=loss, dx=dx, dweight=g.t() @ x)


def _exact_lookup(s):
    table, index, grad = s["table"].double(), s["index"], s["grad"].double()
    total = torch.zeros_like(table).index_put_((index,), grad, accumulate=True)
    return dict(rows=s["scale"] * torch.index_select(table, 0, index), dtable=s["scale"] * total)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "checkpoint" and case["form"] == "copy":
        return _exact_read_back(s["x"])
    if case["op"] == "checkpoint":
        return _exact_block(s)
    return _exact_loss(s) if case["op"] == "loss" else _exact_lookup(s)
