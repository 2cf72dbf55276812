"""The operators that train a head on node features whose speed is tracked: linear cross entropy, Newton-Schulz
orthogonalisation, group norm with an activation.

Three operators, by the field ``kind`` of a case:

  loss   linear_cross_entropy(x, weight, targets, reduction): the cross entropy of the logits x @ weight^T, rows whose
         target is -100 left out (``ignored``: their share); with ``train`` also the gradients of x and weight.
  ortho  orthogonalize(m): five Newton-Schulz steps X <- a X + (b A + c A A) X, A = X X^T, from X = m / (|m| + eps), on
         every matrix of a batch: the update of weight blocks by momentum that the Muon optimiser takes.
  group  group_norm(x, groups, weight, bias, activation): mean and variance over the rows of a structure and the
         channels of a group, then an activation; with ``train`` also the gradients of x, weight and bias.  ``structs``
         structures of ``rows`` rows in all: of equal size, or with ``ragged`` of sizes between none and a few times
         the mean, given by offsets, ``tail`` rows behind the last one.  ``stride`` n: the rows are every n-th one of
         a larger array.

``dtype`` is that of x, weight, bias and m; losses are float32.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5                             # of the group norm
NS = (3.4445, -4.7750, 2.0315)         # a, b, c of a Newton-Schulz step
NS_STEPS, NS_EPS = 5, 1e-7
IGNORE = -100


def listed():
    return [
        # the element of one trial atom from its scalars, one class per element: launch latency
        dict(name="loss_atom", kind="loss", dtype="f32", rows=1, dim=128, classes=89, ignored=0.0, reduction="none",
             train=False),
        # one token scored against a large vocabulary of an odd size: the weights are read once
        dict(name="loss_token", kind="loss", dtype="bf16", rows=1, dim=4096, classes=100003, ignored=0.0,
             reduction="none", train=False),
        # masked elements of the 98,304-atom water box recovered from the atoms' scalars: most rows are not asked for
        dict(name="loss_elements_train", kind="loss", dtype="f32", rows=98304, dim=128, classes=89, ignored=0.85,
             reduction="mean", train=True),
        # a batch of 8192 tokens and a vocabulary of 131072: bound by the matrix cores
        dict(name="loss_vocabulary_train", kind="loss", dtype="bf16", rows=8192, dim=2048, classes=131072, ignored=0.0,
             reduction="mean", train=True),
        # ragged: odd sizes, some rows left out, a weight for every row's loss
        dict(name="loss_ragged_train", kind="loss", dtype="f16", rows=3001, dim=777, classes=32003, ignored=0.1,
             reduction="none", train=True),
        # the blocks of one mixture of 8 experts, scalars or vectors
        dict(name="ortho_blocks", kind="ortho", dtype="f32", batch=8, rows=128, cols=128),
        # as many blocks as elements, odd sizes, more rows than columns
        dict(name="ortho_ragged", kind="ortho", dtype="f32", batch=89, rows=201, cols=137),
        # 64 wide expert blocks
        dict(name="ortho_wide", kind="ortho", dtype="bf16", batch=64, rows=1024, cols=1024),
        # one large projection, twice as wide as high
        dict(name="ortho_large", kind="ortho", dtype="bf16", batch=1, rows=4096, cols=8192),
        # scalars of the 192-atom water cell: launch latency
        dict(name="group_atoms_192", kind="group", dtype="f32", structs=1, rows=192, dim=128, groups=8,
             activation="silu", ragged=False, tail=0, stride=4, train=False),
        # a training batch of small molecules
        dict(name="group_molecules_train", kind="group", dtype="f32", structs=4096, rows=90001, dim=128, groups=8,
             activation="silu", ragged=True, tail=100, stride=1, train=True),
        # every atom of the 500,000-atom alloy in one structure
        dict(name="group_alloy_train", kind="group", dtype="bf16", structs=1, rows=500000, dim=128, groups=16,
             activation="gelu", ragged=False, tail=0, stride=1, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dims(rng, lo, hi):
    n = _log_int(rng, lo, hi)
    return 8 * max(1, n // 8) if rng.random() < 0.6 else n


def draw(rng):
    kind = rng.choice(["loss", "ortho", "group"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "loss":
        dim, classes = _dims(rng, 16, 4096), _dims(rng, 8, 131072)
        # of 32-bit rows a tenth of the products
        most = min(98304, 1.07e9 / classes, (2e11 if dtype == "f32" else 2e12) / (dim * classes), 4e8 / dim)
        return dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, max(2, most)), dim=dim, classes=classes,
                    ignored=rng.choice([0.0, 0.0, 0.1, 0.85]), reduction=rng.choice(["mean", "sum", "none"]),
                    train=rng.random() < 0.7)
    if kind == "ortho":
        rows, cols = _dims(rng, 16, 4096), _dims(rng, 16, 4096)
        lo, hi = min(rows, cols), max(rows, cols)
        most = min(89, (4e10 if dtype == "f32" else 1.2e11) / (lo * lo * hi), 8e7 / (lo * hi))
        return dict(kind=kind, dtype=dtype, batch=_log_int(rng, 1, max(2, most)), rows=rows, cols=cols)
    groups = rng.choice([1, 2, 4, 8, 16, 32])
    dim = groups * max(1, _log_int(rng, 16, 2048) // groups)
    rows = _log_int(rng, 1, min(500000, 64000000 // dim))
    structs = _log_int(rng, 1, min(rows, 8192))
    ragged = rng.random() < 0.5
    if not ragged:
        rows = structs * (rows // structs)
    return dict(kind=kind, dtype=dtype, structs=structs, rows=rows, dim=dim, groups=groups,
                activation=rng.choice(["none", "silu", "gelu"]), ragged=ragged,
                tail=rng.choice([0, 0, 17]) if ragged else 0, stride=rng.choice([1, 1, 4]), train=rng.random() < 0.6)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "loss":
        T, D, V, train = case["rows"], case["dim"], case["classes"], case["train"]
        asked = max(1, round(T * (1 - case["ignored"])))
        loss = 4 * (T if case["reduction"] == "none" else 1)
        return {"bytes": ((asked + V) * D + ((T + V) * D if train else 0)) * es + 8 * T + loss,
                "flops": (6 if train else 2) * asked * D * V}
    if case["kind"] == "ortho":
        m, n = sorted((case["rows"], case["cols"]))
        # A and A A are symmetric: half of each
        return {"bytes": 2 * case["batch"] * m * n * es,
                "flops": NS_STEPS * case["batch"] * (m * m * n + m * m * m + 2 * m * m * n)}
    n, train = case["rows"] * case["dim"], case["train"]
    return {"bytes": (4 if train else 2) * (n + case["dim"]) * es, "flops": (40 if train else 12) * n}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device=DEV)


def prepare(case, seed):
    s = {"case": case}
    {"loss": _inputs_loss, "ortho": _inputs_ortho, "group": _inputs_group}[case["kind"]](s, case, _generator(seed))
    return s


def _inputs_loss(s, case, gen):
    T, D, V, dt = case["rows"], case["dim"], case["classes"], DTYPES[case["dtype"]]
    w = 2 / math.sqrt(D) * _randn(gen, V, D)
    # uneven classes, and rows between unsure and certain of theirs
    y = torch.minimum((V * _rand(gen, T) ** 3).long(), torch.tensor(V - 1, device=DEV))
    s["x"] = (_randn(gen, T, D) + 3 * _rand(gen, T, 1) * w[y]).to(dt)
    s["w"] = w.to(dt)
    s["targets"] = y.masked_fill(_rand(gen, T) < case["ignored"], IGNORE)
    if case["train"]:
        # the gradient that comes in: of the mean 1, of rows a weight each
        s["dloss"] = 0.1 + _rand(gen, T) if case["reduction"] == "none" else torch.ones((), device=DEV)
        s["x"].requires_grad_()
        s["w"].requires_grad_()


def _inputs_ortho(s, case, gen):
    # a gradient: a few strong directions over a weak rest
    E, m, n = case["batch"], case["rows"], case["cols"]
    r = max(1, min(m, n) // 8)
    strong = torch.bmm(_randn(gen, E, m, r) * torch.exp(_randn(gen, E, 1, r)), _randn(gen, E, r, n)) / math.sqrt(r)
    s["m"] = (0.01 * (strong + 0.3 * _randn(gen, E, m, n))).to(DTYPES[case["dtype"]])


def _inputs_group(s, case, gen):
    T, C, S, dt = case["rows"], case["dim"], case["structs"], DTYPES[case["dtype"]]
    shape = (T + case["tail"],) if case["ragged"] else (S, T // S)
    # rows of different scale and offset, as features of different atoms have
    x = _randn(gen, *shape, case["stride"], C) * torch.exp(0.5 * _randn(gen, *shape, case["stride"], 1))
    s["x"] = (x + 0.5 * _randn(gen, *shape, case["stride"], 1)).to(dt)[..., 0, :]
    s["w"], s["b"] = (1 + 0.2 * _randn(gen, C)).to(dt), (0.2 * _randn(gen, C)).to(dt)
    s["offsets"] = None
    if case["ragged"]:
        cuts = torch.sort((_rand(gen, S - 1) * (T + 1)).int()).values
        zero = torch.zeros(1, dtype=torch.int32, device=DEV)
        s["offsets"] = torch.cat([zero, cuts, zero + T])
    if case["train"]:
        s["dy"] = _randn(gen, *shape, C).to(dt)
        for name in "xwb":
            s[name].requires_grad_()


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"loss": _own_loss, "ortho": _own_ortho, "group": _own_group}[kind](s)
    with torch.no_grad():
        return {"loss": _loss, "ortho": _ortho, "group": _group}[kind](s)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mace-million_amd")
    if at not in sys.path:
        sys.path.insert(0, at)


def _own_loss(s):
    _package()
    from mace_onegpu.cross_entropy import linear_cross_entropy
    loss = linear_cross_entropy(s["x"], s["w"], s["targets"], ignore_index=IGNORE, reduction=s["case"]["reduction"])
    if not s["case"]["train"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), s["dloss"])
    return {"loss": loss, "dx": dx, "dw": dw}


def _own_ortho(s):
    _package()
    from mace_onegpu.muon import orthogonalize
    return {"x": orthogonalize(s["m"], steps=NS_STEPS, coefficients=NS, eps=NS_EPS)}


def _own_group(s):
    _package()
    from mace_onegpu.group_norm import group_norm
    c = s["case"]
    y = group_norm(s["x"], c["groups"], s["w"], s["b"], EPS, activation=None if c["activation"] == "none" else
                   c["activation"], offsets=s["offsets"])
    if not c["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _loss(s):
    c, y = s["case"], s["targets"]
    x, w = s["x"].float(), s["w"].float()
    asked = y != IGNORE
    at = torch.where(asked, y, 0)[:, None]
    logits = torch.mm(x, w.t())
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at)
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    loss = torch.where(asked, (top + torch.log(total) - picked).squeeze(1), 0.0)
    count = asked.sum().clamp_min(1)
    out = {"loss": loss if c["reduction"] == "none" else loss.sum() / (count if c["reduction"] == "mean" else 1)}
    if c["train"]:
        g = torch.where(asked, s["dloss"] / (count if c["reduction"] == "mean" else 1), 0.0)[:, None]
        d = p.mul_(g / total).scatter_add_(1, at, -g)
        dt = s["x"].dtype
        out.update(dx=torch.mm(d, w).to(dt), dw=torch.mm(d.t(), x).to(dt))
    return out


def _ortho(s):
    m = s["m"].float()
    a, b, c = NS
    tall = m.shape[1] > m.shape[2]
    x = m.transpose(1, 2).contiguous() if tall else m
    x = x / (torch.sqrt((x.double() ** 2).sum((1, 2), keepdim=True)).float() + NS_EPS)
    for _ in range(NS_STEPS):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return {"x": (x.transpose(1, 2) if tall else x).to(s["m"].dtype).contiguous()}


def _act(z, kind):
    """(act(z), act'(z))"""
    if kind == "silu":
        q = 1 / (1 + torch.exp(-z))
        return z * q, q * (1 + z * (1 - q))
    if kind == "gelu":
        q = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * q, q + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def _group(s):
    c, dt = s["case"], s["x"].dtype
    C, G, S = c["dim"], c["groups"], c["structs"]
    x = s["x"].float().reshape(-1, G, C // G)
    w, b = s["w"].float().view(G, -1), s["b"].float().view(G, -1)
    T = x.shape[0]
    if c["ragged"]:
        # sums over structures of any size, in 64 bits
        row = torch.arange(T, device=DEV)
        of = torch.searchsorted(s["offsets"].long(), row, right=True) - 1
        inside = (of < S).view(T, 1, 1)
        of = of.clamp_max(S - 1)
        n = (s["offsets"][1:] - s["offsets"][:-1]).clamp_min(1).view(S, 1, 1) * (C // G)

        def mean(v):
            rows = torch.where(inside, v.sum(2, keepdim=True), 0.0).double()
            return (torch.zeros(S, G, 1, dtype=torch.float64, device=DEV).index_add_(0, of, rows) / n).float()[of]
    else:
        inside = torch.ones(1, 1, 1, dtype=torch.bool, device=DEV)

        def mean(v):
            m = v.view(S, T // S, G, C // G).mean((1, 3), keepdim=True)
            return m.expand(S, T // S, G, 1).reshape(T, G, 1)
    xc = x - mean(x)
    r = 1 / torch.sqrt(mean(xc * xc) + EPS)
    h = xc * r
    y, slope = _act(h * w + b, c["activation"])
    shape = s["x"].shape
    out = {"y": torch.where(inside, y, 0.0).to(dt).view(shape)}
    if c["train"]:
        dz = torch.where(inside, s["dy"].float().view(x.shape) * slope, 0.0)
        g = dz * w
        dx = r * (g - mean(g) - h * mean(g * h))
        out.update(dx=torch.where(inside, dx, 0.0).to(dt).view(shape),
                   dw=torch.where(inside, dz * h, 0.0).sum(0).view(C).to(dt), db=dz.sum(0).view(C).to(dt))
    return out


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"loss": _exact_loss, "ortho": _exact_ortho, "group": _exact_group}[case["kind"]](s)


def _exact_loss(s):
    """Blocks of rows, from log probabilities."""
    c, y = s["case"], s["targets"]
    w = s["w"].double()
    asked = (y != IGNORE).double()
    weight = asked / asked.sum().clamp_min(1) if c["reduction"] == "mean" else asked
    T, V = y.shape[0], w.shape[0]
    losses, dx, dw = [], [], torch.zeros_like(w)
    step = max(1, 200000000 // V)
    for i in range(0, T, step):
        x, yi = s["x"][i:i + step].double(), y[i:i + step].clamp_min(0)
        logp = torch.log_softmax(torch.mm(x, w.t().contiguous()), 1)
        losses.append(-logp[torch.arange(yi.numel(), device=DEV), yi] * asked[i:i + step])
        if c["train"]:
            one = torch.nn.functional.one_hot(yi, V)
            d = torch.exp(logp)
            d -= one
            del one, logp
            d *= (weight * s["dloss"].double())[i:i + step, None]
            dx.append(torch.mm(d, w))
            dw += torch.mm(d.t().contiguous(), x)
    loss = torch.cat(losses)
    out = {"loss": loss if c["reduction"] == "none" else (loss * weight).sum()}
    if c["train"]:
        out.update(dx=torch.cat(dx), dw=dw)
    return out


def _exact_ortho(s):
    """Row by row of the batch, the polynomial on the other side: Y <- Y (a + G (b + c G)), G = Y^T Y."""
    out = []
    a, b, c = NS
    for m in s["m"].double():
        wide = m.shape[1] > m.shape[0]
        y = m.t().contiguous() if wide else m
        y = y / (torch.linalg.matrix_norm(y) + NS_EPS)
        one = torch.eye(y.shape[1], dtype=torch.float64, device=DEV)
        for _ in range(NS_STEPS):
            gram = torch.mm(y.t().contiguous(), y)
            y = torch.mm(y, a * one + torch.mm(gram, b * one + c * gram))
        out.append(y.t() if wide else y)
    return {"x": torch.stack(out)}


def _exact_group(s):
    """Normalised rows by structure; gradients by the chain rule of mean and deviation."""
    c = s["case"]
    C, G, S = c["dim"], c["groups"], c["structs"]
    x = s["x"].double().reshape(-1, C)
    T = x.shape[0]
    if s["offsets"] is None:
        bounds = torch.arange(S + 1, device=DEV) * (T // S)
    else:
        bounds = s["offsets"].long()
    sizes = bounds[1:] - bounds[:-1]
    of = torch.repeat_interleave(torch.arange(S, device=DEV), sizes)
    t0, t1 = int(bounds[0]), int(bounds[-1])
    n = (sizes * (C // G)).clamp_min(1).double()[:, None].expand(S, G)

    def sums(v):                                           # [rows, C] -> [S, G]
        v = v.view(-1, G, C // G).sum(2)
        total = torch.cat([torch.zeros(1, G, dtype=torch.float64, device=DEV), v.cumsum(0)])
        return total[bounds[1:] - t0] - total[bounds[:-1] - t0]

    def spread(v):                                         # [S, G] -> [rows, C]
        return v[of].repeat_interleave(C // G, 1)

    xi, w, b = x[t0:t1], s["w"].double(), s["b"].double()
    centred = xi - spread(sums(xi) / n)
    sigma = torch.sqrt(sums(centred.square()) / n + EPS)
    h = centred / spread(sigma)
    z = h * w + b
    kind = c["activation"]
    if kind == "silu":
        q = torch.sigmoid(z)
        y, slope = z * q, q + z * q * torch.sigmoid(-z)
    elif kind == "gelu":
        q = torch.special.ndtr(z)
        y, slope = z * q, q + z * torch.exp(-z.square() / 2) * 0.3989422804014327
    else:
        y, slope = z, torch.ones_like(z)

    def whole(v):
        out = torch.zeros_like(x)
        out[t0:t1] = v
        return out.view(s["x"].shape)

    out = {"y": whole(y)}
    if c["train"]:
        dz = s["dy"].double().reshape(-1, C)[t0:t1] * slope
        dh = dz * w
        dx = (spread(n) * dh - spread(sums(dh)) - h * spread(sums(dh * h))) / spread(n * sigma)
        out.update(dx=whole(dx), dw=(dz * h).sum(0), db=dz.sum(0))
    return out
