"""The operators of a mixture of expert blocks whose speed is tracked: layer norm, routing, the experts' products.

A mixture gives every atom (or token) a few of E weight blocks with gates, where the species-block linears of the
model give it the one block of its species.  Three operators, by the field ``kind`` of a case:

  norm    layer_norm(x, weight, bias): y = (x - mean) / sqrt(var + eps) * w + b over the last axis; with ``train`` also
          the gradients of x, w and b.  ``stride`` n: the rows are every n-th one of a larger array (n = 4: the scalar
          component of [atoms, 4, channels] features).
  route   route(logits, k): the k experts of largest logit + bias, ties to the lowest index, expert -1 and gate 0
          where a row has fewer experts whose logit is not -inf; gates from softmax or sigmoid scores, renormalised
          over the chosen or not; with ``groups`` only the ``top_groups`` groups of largest key are open.  The bias
          takes part in the choice only.  With ``train`` also the gradient of the logits.
  linear  expert_linear(x, weight, plan, gates): y[t, m] = sum_j gates[t, j] x[t, m] @ W[experts[t, j]], the plan (slots
          sorted by expert) made in the pass, as every new routing needs one; with ``train`` also the gradients of x,
          W and the gates.  ``comps`` components of a row share its experts (3: the vectors of atoms); ``slice``: x
          is those components of [rows, 4, D] features.

``dtype`` is that of x, the weights and the logits; gates are float32.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


def listed():
    return [
        # norm of the scalar features of the 192-atom water cell, the smallest evaluation in use: launch latency
        dict(name="norm_atoms_192", kind="norm", dtype="f32", rows=192, dim=128, stride=4, train=False),
        # a normalised hidden layer (64 wide) of the radial network on the 16384 x 90 edges of a benchmark chunk
        dict(name="norm_radial_train", kind="norm", dtype="f32", rows=1474560, dim=64, stride=1, train=True),
        # wide rows in half the bits, an uneven number of them
        dict(name="norm_wide_train", kind="norm", dtype="bf16", rows=8191, dim=4096, stride=1, train=True),
        # one trial atom
        dict(name="route_atom", kind="route", dtype="f32", rows=1, experts=8, k=2, scoring="softmax",
             renormalize=True, groups=1, top_groups=1, bias=False, masked=0.0, train=False),
        # every atom of the 500,000-atom alloy, training
        dict(name="route_alloy_train", kind="route", dtype="f32", rows=500000, experts=16, k=2, scoring="softmax",
             renormalize=True, groups=1, top_groups=1, bias=True, masked=0.0, train=True),
        # many experts in groups, sigmoid scores with a balance bias
        dict(name="route_grouped_train", kind="route", dtype="bf16", rows=65536, experts=256, k=8, scoring="sigmoid",
             renormalize=True, groups=8, top_groups=4, bias=True, masked=0.0, train=True),
        # as many experts as elements, some of them closed to some atoms, plain softmax gates
        dict(name="route_masked", kind="route", dtype="f16", rows=98304, experts=89, k=3, scoring="softmax",
             renormalize=False, groups=1, top_groups=1, bias=False, masked=0.1, train=False),
        # one trial atom's scalars through its two blocks
        dict(name="linear_atom", kind="linear", dtype="f32", rows=1, comps=1, slice=False, dim=128, out=128,
             experts=8, k=2, closed=0.0, train=False),
        # inference on the scalars of the 98,304-atom water box
        dict(name="linear_water_98304", kind="linear", dtype="f32", rows=98304, comps=1, slice=True, dim=128, out=128,
             experts=8, k=2, closed=0.0, train=False),
        # training on the vectors of one benchmark chunk of 16384 atoms
        dict(name="linear_vectors_train", kind="linear", dtype="f32", rows=16384, comps=3, slice=True, dim=128,
             out=128, experts=16, k=2, closed=0.0, train=True),
        # wide blocks, many experts, bf16: bound by the matrix cores
        dict(name="linear_wide_train", kind="linear", dtype="bf16", rows=16384, comps=1, slice=False, dim=1024,
             out=1024, experts=64, k=4, closed=0.0, train=True),
        # ragged: as many experts as elements, odd widths, some slots without an expert
        dict(name="linear_ragged_train", kind="linear", dtype="f16", rows=4001, comps=1, slice=False, dim=201,
             out=137, experts=89, k=3, closed=0.1, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "route", "linear", "linear"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.6
    if kind == "norm":
        dim = _log_int(rng, 16, 8192)
        if rng.random() < 0.6:
            dim = 8 * max(1, dim // 8)
        rows = _log_int(rng, 1, min(1500000, 90000000 // dim))
        return dict(kind=kind, dtype=dtype, rows=rows, dim=dim, stride=rng.choice([1, 1, 4]), train=train)
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * max(2, _log_int(rng, 4, 256) // groups)
        k = min(_log_int(rng, 1, 8), experts)
        rows = _log_int(rng, 1, min(500000, 16000000 // experts))
        return dict(kind=kind, dtype=dtype, rows=rows, experts=experts, k=k, scoring=rng.choice(["softmax", "sigmoid"]),
                    renormalize=rng.random() < 0.6, groups=groups, top_groups=max(1, groups // 2),
                    bias=rng.random() < 0.5, masked=rng.choice([0.0, 0.0, 0.1]), train=train)
    dim, out = (_log_int(rng, 32, 1024) for _ in range(2))
    if rng.random() < 0.7:
        dim, out = 8 * (dim // 8), 8 * (out // 8)
    experts, comps = _log_int(rng, 2, 89), rng.choice([1, 1, 3])
    k = min(rng.choice([1, 2, 2, 4]), experts)
    most = min(4e10 / (k * comps * dim * out), 6e7 / (k * comps * max(dim, out)))
    return dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, max(2, min(200000, int(most)))), comps=comps,
                slice=rng.random() < 0.5, dim=dim, out=out, experts=experts, k=k, closed=rng.choice([0.0, 0.0, 0.1]),
                train=train)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    T, train = case["rows"], case["train"]
    if case["kind"] == "norm":
        n = T * case["dim"]
        return {"bytes": (4 if train else 2) * n * es + (4 if train else 2) * case["dim"] * es,
                "flops": (22 if train else 8) * n}
    if case["kind"] == "route":
        n, slots = T * case["experts"], T * case["k"]
        return {"bytes": (2 if train else 1) * n * es + (12 if train else 8) * slots, "flops": 4 * n}
    D, F, S = case["dim"], case["out"], T * case["k"]
    w = min(case["experts"], S) * D * F * es
    b = T * case["comps"] * (D + F) * es + w + 8 * S
    return {"bytes": 2 * b - (4 * S if train else 0) if train else b,
            "flops": (6 if train else 2) * S * case["comps"] * D * F}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def prepare(case, seed):
    gen, dt = _generator(seed), DTYPES[case["dtype"]]
    T, train = case["rows"], case["train"]
    s = {"case": case}
    if case["kind"] == "norm":
        D, n = case["dim"], case["stride"]
        # rows of different scale and offset, as features of different atoms have
        x = _randn(gen, T, n, D) * torch.exp(0.5 * _randn(gen, T, n, 1)) + 0.5 * _randn(gen, T, n, 1)
        s["x"] = x.to(dt)[:, 0, :]
        s["w"], s["b"] = (1 + 0.2 * _randn(gen, D)).to(dt), (0.2 * _randn(gen, D)).to(dt)
        if train:
            s["dy"] = _randn(gen, T, D).to(dt)
            for name in "xwb":
                s[name].requires_grad_()
        return s
    E, k = case["experts"], case["k"]
    if case["kind"] == "route":
        x = 1.5 * _randn(gen, T, E)
        if case["masked"]:
            # single closed experts, and now and then an atom with none open
            shut = torch.rand(T, E, generator=gen, device=DEV) < case["masked"]
            shut |= torch.rand(T, 1, generator=gen, device=DEV) < 0.02
            x = x.masked_fill(shut, -math.inf)
        s["logits"] = x.to(dt)
        s["bias"] = 0.3 * _randn(gen, E) if case["bias"] else None
        if train:
            s["dgates"] = _randn(gen, T, k)
            s["logits"].requires_grad_()
        return s
    D, F, M = case["dim"], case["out"], case["comps"]
    if case["slice"]:
        first = 0 if M == 1 else 1
        s["x"] = _randn(gen, T, 4, D).to(dt)[:, first:first + M, :]
    else:
        s["x"] = _randn(gen, T, M, D).to(dt)
    s["w"] = (_randn(gen, E, D, F) / math.sqrt(D)).to(dt)
    # uneven popularity: k different experts a row, drawn by popularity
    u = torch.rand(T, E, generator=gen, device=DEV).clamp(1e-6, 1 - 1e-6)
    liking = 0.7 * _randn(gen, E) - torch.log(-torch.log(u))
    e = liking.topk(k, 1).indices.to(torch.int32)
    if case["closed"]:
        e = e.masked_fill(torch.rand(T, k, generator=gen, device=DEV) < case["closed"], -1)
    s["experts"] = e
    s["gates"] = torch.softmax(_randn(gen, T, k), 1)
    if train:
        s["dy"] = _randn(gen, T, M, F).to(dt)
        for name in ("x", "w", "gates"):
            s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"norm": _own_norm, "route": _own_route, "linear": _own_linear}[kind](s)
    with torch.no_grad():
        return {"norm": _norm, "route": _route, "linear": _linear}[kind](s)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mace-million_amd")
    if at not in sys.path:
        sys.path.insert(0, at)


def _own_norm(s):
    _package()
    from mace_onegpu.layer_norm import layer_norm
    y = layer_norm(s["x"], s["w"], s["b"], EPS)
    if not s["case"]["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _own_route(s):
    _package()
    from mace_onegpu.experts import route
    c = s["case"]
    gates, experts = route(s["logits"], c["k"], scoring=c["scoring"], bias=s["bias"], groups=c["groups"],
                           top_groups=c["top_groups"], renormalize=c["renormalize"])
    if not c["train"]:
        return {"gates": gates, "experts": experts}
    (dlogits,) = torch.autograd.grad(gates, s["logits"], s["dgates"])
    return {"gates": gates, "experts": experts, "dlogits": dlogits}


def _own_linear(s):
    _package()
    from mace_onegpu.experts import expert_linear, plan_experts
    y = expert_linear(s["x"], s["w"], plan_experts(s["experts"], s["case"]["experts"]), s["gates"])
    if not s["case"]["train"]:
        return {"y": y}
    dx, dw, dgates = torch.autograd.grad(y, (s["x"], s["w"], s["gates"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw, "dgates": dgates}


def _norm(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    xc = x - x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xh = xc * r
    dt = s["x"].dtype
    out = {"y": (xh * w + b).to(dt)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        out.update(dx=dx.to(dt), dw=(dy * xh).sum(0).to(dt), db=dy.sum(0).to(dt))
    return out


def _route(s):
    c = s["case"]
    x = s["logits"].float()
    T, E = x.shape
    k, sigmoid = c["k"], c["scoring"] == "sigmoid"
    # a logit of -inf stays -inf: such experts sort behind every other
    key = x if s["bias"] is None else x + s["bias"]
    if c["groups"] > 1:
        best = key.view(T, c["groups"], -1).amax(2)
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(
            1, torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]], True)
        key = key.view(T, c["groups"], -1).masked_fill(~open_[:, :, None], -math.inf).view(T, E)
    top, chosen = (t[:, :k] for t in torch.sort(key, dim=1, descending=True, stable=True))
    used = top > -math.inf
    xc = x.gather(1, chosen)
    score = torch.minimum(x, torch.zeros_like(x)) - torch.log1p(torch.exp(-x.abs())) if sigmoid else x   # its logarithm
    if c["renormalize"]:
        at = score.gather(1, chosen).masked_fill(~used, -math.inf)
        at = torch.exp(at - at.amax(1, keepdim=True)).masked_fill(~used, 0)
        gates = at / at.sum(1, keepdim=True)
    elif sigmoid:
        gates = 1 / (1 + torch.exp(-xc))
    else:
        p = torch.exp(x - x.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        gates = p.gather(1, chosen)
    gates = torch.where(used, gates, 0.0)
    out = {"gates": gates, "experts": torch.where(used, chosen, -1).to(torch.int32)}
    if c["train"]:
        dg = torch.where(used, s["dgates"], 0.0)
        if c["renormalize"]:
            d = gates * (dg - (gates * dg).sum(1, keepdim=True))
            d = d / (1 + torch.exp(xc)) if sigmoid else d
        elif sigmoid:
            d = dg * gates / (1 + torch.exp(xc))
        else:
            d = gates * dg
        d = torch.zeros_like(x).scatter_(1, chosen, torch.where(used, d, 0.0))
        if not c["renormalize"] and not sigmoid:
            d = d - torch.where(x > -math.inf, p, 0.0) * (gates * dg).sum(1, keepdim=True)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _linear(s):
    """Rows gathered by expert into [E, most rows of one expert], one batched product, and back."""
    x, w, g, e = s["x"].float(), s["w"].float(), s["gates"], s["experts"].reshape(-1)
    dt = s["x"].dtype
    (T, M, D), (E, _, F), k = x.shape, w.shape, g.shape[1]
    key = torch.where(e < 0, E, e).long()
    order = torch.sort(key, stable=True).indices
    order = order[:int((e >= 0).sum())]
    counts = torch.bincount(key, minlength=E + 1)[:E]
    most = max(1, int(counts.max()))
    at = key[order] * most + torch.arange(order.numel(), device=DEV) - (counts.cumsum(0) - counts)[key[order]]
    token, gate = order // k, g.reshape(-1)[order][:, None, None]

    def spread(rows):                                      # [slots, M, n] in expert order -> [E, most M, n]
        out = torch.zeros(E * most, M, rows.shape[2], device=DEV)
        out[at] = rows
        return out.view(E, most * M, rows.shape[2])

    def slots(pad):                                        # and back to [T, k, M, n]
        out = torch.zeros(T * k, M, pad.shape[2], device=DEV)
        out[order] = pad.view(E * most, M, pad.shape[2])[at]
        return out.view(T, k, M, pad.shape[2])

    xs = spread(x[token])
    out = {"y": (slots(torch.bmm(xs, w)) * g[:, :, None, None]).sum(1).to(dt)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        z = slots(torch.bmm(spread(dy[token]), w.transpose(1, 2).contiguous()))
        out["dx"] = (z * g[:, :, None, None]).sum(1).to(dt)
        out["dgates"] = (z * x[:, None]).sum((2, 3))
        out["dw"] = torch.bmm(xs.transpose(1, 2).contiguous(), spread(dy[token] * gate)).to(dt)
    return out


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "route": _exact_route, "linear": _exact_linear}[case["kind"]](s)


def _exact_norm(s):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    xh = (x - mean) * (var + EPS) ** -0.5
    out = {"y": xh * w + b}
    if s["case"]["train"]:
        dy = s["dy"].double()
        n = x.shape[1]
        g = dy * w
        # the Jacobian of the norm applied to g: (n g - sum g - xh sum g xh) / (n sigma)
        out["dx"] = (n * g - g.sum(1, True) - xh * (g * xh).sum(1, True)) / (n * (var + EPS) ** 0.5)
        out["dw"], out["db"] = (dy * xh).sum(0), dy.sum(0)
    return out


def _exact_route(s):
    """The experts as k times the largest remaining key; gates from log scores."""
    c = s["case"]
    x = s["logits"].double()
    T, E = x.shape
    key = s["logits"].float()
    if s["bias"] is not None:
        key = key + s["bias"]                              # the choice is defined by this float32 sum
    rest = key.double()
    G = c["groups"]
    if G > 1:
        best = rest.view(T, G, E // G).max(2).values
        # rank of a group: those with a larger key, and equal ones before it
        ahead = (best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None])
                                                         & torch.ones(G, G, dtype=torch.bool, device=DEV).tril(-1))
        shut = (ahead.sum(2) >= c["top_groups"]).repeat_interleave(E // G, 1)
        rest = torch.where(shut, -math.inf, rest)
    logs = torch.nn.functional.logsigmoid(x) if c["scoring"] == "sigmoid" else x - torch.logsumexp(x, 1, True)
    picked, which, number = [], [], torch.arange(E, device=DEV)
    for _ in range(c["k"]):
        best = rest.max(1, keepdim=True).values
        first = torch.where(rest == best, number, E).min(1, keepdim=True).values.clamp_max(E - 1)
        picked.append(best > -math.inf)
        which.append(first)
        rest = rest.scatter(1, first, -math.inf)
    used, e = torch.cat(picked, 1), torch.cat(which, 1)
    l = torch.where(used, logs.gather(1, e), -math.inf)
    total = torch.logsumexp(l, 1, True) if c["renormalize"] else torch.zeros_like(l[:, :1])
    gates = torch.where(used, torch.exp(l - torch.where(total > -math.inf, total, 0.0)), 0.0)
    out = {"gates": gates, "experts": None}
    if c["train"]:
        dlog = gates * torch.where(used, s["dgates"].double(), 0.0)      # by the log of a chosen score
        whole = dlog.sum(1, True)
        if c["renormalize"]:
            dlog = dlog - gates * whole
        d = torch.zeros_like(x).scatter_add_(1, e, dlog)
        if c["scoring"] == "sigmoid":
            d = d * torch.sigmoid(-x)
        elif not c["renormalize"]:
            d = d - torch.nan_to_num(torch.softmax(x, 1)) * whole
        out["dlogits"] = torch.nan_to_num(d)
    return out


def _exact_linear(s):
    """Expert by expert."""
    x, w, g, e = s["x"].double(), s["w"].double(), s["gates"].double(), s["experts"]
    train = s["case"]["train"]
    y = torch.zeros(x.shape[0], x.shape[1], w.shape[2], dtype=torch.float64, device=DEV)
    if train:
        dy, dx, dw, dg = s["dy"].double(), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(g)
    for i in range(w.shape[0]):
        t, j = (e == i).nonzero(as_tuple=True)
        if not t.numel():
            continue
        xi, gi = x[t], g[t, j][:, None, None]
        y.index_add_(0, t, gi * (xi @ w[i]))
        if train:
            z = dy[t] @ w[i].T.contiguous()
            dx.index_add_(0, t, gi * z)
            dg[t, j] = (xi * z).sum((1, 2))
            dw[i] = (gi * xi).flatten(0, 1).T @ dy[t].flatten(0, 1)
    out = {"y": y}
    if train:
        out.update(dx=dx, dw=dw, dgates=dg)
    return out
