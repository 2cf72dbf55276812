"""plan_experts against a stable sort (exact), and expert_linear with its gradients against plain sums in 64 bits.

Tolerances, element by element: a sum of n products in float32 is off by at most (n + 16) u sum |terms|, u = 2^-24 (16
for the gate, the joining of the k slots, and products of split operands, 3 u each); rounding to the output's type adds
half a unit in its last place, and dW of 16-bit types may round gate x dy to that type before the product: one more
half unit of the sum of magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


# ------------------------------------------------------------------------------------------------ plan
@pytest.mark.parametrize("E", [1, 2, 64, 89, 512, 513, 1024])
@pytest.mark.parametrize("T,k", [(0, 2), (1, 1), (1, 8), (63, 1), (65, 2), (2048, 2), (2049, 2), (8192, 2), (5462, 3),
                                 (70001, 4)])
def test_plan_is_a_stable_sort(T, k, E):
    from mace_onegpu.experts import plan_experts
    g = torch.Generator().manual_seed(T + E)
    e = torch.randint(-1, E + (E > 1), (T, k), generator=g, dtype=torch.int32)      # -1 and E: no expert
    for experts in (e, torch.full_like(e, E - 1), e.long() * 2 ** 32 + e.long()):
        plan = plan_experts(experts.cuda(), E)
        flat = experts.reshape(-1).long()
        valid = (flat >= 0) & (flat < E)
        keys = torch.where(valid, flat, E)
        n = int(valid.sum())
        counts = torch.bincount(keys, minlength=E + 1)[:E]
        offsets = torch.zeros(E + 1, dtype=torch.int64)
        offsets[1:] = counts.cumsum(0)
        assert torch.equal(plan.offsets.cpu().long(), offsets)
        assert torch.equal(plan.counts.cpu().long(), counts)
        assert torch.equal(plan.order[:n].cpu().long(), torch.sort(keys, stable=True).indices[:n])


@pytest.mark.parametrize("T,k,E", [(700001, 4, 8), (300000, 1, 1024), (1500000, 2, 64)])
def test_plan_of_long_lists(T, k, E):
    """Lists whose tiles' counts are summed by a launch of their own, against a stable sort on the GPU."""
    from mace_onegpu.experts import plan_experts
    g = torch.Generator(device="cuda").manual_seed(T)
    e = torch.randint(-1, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    plan = plan_experts(e, E)
    keys = torch.where(e < 0, E, e).reshape(-1)
    counts = torch.bincount(keys, minlength=E + 1)
    assert torch.equal(plan.counts.long(), counts[:E]) and int(plan.offsets[-1]) == int(counts[:E].sum())
    n = int(plan.offsets[-1])
    assert torch.equal(plan.order[:n].long(), torch.sort(keys, stable=True).indices[:n])


# ------------------------------------------------------------------------------------------------ products
def _reference(x, w, experts, gates, dy):
    """(results, sums of magnitudes) of [T, M, D] inputs, 64 bits."""
    x, w, dy = x.double(), w.double(), dy.double()
    T, M, D = x.shape
    E, _, F = w.shape
    k = experts.shape[1]
    gates = torch.ones(T, k, dtype=torch.float64) if gates is None else gates.double()
    out = dict(y=torch.zeros(T, M, F, dtype=torch.float64), dx=torch.zeros_like(x), dw=torch.zeros_like(w),
               dg=torch.zeros(T, k, dtype=torch.float64))
    mag = {n: torch.zeros_like(t) for n, t in out.items()}
    for e in range(E):
        t, j = ((experts == e).nonzero(as_tuple=True))
        if not t.numel():
            continue
        g = gates[t, j][:, None, None]
        for o, a, b, c, v in ((out, x, w[e], dy, g), (mag, x.abs(), w[e].abs(), dy.abs(), g.abs())):
            o["y"].index_add_(0, t, v * (a[t] @ b))
            z = c[t] @ b.T
            o["dx"].index_add_(0, t, v * z)
            o["dg"][t, j] = (a[t] * z).sum((1, 2))
            o["dw"][e] = torch.einsum("tmd,tmf->df", v * a[t], c[t])
    return out, mag


def _make(T, M, D, F, E, k, dtype, seed, closed=0.0, unused=()):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, M, D, generator=g).to(dtype)
    w = (torch.randn(E, D, F, generator=g) / D ** 0.5).to(dtype)
    score = torch.rand(T, E, generator=g)
    score[:, list(unused)] = -1
    experts = score.topk(k, 1).indices.to(torch.int32)
    experts[torch.rand(T, k, generator=g) < closed] = -1
    gates = torch.softmax(torch.randn(T, k, generator=g), 1)
    dy = torch.randn(T, M, F, generator=g).to(dtype)
    return x, w, experts, gates, dy


def _check(got, ref, mag, terms, dtype):
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    for name, t in got.items():
        out = torch.float32 if name == "dg" else dtype
        bound = (terms[name] + 16) * U * mag[name] + HALF_ULP[out] * ref[name].abs() + tiny
        if name == "dw" and dtype != torch.float32:
            bound = bound + HALF_ULP[dtype] * mag[name]
        err = (t.detach().double().cpu().view(ref[name].shape) - ref[name]).abs()
        assert t.dtype == out and bool((err <= bound).all()), (name, float((err - bound).max()), float(err.max()))


def _run_and_check(x, w, experts, gates, dy, dtype, view=None):
    from mace_onegpu.experts import expert_linear, plan_experts
    T, M, D = x.shape
    E, _, F = w.shape
    ref, mag = _reference(x, w, experts, gates, dy)
    xg, wg = (view(x) if view else x.cuda()).requires_grad_(), w.cuda().requires_grad_()
    gg = gates.cuda().requires_grad_() if gates is not None else None
    plan = plan_experts(experts.cuda(), E)
    y = expert_linear(xg, wg, plan, gg)
    inputs = [t for t in (xg, wg, gg) if t is not None]
    grads = torch.autograd.grad(y, inputs, dy.cuda())
    got = dict(zip(("y", "dx", "dw", "dg"), (y,) + grads))
    counts = int(plan.counts.max()) if T else 0
    terms = dict(y=D, dx=F, dg=F + M * D, dw=counts * M)
    _check(got, ref, mag, terms, dtype)
    with torch.no_grad():
        assert torch.equal(expert_linear(xg, wg, plan, gg), y)
    again = torch.autograd.grad(expert_linear(xg, wg, plan, gg), inputs, dy.cuda())
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,M,D,F,E,k", [
    (1, 1, 128, 128, 8, 2), (1, 3, 64, 32, 4, 4), (5, 1, 1, 1, 2, 1), (3, 1, 7, 513, 3, 2), (2, 1, 1000, 24, 5, 1),
    (17, 1, 130, 66, 3, 2), (64, 1, 128, 128, 1, 1), (65, 3, 128, 128, 4, 2), (200, 5, 33, 47, 7, 3),
    (300, 1, 256, 192, 16, 4), (129, 2, 201, 137, 89, 3), (1000, 1, 64, 128, 2, 2), (513, 1, 320, 264, 6, 2),
    (2500, 1, 40, 72, 5, 1), (40, 1, 1024, 512, 3, 2)])
def test_products_and_gradients(T, M, D, F, E, k, dtype):
    _run_and_check(*_make(T, M, D, F, E, k, dtype, T + D + F), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k", [(9, 3), (400, 2)])
def test_slots_and_experts_without_partner(T, k, dtype):
    """Slots without an expert, rows without any, experts without rows; their outputs and gradients are 0, not stale."""
    x, w, experts, gates, dy = _make(T, 2, 72, 56, 9, k, dtype, 11, closed=0.3, unused=(0, 4, 8))
    experts[2] = -1
    experts[5] = 9
    _run_and_check(x, w, experts, gates, dy, dtype)
    experts[:] = -1
    _run_and_check(x, w, experts, gates, dy, dtype)


@pytest.mark.parametrize("T", [6, 300])
def test_without_gates_and_repeated_experts(T):
    x, w, experts, gates, dy = _make(T, 1, 64, 64, 4, 3, torch.float32, 12)
    _run_and_check(x, w, experts, None, dy, torch.float32)
    experts[:, 1] = experts[:, 0]                   # a row may name one expert twice
    ref, mag = _reference(x, w, experts, gates, dy)
    from mace_onegpu.experts import expert_linear, plan_experts
    y = expert_linear(x.cuda(), w.cuda(), plan_experts(experts.cuda(), 4), gates.cuda())
    _check(dict(y=y), ref, mag, dict(y=64), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [3, 150])
def test_strided_rows(T, dtype):
    """Components 1 .. 3 of ir_mul features in place, rows off any 16-byte boundary, and a transposed x."""
    x, w, experts, gates, dy = _make(T, 3, 128, 128, 4, 2, dtype, 13)

    def slice_of_features(t):
        whole = torch.randn(T, 4, 128).to(dtype).cuda()
        whole[:, 1:] = t.cuda()
        return whole[:, 1:]

    def off_by_one(t):
        whole = torch.zeros(T, 3, 131, dtype=dtype, device="cuda")
        whole[:, :, 1:129] = t.cuda()
        return whole[:, :, 1:129]

    def transposed(t):
        return t.cuda().permute(2, 1, 0).contiguous().permute(2, 1, 0)

    for view in (slice_of_features, off_by_one, transposed):
        _run_and_check(x, w, experts, gates, dy, dtype, view)


def test_two_axes_no_rows_and_expanded_cotangent():
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, experts, gates, dy = (t.cuda() for t in _make(77, 1, 64, 48, 4, 2, torch.float32, 14))
    plan = plan_experts(experts, 4)
    assert torch.equal(expert_linear(x[:, 0], w, plan, gates), expert_linear(x, w, plan, gates)[:, 0])
    xg = x[:, 0].detach().requires_grad_()
    (a,) = torch.autograd.grad(expert_linear(xg, w, plan, gates).sum(), xg)
    (b,) = torch.autograd.grad(expert_linear(xg, w, plan, gates), xg, torch.ones(77, 48, device="cuda"))
    assert torch.equal(a, b)
    none = plan_experts(experts[:0], 4)
    x0, w0 = x[:0].detach().requires_grad_(), w.detach().requires_grad_()
    y = expert_linear(x0, w0, none, gates[:0])
    dx, dw = torch.autograd.grad(y, (x0, w0), torch.empty(0, 1, 48, device="cuda"))
    assert y.shape == (0, 1, 48) and dx.shape == (0, 1, 64) and not dw.any()


@pytest.mark.parametrize("T", [4, 90])
def test_gradient_against_differences(T):
    """The product is linear in each input: one difference with a step of any size is the derivative up to roundings."""
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, experts, gates, dy = (t.cuda() for t in _make(T, 2, 96, 80, 5, 2, torch.float32, 15))
    plan = plan_experts(experts, 5)
    args = [t.requires_grad_() for t in (x, w, gates)]
    f = lambda *a: float((expert_linear(a[0], a[1], plan, a[2]).detach().double() * dy.double()).sum())  # noqa: E731
    grads = torch.autograd.grad(expert_linear(x, w, plan, gates), args, dy)
    g = torch.Generator().manual_seed(1)
    for i in range(3):
        v = torch.randn(args[i].shape, generator=g).cuda()
        slope = (f(*[a + v if q == i else a for q, a in enumerate(args)])
                 - f(*[a - v if q == i else a for q, a in enumerate(args)])) / 2
        terms = (grads[i].double() * v.double())
        assert abs(slope - float(terms.sum())) < 1e-4 * float(terms.abs().sum())


def test_large_rows_and_many_experts():
    """Rows beyond one tile of every variant, uneven load; against 64-bit products on the GPU."""
    from mace_onegpu.experts import expert_linear, plan_experts
    for dtype in DTYPES:
        x, w, experts, gates, dy = _make(20011, 1, 128, 128, 8, 2, dtype, 16)
        experts[:12000, 0] = 3
        experts[:12000, 1] = 5
        _run_and_check(x, w, experts, gates, dy, dtype)


def test_graph_replay():
    from mace_onegpu.experts import expert_linear, plan_experts, route
    g = torch.Generator().manual_seed(5)
    w = torch.randn(8, 128, 128, generator=g).cuda()
    for T in (1, 500):
        x, logits = torch.randn(T, 128, generator=g).cuda(), torch.randn(T, 8, generator=g).cuda()

        def step():
            gates, experts = route(logits, 2)
            return expert_linear(x, w, plan_experts(experts, 8), gates)
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step()
        for _ in range(3):
            x.copy_(torch.randn(T, 128, generator=g))
            logits.copy_(torch.randn(T, 8, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, step())


# ------------------------------------------------------------------------------------------------ the variants
def _rows_reference(x, w, experts, k, transposed):
    """[S, M, N] products of every slot, 64 bits (zeros without an expert), and sums of magnitudes."""
    T, M, K = x.shape
    E = w.shape[0]
    N = w.shape[1] if transposed else w.shape[2]
    out = torch.zeros(T * k, M, N, dtype=torch.float64)
    mag = torch.zeros_like(out)
    flat, xd, wd = experts.reshape(-1), x.double(), w.double()
    for e in range(E):
        s = (flat == e).nonzero()[:, 0]
        b = wd[e].T if transposed else wd[e]
        out[s] = xd[s // k] @ b
        mag[s] = xd[s // k].abs() @ b.abs()
    return out, mag


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("transposed", [0, 1])
@pytest.mark.parametrize("T,M,K,N,E,k,off", [
    (1, 1, 1, 1, 1, 1, 0), (3, 2, 31, 33, 2, 2, 0), (130, 1, 64, 128, 2, 1, 0), (70, 3, 72, 136, 3, 2, 0),
    (257, 1, 129, 257, 2, 1, 0), (200, 1, 200, 40, 70, 3, 0), (90, 1, 64, 64, 5, 2, 1), (2100, 1, 136, 264, 2, 1, 0),
    (1500, 1, 512, 520, 2, 2, 0)])
def test_rows_of_slots(T, M, K, N, E, k, off, transposed, dtype):
    """mm_expert_rows on its own: tiles of both sizes, cut tiles, odd widths, unaligned rows, slots without an
    expert."""
    from mace_onegpu._lib import K as L, stream
    from mace_onegpu.experts import plan_experts
    g = torch.Generator().manual_seed(T + K + N)
    x = torch.randn(T, M, K, generator=g).to(dtype)
    w = torch.randn(*((E, N, K) if transposed else (E, K, N)), generator=g).to(dtype)
    experts = torch.randint(-1 if T > 1 else 0, E, (T, k), generator=g, dtype=torch.int32)
    wide = torch.zeros(T, M, K + 3 * off, dtype=dtype, device="cuda")
    wide[:, :, off:off + K] = x.cuda()
    xg = wide[:, :, off:off + K]
    plan = plan_experts(experts.cuda(), E)
    out = torch.full((T * k, M, N), 7.0, device="cuda")
    L.mm_expert_rows(xg, xg.stride(0), xg.stride(1), DTYPES.index(dtype), T * k, k, M, K, N, w.cuda(), transposed, E,
                     plan.offsets, plan.order, out, stream())
    ref, mag = _rows_reference(x, w, experts, k, transposed)
    used = (experts.reshape(-1) >= 0)
    err = (out.cpu().double() - ref).abs()
    assert bool((err[used] <= ((K + 16) * U * mag + 1e-37)[used]).all())
    assert bool((out.cpu()[~used] == 7.0).all())                      # rows of no expert are left alone


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("transposed", [0, 1])
@pytest.mark.parametrize("T,M,K,N,E,k,off", [
    (1, 1, 3, 5, 1, 1, 0), (300, 1, 64, 128, 3, 1, 0), (300, 3, 72, 136, 3, 2, 0), (77, 5, 33, 201, 2, 2, 0),
    (1000, 1, 128, 128, 21, 2, 0), (3000, 3, 128, 128, 2, 2, 0),
    (5000, 1, 32, 128, 3, 2, 0), (2500, 2, 100, 60, 2, 2, 1), (129, 64, 40, 24, 2, 1, 0), (400, 1, 200, 260, 4, 2, 1),
    (2000, 1, 128, 64, 4, 2, 0)])
def test_joined_rows(T, M, K, N, E, k, off, transposed, dtype):
    """mm_expert_joined on its own: pairs of different and equal experts, one or no expert, and dgates of one choice."""
    import ctypes

    from mace_onegpu._lib import K as L, stream
    from mace_onegpu.experts import plan_experts
    g = torch.Generator().manual_seed(T + K + N)
    x = torch.randn(T, M, K, generator=g).to(dtype)
    w = torch.randn(*((E, N, K) if transposed else (E, K, N)), generator=g).to(dtype)
    experts = torch.randint(-1, E + 1, (T, k), generator=g, dtype=torch.int32)
    gates = torch.randn(T, k, generator=g)
    wide = torch.zeros(T, M, K + 3 * off, dtype=dtype, device="cuda")
    wide[:, :, off:off + K] = x.cuda()
    xg, code = wide[:, :, off:off + K], DTYPES.index(dtype)
    if k == 1:
        plan = plan_experts(experts.cuda(), E)
        offsets, order = plan.offsets, plan.order
    else:
        pairs = (E + 1) * (E + 2) // 2
        n = ctypes.c_long(0)
        L.mm_expert_plan_scratch(T, pairs - 1, ctypes.byref(n))
        offsets = torch.empty(pairs, dtype=torch.int32, device="cuda")
        order = torch.empty(T, dtype=torch.int32, device="cuda")
        L.mm_expert_plan_pairs(experts.cuda(), T, E, offsets, order, torch.empty(n.value + 1, dtype=torch.int32,
                                                                                  device="cuda"), stream())
        clean = torch.where((experts < 0) | (experts >= E), E, experts).sort(1).values.long()
        ids = [(a, b) for a in range(E + 1) for b in range(a, E + 1)]
        key = torch.tensor([ids.index(tuple(p)) for p in clean.tolist()])
        assert torch.equal(order.cpu().long(), torch.sort(key, stable=True).indices)
        first = torch.bincount(key, minlength=pairs).cumsum(0) - torch.bincount(key, minlength=pairs)
        assert torch.equal(offsets.cpu().long(), first)
    z, mag = (t.view(T, k, M, N) for t in _rows_reference(x, w, torch.where(experts >= E, -1, experts), k, transposed))
    ref, bound = (z * gates.double()[:, :, None, None]).sum(1), (mag * gates.double().abs()[:, :, None, None]).sum(1)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    out = torch.full((T, M, N), 7.0, device="cuda").to(dtype)
    with_dg = transposed and N <= 128 and (k == 1 or (dtype == torch.float32 and K <= 128 and M <= 16))
    xs = torch.randn(T, M, N, generator=g).to(dtype)
    dg = torch.full((T, k), 7.0, device="cuda") if with_dg else None
    xsg = xs.cuda()
    L.mm_expert_joined(xg, xg.stride(0), xg.stride(1), code, T, k, M, K, N, w.cuda(), transposed, E, gates.cuda(),
                       experts.cuda(), offsets, order, out, xsg, M * N, N, dg, stream())
    err = (out.cpu().double() - ref).abs()
    assert bool((err <= (K + 16) * U * bound + HALF_ULP[dtype] * ref.abs() + tiny).all()), float(err.max())
    if with_dg:
        want, most = (z * xs.double()[:, None]).sum((2, 3)), (mag * xs.double().abs()[:, None]).sum((2, 3))
        assert bool(((dg.cpu().double() - want).abs() <= (K + M * N + 16) * U * most + 1e-37).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,F,E,k", [(9000, 128, 128, 6, 2), (30000, 72, 40, 5, 1), (3000, 256, 256, 4, 2)])
def test_paths_of_many_rows(T, D, F, E, k, dtype):
    """The products as they are chosen for many rows, inference and training, give the same result as slot by slot."""
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, experts, gates, dy = _make(T, 1, D, F, E, k, dtype, 17, closed=0.05)
    ref, mag = _reference(x, w, experts, gates, dy)
    plan = plan_experts(experts.cuda(), E)
    y = expert_linear(x.cuda(), w.cuda(), plan, gates.cuda())
    _check(dict(y=y), ref, mag, dict(y=D), dtype)
    xg = x.cuda().requires_grad_()
    (dx,) = torch.autograd.grad(expert_linear(xg, w.cuda(), plan, gates.cuda()), xg, dy.cuda())
    _check(dict(dx=dx), ref, mag, dict(dx=F), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,M,D,F,E,k", [
    (11000, 3, 112, 32, 3, 2), (40001, 1, 64, 64, 2, 2), (9000, 1, 64, 64, 5, 1), (5000, 1, 300, 24, 4, 3),
    (4000, 1, 48, 300, 3, 2), (6000, 2, 16, 16, 5, 4), (3001, 1, 201, 57, 7, 3)])
def test_narrow_blocks(T, M, D, F, E, k, dtype):
    """Blocks of up to 64 columns or rows: narrow tiles, and held blocks whose waves share the rows of a stage."""
    _run_and_check(*_make(T, M, D, F, E, k, dtype, T + D, closed=0.02), dtype)
