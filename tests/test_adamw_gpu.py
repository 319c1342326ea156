"""AdamW over many tensors against its formula in 64 bits; the 8-bit moments against what a block's scale and e4m3 can hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HYPER = dict(beta1=0.9, beta2=0.99, eps=1e-8, grad_scale=0.5)
SIZES = [1, 3, 255, 256, 257, 1023, 4096, 4097, 20000, 64, 7]


def _make(sizes, gdtype=torch.float32, bits=32, copies=None, seed=0):
    from avsi_amd import ops
    g = torch.Generator().manual_seed(seed)
    r = lambda n: torch.randn(n, generator=g).cuda()                                                                   # noqa: E731
    params = [0.1 * r(n) for n in sizes]
    grads = [(r(n) * 10 ** float(torch.rand((), generator=g) * 4 - 4)).to(gdtype) for n in sizes]
    cps = None if copies is None else [None if i % 3 == 2 else torch.zeros(n, dtype=copies, device="cuda") for i, n in enumerate(sizes)]
    decay = [0.1 if i % 2 else 0.0 for i in range(len(sizes))]
    return ops.AdamwPlan(params, grads, weight_decay=decay, bits=bits, copies=cps), params, grads, cps, decay


def _moments(plan, i, n):
    """(m, v) of parameter i as float64, and the scales of its blocks spread over it (or None)."""
    o = plan.offsets[i]
    m, v = (plan.state[k][o:o + n].double() for k in ("m", "v"))
    if plan.bits == 32:
        return m, v, None, None
    s = [plan.state[k][o // 256:o // 256 + -(-n // 256)].double().repeat_interleave(256)[:n] for k in ("m_scale", "v_scale")]
    return m * s[0], (v * s[1]) ** 2, s[0], s[1]


def _step(plan, params, grads, cps, decay, step, lr):
    """One step, held to the formula from the state in front of it.  Bounds: half a step for every operation -- 3 on each term of m, 4
    of v, 16 more up to the quotient, 3 on the decay, 2 on the weight -- and the seven numbers of the step as floats."""
    from avsi_amd import ops
    sizes = [p.numel() for p in params]
    before = [(p.double().clone(), *_moments(plan, i, n)) for i, (p, n) in enumerate(zip(params, sizes))]
    ops.adamw(plan, step, lr, **HYPER)
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    for i, n in enumerate(sizes):
        w, m, v, _, _ = before[i]
        g = grads[i].double().reshape(-1) * HYPER["grad_scale"]
        m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        em, ev = 6 * U * (b1 * m.abs() + (1 - b1) * g.abs()), 8 * U * v1
        d = torch.sqrt(v1 / (1 - b2 ** step)) + HYPER["eps"]
        up = m1 / (1 - b1 ** step) / d
        want = w - lr * (up + decay[i] * w)
        tol = lr * (em / (1 - b1 ** step) / d + 24 * U * up.abs() + 4 * U * decay[i] * w.abs()) + 2 * U * (w.abs() + want.abs())
        assert bool(((params[i].double().reshape(-1) - want.reshape(-1)).abs() <= tol.reshape(-1)).all()), i
        gm, gv, sm, sv = _moments(plan, i, n)
        if plan.bits == 32:
            assert bool(((gm - m1).abs() <= em).all()) and bool(((gv - v1).abs() <= ev).all()), i
        else:
            for got, true, s, e in ((gm, m1, sm, em), (gv.sqrt(), v1.sqrt(), sv, 6 * U * v1.sqrt())):
                blocks = torch.nn.functional.pad(true.abs(), (0, -n % 256)).view(-1, 256).amax(1).repeat_interleave(256)[:n]
                assert bool(((s * 448 - blocks).abs() <= 12 * U * blocks).all()), i
                # e4m3: half of a step is 2^-4 of the value, 2^-10 of the scale below its normal range
                half = torch.maximum(2.0 ** -4 * true.abs(), 2.0 ** -10 * s)
                small = (true > 0) & (true < 2.0 ** -10 * s) & (s is sv)
                assert bool(((got - true).abs() <= torch.where(small, 2.0 ** -9 * s, half * (1 + 32 * U) + e)).all()), i
            assert bool((gv[v1 > 0] > 0).all())
        if cps is not None and cps[i] is not None:
            assert torch.equal(cps[i], params[i].to(cps[i].dtype))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gdtype,copies", [(torch.float32, None), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)], ids=str)
def test_adamw_matches_the_formula(bits, gdtype, copies):
    plan, params, grads, cps, decay = _make(SIZES, gdtype, bits, copies)
    for step in (1, 2, 3):
        _step(plan, params, grads, cps, decay, step, 1e-3)
        for g in grads:
            g.mul_(-0.5)
    if bits == 8:      # the padding between the tensors has stayed zero
        used = torch.zeros(plan.numel, dtype=torch.bool, device="cuda")
        for o, p in zip(plan.offsets, params):
            used[o:o + p.numel()] = True
        assert bool((plan.state["m"].float()[~used] == 0).all()) and bool((plan.state["v"].float()[~used] == 0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes(bits):
    plan, params, grads, cps, decay = _make([(37 * k) % 600 for k in range(131)], bits=bits)      # (some are empty)
    _step(plan, params, grads, cps, decay, 1, 1e-2)


def test_shapes_and_lists_of_states():
    from avsi_amd import ops
    p = [torch.randn(5, 7, device="cuda"), torch.randn(3, device="cuda"), torch.randn(2, 3, 4, device="cuda")]
    g = [torch.randn_like(x) for x in p]
    q = [x.clone() for x in p]
    m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
    one, two = ops.AdamwPlan(p, g), ops.AdamwPlan(q, g, state={"m": m, "v": v})
    for s in (1, 2):
        ops.adamw(one, s, 1e-2), ops.adamw(two, s, 1e-2)
    assert all(torch.equal(a, b) for a, b in zip(p, q))
    assert all(torch.equal(one.state["m"][o:o + x.numel()].view_as(x), x) for o, x in zip(one.offsets, m))
    # a checkpoint's state goes on where it was
    r = [x.clone() for x in p]
    three = ops.AdamwPlan(r, g, state={k: t.clone() for k, t in one.state.items()})
    ops.adamw(one, 3, 1e-2), ops.adamw(three, 3, 1e-2)
    assert all(torch.equal(a, b) for a, b in zip(p, r))


def test_unaligned_tensors():
    # views of one flat buffer at odd offsets, as a model's variables lie
    from avsi_amd import ops
    flat, grad = torch.randn(3000, device="cuda"), torch.randn(3000, device="cuda")
    cuts = [(1, 258), (259, 1500), (1759, 1001)]
    cut = lambda t: [t[a:a + n] for a, n in cuts]                                                                      # noqa: E731
    a, b = flat.clone(), flat.clone()
    one = ops.AdamwPlan(cut(a), cut(grad), bits=8)
    two = ops.AdamwPlan([t.clone() for t in cut(b)], [t.clone() for t in cut(grad)], bits=8)
    ops.adamw(one, 1, 1e-2), ops.adamw(two, 1, 1e-2)
    for got, want in zip(cut(a), two._params):
        assert torch.equal(got, want)
    assert a[0] == flat[0] and torch.equal(a[2760:], flat[2760:]) and all(torch.equal(one.state[k].view(torch.uint8), two.state[k].view(torch.uint8))
                                                                          for k in one.state)


def test_eight_bit_codes_are_torch_e4m3():
    """Every e4m3 value and the middles between neighbours, through m = (1 - beta1) g of a first step with beta1 = 0: the codes are
    torch's own (to nearest, ties to even), since the block's largest value makes the scale exactly 1."""
    from avsi_amd import ops
    codes = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn).float()
    vals = torch.sort(codes[codes.isfinite() & (codes >= 0)].unique())[0]
    mids = (vals[1:] + vals[:-1]) / 2
    x = torch.cat([vals, mids, -mids, -vals])
    x = torch.cat([torch.cat([x, torch.zeros(-len(x) % 255)]).view(-1, 255), torch.full((-(-len(x) // 255), 1), 448.0)], 1).reshape(-1).cuda()
    w = torch.zeros_like(x)
    plan = ops.AdamwPlan([w], [x], weight_decay=0.0, bits=8)
    ops.adamw(plan, 1, 0.0, beta1=0.0, beta2=0.0, eps=1.0)
    assert bool((plan.state["m_scale"] == 1).all())
    assert torch.equal(plan.state["m"].float(), x.to(torch.float8_e4m3fn).float())
    # v: the root of g^2 is |g| here; above zero it keeps at least the smallest code
    want = torch.where(x != 0, x.abs().to(torch.float8_e4m3fn).float().clamp(min=2.0 ** -9), torch.zeros_like(x))
    assert torch.equal(plan.state["v"].float(), want)


def test_tiny_and_zero_blocks():
    from avsi_amd import ops
    g = torch.zeros(1024, device="cuda")
    g[256:512] = 1e-30
    g[512:768] = 1e-42
    g[768] = 1.0
    w = torch.ones(1024, device="cuda")
    plan = ops.AdamwPlan([w], [g], weight_decay=0.0, bits=8)
    for s in (1, 2, 3):
        ops.adamw(plan, s, 1e-3)
    assert bool(w.isfinite().all()) and bool((w[:256] == 1).all()) and bool((plan.state["m_scale"][:1] == 0).all())
    assert all(bool(plan.state[k].float().isfinite().all()) for k in plan.state)


def test_non_finite_gradients():
    """32 bits: a NaN stays in its element.  8 bits: its weight is NaN at once, and its block's moments are."""
    from avsi_amd import ops
    for bits in (32, 8):
        for bad in (float("nan"), float("inf")):
            w, g = torch.ones(1000, device="cuda"), torch.full((1000,), 0.1, device="cuda")
            g[300] = bad
            plan = ops.AdamwPlan([w], [g], bits=bits)
            ops.adamw(plan, 1, 1e-3)
            assert w.isnan().nonzero().flatten().tolist() == [300]
            if bits == 8:
                m = plan.state["m"].float() * plan.state["m_scale"].repeat_interleave(256)
                assert m.isnan().nonzero().flatten().tolist() == list(range(256, 512))


def test_skip_guard_and_refusals():
    from avsi_amd import _lib, ops
    plan, params, grads, _, _ = _make([500, 3000], bits=8)
    before = [p.clone() for p in params]
    for word in (1.0, float("nan")):
        ops.adamw(plan, 1, 1e-3, skip=torch.tensor([0.0, word], device="cuda"))
        assert all(torch.equal(a, b) for a, b in zip(params, before)) and bool((plan.state["m"].float() == 0).all())
    ops.adamw(plan, 1, 1e-3, skip=torch.zeros(8, device="cuda"))
    assert not torch.equal(params[0], before[0])
    for kw in (dict(step=0, lr=1.0), dict(step=1, lr=1.0, beta1=1.0), dict(step=1, lr=1.0, eps=-1.0), dict(step=1, lr=1.0, skip=torch.zeros(9, device="cuda")),
               dict(step=1, lr=1.0, skip=torch.zeros(2))):
        with pytest.raises(_lib.AvsiError):
            ops.adamw(plan, **kw)
    x = torch.zeros(100, device="cuda")
    for args, kw in ((([x, x], [x.clone(), x.clone()]), {}), (([x[:60], x[50:]], [x[:60].clone(), x[50:].clone()]), {}), (([x], [x]), {}),
                     (([x], [x.clone()]), dict(state={"m": [x], "v": [x.clone()]})), (([x], [x.clone()]), dict(state={"m": x.clone()})),
                     (([x], [x.clone()]), dict(state={"m": x.clone(), "v": x.clone()})),
                     (([x], [torch.zeros(100)]), {})):
        with pytest.raises(_lib.AvsiError):
            ops.AdamwPlan(*args, **kw)
    # tensors that moved, and other gradients
    y, g = torch.zeros(100, device="cuda"), torch.ones(100, device="cuda")
    plan = ops.AdamwPlan([y], [g])
    y.data = torch.zeros(100, device="cuda")
    with pytest.raises(_lib.AvsiError, match="moved"):
        ops.adamw(plan, 1, 1e-3)
    plan = ops.AdamwPlan([y], [g])
    plan.set_grads([torch.full((100,), -1.0, device="cuda", dtype=torch.bfloat16)])
    ops.adamw(plan, 1, 1e-3)
    assert bool((y > 0).all())
    with pytest.raises(_lib.AvsiError):
        plan.set_grads([y])
    with pytest.raises(_lib.AvsiError):
        plan.set_grads([torch.zeros(99, device="cuda")])


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_streams_and_graph(bits):
    from avsi_amd import ops
    one, p1, g1, _, _ = _make(SIZES, bits=bits, seed=4)
    two, p2, g2, _, _ = _make(SIZES, bits=bits, seed=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.adamw(one, 5, 1e-3)
    torch.cuda.current_stream().wait_stream(side)
    ops.adamw(two, 5, 1e-3)
    assert all(torch.equal(a, b) for a, b in zip(p1, p2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adamw(one, 5, 1e-3)
    for _ in range(4):
        for g in g1 + g2:
            g.mul_(-0.7)
        graph.replay()
        ops.adamw(two, 5, 1e-3)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(p1, p2))
        assert all(torch.equal(one.state[k].view(torch.uint8), two.state[k].view(torch.uint8)) for k in one.state)
