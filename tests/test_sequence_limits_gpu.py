"""The operators of token sequences and AdamW where sizes end: tensors of more than 2^31 values, time strides at their limit, single
steps of any stride, and calls that run at once or out of two graphs that share their memory."""
import pytest
import torch

from oracle import sequence as O

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _need(gib):
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip("needs %d GiB of free memory" % gib)


def _near(name, got, want, bound):
    u = torch.finfo(got.dtype).eps / 2
    over = (got.double() - want).abs() / (bound + 1.01 * u * (want.abs() + bound) + 1e-30)
    assert bool((over <= 1).all()), "%s: %.2f times its bound" % (name, float(over.nan_to_num(nan=9e9).max()))


def _d(c):
    return {k: (v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v) for k, v in c.items()}


def _scan_case(B, T, D, N, G=1, dtype=BF16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, t=torch.float32: torch.randn(*s, generator=g, device="cuda", dtype=t)                               # noqa: E731
    return {"u": r(B, T, D, t=dtype), "dt": r(B, T, D, t=dtype).sub_(2), "A": -torch.exp(r(D, N)), "B": r(B, T, G, N, t=dtype),
            "C": r(B, T, G, N, t=dtype), "D": r(D), "z": r(B, T, D, t=dtype), "dt_bias": 0.3 * r(D)}, r(B, T, D, t=dtype)


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def test_scan_of_more_than_two_to_the_31_values():
    _need(60)
    from avsi_amd import ops
    T, D = 2100, 1 << 20
    c, dout = _scan_case(1, T, D, 4)
    out, new, kept = ops.selective_scan(**c, want_state=True, keep=True)
    du, ddt, dA, _, _, dD, dz, dbias = ops.selective_scan_bwd(dout, **c, kept=kept)
    last = slice(D - 64, D)
    part = {k: v[..., last] if k in ("u", "dt", "z") else v[last] if k in ("A", "D", "dt_bias") else v for k, v in c.items()}
    val, err = O.scan(**_d(part), dout=dout[..., last].double())
    for k, got in (("out", out[..., last]), ("state", new[:, last]), ("du", du[..., last]), ("ddt", ddt[..., last]), ("dA", dA[last]),
                   ("dD", dD[last]), ("dz", dz[..., last]), ("ddt_bias", dbias[last])):
        _near(k, got, val[k], err[k])


def test_scan_time_strides_at_their_limit():
    _need(20)
    from avsi_amd import ops
    B, T, D, N, step = 1, 35, 70, 8, 1 << 26
    c, dout = _scan_case(B, T, D, N, seed=1)
    want = ops.selective_scan(**c, keep=True)
    grads = ops.selective_scan_bwd(dout, **c, kept=want[2])
    buf = torch.empty((T - 1) * step + 1024, dtype=BF16, device="cuda")
    far, at = dict(c), 0
    for k in ("u", "dt", "z", "B", "C"):
        n = c[k][0, 0].numel()
        shape = c[k].shape
        v = torch.as_strided(buf, shape, (0, step, 1) if len(shape) == 3 else (0, step, shape[-1], 1), at)
        v.copy_(c[k])
        far[k], at = v, at + (n + 7) // 8 * 8
    far_dout = torch.as_strided(buf, dout.shape, (0, step, 1), at).copy_(dout)
    got = ops.selective_scan(**far, keep=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    for a, b in zip(ops.selective_scan_bwd(far_dout, **far, kept=got[2]), grads):
        assert torch.equal(a, b)
    wide = torch.as_strided(buf, (1, 2, D), (0, step + 1, 1))
    with pytest.raises(Exception, match="(?i)unsupported|not supported"):
        ops.selective_scan(wide, c["dt"][:, :2], c["A"], c["B"][:, :2], c["C"][:, :2])


def test_a_single_step_has_no_time_stride():
    from avsi_amd import ops
    c, dout = _scan_case(3, 1, 40, 16, seed=2)
    odd = lambda t: torch.as_strided(t, t.shape, (t.stride(0), 1 << 40) + t.stride()[2:])                              # noqa: E731
    far = {k: odd(v) if v.dim() >= 3 else v for k, v in c.items()}
    want, got = ops.selective_scan(**c, keep=True), ops.selective_scan(**far, keep=True)
    assert torch.equal(got[0], want[0])
    for a, b in zip(ops.selective_scan_bwd(odd(dout), **far, kept=got[2]), ops.selective_scan_bwd(dout, **c, kept=want[2])):
        assert torch.equal(a, b)
    w = torch.randn(40, 4, device="cuda")
    assert torch.equal(ops.causal_conv(odd(c["u"]), w)[0], ops.causal_conv(c["u"], w)[0])
    for a, b in zip(ops.causal_conv_bwd(odd(dout), odd(c["u"]), w)[:2], ops.causal_conv_bwd(dout, c["u"], w)[:2]):
        assert torch.equal(a, b)


def test_conv_of_more_than_two_to_the_31_values():
    _need(30)
    from avsi_amd import ops
    T, D = 2100, 1 << 20
    x, dy = torch.randn(2, 1, T, D, device="cuda", dtype=BF16).unbind(0)
    w, bias = torch.randn(D, 4, device="cuda"), torch.randn(D, device="cuda")
    y, _ = ops.causal_conv(x, w, bias)
    dx, dw, db = ops.causal_conv_bwd(dy, x, w, bias)
    k = slice(D - 64, D)
    part = x[..., k].double(), w[k].double(), bias[k].double()
    (val, err), (grad, grad_err) = O.conv_forward(*part), O.conv_backward(dy[..., k].double(), *part)
    _near("y", y[..., k], val["y"], err["y"])
    for name, got in (("dx", dx[..., k]), ("dw", dw[k]), ("dbias", db[k])):
        _near(name, got, grad[name], grad_err[name])


def test_layer_norm_of_more_than_two_to_the_31_values():
    _need(30)
    from avsi_amd import ops
    M, C = (1 << 21) + 5, 1032
    x, dy = torch.randn(2, M, C, device="cuda", dtype=BF16).unbind(0)
    gamma, beta = torch.randn(2, C, device="cuda").unbind(0)
    y, mean, rstd = ops.layer_norm(x, gamma, beta)
    dx, _, dbeta = ops.layer_norm_bwd(dy, x, mean, rstd, gamma)
    few = ops.layer_norm(x[-3:], gamma, beta)
    assert torch.equal(y[-3:], few[0]) and torch.equal(mean[-3:], few[1])
    assert torch.equal(dx[-3:], ops.layer_norm_bwd(dy[-3:], x[-3:], *few[1:], gamma)[0])
    # 512 workgroups add at most M / 512 + 1 rows each, one behind the other, and then their 512 sums are added
    want, size = torch.zeros(C, dtype=torch.float64, device="cuda"), torch.zeros(C, dtype=torch.float64, device="cuda")
    for part in dy.split(1 << 17):
        want += part.double().sum(0)
        size += part.double().abs().sum(0)
    assert bool(((dbeta.double() - want).abs() <= (M // 512 + 1024) * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_more_than_two_to_the_31_values(bits):
    _need(45)
    from avsi_amd import ops
    n, tail = (1 << 31) + 1000, 1256
    w = torch.empty(n, device="cuda").normal_()
    g = torch.empty(n, device="cuda", dtype=BF16).normal_()
    few, few_g = w[n - tail:].clone(), g[n - tail:].clone()
    assert (n - tail) % 256 == 0
    plan, small = ops.AdamwPlan([w], [g], bits=bits), ops.AdamwPlan([few], [few_g], bits=bits)
    for step in (1, 2):
        ops.adamw(plan, step, 1e-3)
        ops.adamw(small, step, 1e-3)
    assert torch.equal(w[n - tail:], few)
    for k in plan.state:
        a, b = plan.state[k].view(torch.uint8), small.state[k].view(torch.uint8)
        assert torch.equal(a[a.numel() - b.numel():], b)


def test_calls_at_once_on_two_streams():
    from avsi_amd import ops
    cases = [_scan_case(2, 700, 130, 16, seed=s) for s in (3, 4)]
    w = torch.randn(130, 4, device="cuda")
    gamma = torch.randn(130, device="cuda")

    def run(c, dout):
        out, new, kept = ops.selective_scan(**c, want_state=True, keep=True)
        y, mean, rstd = ops.layer_norm(out, gamma)
        return [out, new, y, *ops.selective_scan_bwd(dout, **c, kept=kept), *ops.causal_conv_bwd(dout, c["u"], w)[:2],
                *ops.layer_norm_bwd(dout, out, mean, rstd, gamma)]

    want = [run(*k) for k in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, k in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(run(*k))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_graphs_that_share_their_memory():
    from avsi_amd import ops
    cases = [_scan_case(2, 900, 70, 16, seed=s) for s in (5, 6)]
    w, gamma = torch.randn(70, 4, device="cuda"), torch.randn(70, device="cuda")

    def run(c, dout):
        x, _ = ops.causal_conv(c["u"], w)
        out, _, kept = ops.selective_scan(x, **{k: v for k, v in c.items() if k != "u"}, keep=True)
        y, mean, rstd = ops.layer_norm(out, gamma)
        dx, dg, _ = ops.layer_norm_bwd(dout, out, mean, rstd, gamma)
        grads = ops.selective_scan_bwd(dx, x, **{k: v for k, v in c.items() if k != "u"}, kept=kept)
        return [y, dg, *grads, *ops.causal_conv_bwd(grads[0], c["u"], w)[:2]]

    want = [run(*k) for k in cases]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for k in cases:
            run(*k)
    torch.cuda.current_stream().wait_stream(s)
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for k in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(run(*k))
        graphs.append(graph)
    for i in (0, 1, 1, 0, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        eager = run(*cases[1 - i])
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[1 - i]))
