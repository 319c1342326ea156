"""Causal convolution and selective scan against the oracle in 64 bits (oracle/sequence.py), whose bounds count the roundings of a
32-bit evaluation; a value written in 16 bits may be half a step further off."""
import pytest
import torch

from oracle import sequence as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _case(B, T, D, N, G=1, K=4, dtype=torch.float32, ragged=False, carry=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)                                                                        # noqa: E731
    c = {"u": r(B, T, D).to(dtype), "dt": (0.7 * r(B, T, D) - 2).to(dtype), "A": -torch.exp(r(D, N)), "B": r(B, T, G, N).to(dtype),
         "C": r(B, T, G, N).to(dtype), "D": r(D), "z": r(B, T, D).to(dtype), "dt_bias": 0.3 * r(D)}
    v = {"x": r(B, T, D).to(dtype), "w": r(D, K), "bias": r(D)}
    s, cs = (0.5 * r(B, D, N), r(B, K - 1, D).to(dtype)) if carry else (None, None)
    lengths = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32) if ragged else None
    cu = lambda t: None if t is None else t.cuda()                                                                     # noqa: E731
    return ({k: cu(t) for k, t in c.items()}, {k: cu(t) for k, t in v.items()}, r(B, T, D).to(dtype).cuda(), cu(s), cu(cs), cu(lengths))


def _d(kw):
    return {k: (v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v) for k, v in kw.items()}


def _near(name, got, want, bound):
    u = torch.finfo(got.dtype).eps / 2
    # (an fp16 value below its normal range is rounded to a step of 2^-24, half of which is absolute)
    tol = bound + 1.01 * u * (want.abs() + bound) + (2.0 ** -25 if got.dtype == torch.float16 else 0) + 1e-30
    assert got.shape == want.shape, name
    over = ((got.double() - want).abs() / tol)
    assert bool((over <= 1).all()), "%s: %.2f times its bound" % (name, float(over.nan_to_num(nan=9e9).max()))


NAMES = ("du", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias")


def _check_scan(c, dout, state, lengths, softplus=True):
    from avsi_amd import ops
    out, new, kept = ops.selective_scan(**c, softplus=softplus, state=state, lengths=lengths, want_state=True, keep=True)
    val, err = O.scan(**_d(c), softplus=softplus, state=None if state is None else state.double(), lengths=lengths, dout=dout.double())
    _near("out", out, val["out"], err["out"])
    _near("state", new, val["state"], err["state"])
    grads = dict(zip(NAMES, ops.selective_scan_bwd(dout, **c, softplus=softplus, kept=kept, state=state, lengths=lengths)))
    for k in NAMES:
        if c.get({"dD": "D", "dz": "z", "ddt_bias": "dt_bias"}.get(k, "u")) is None:
            assert grads[k] is None, k
        else:
            _near(k, grads[k], val[k], err[k])
    return out, new, grads


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,T,D,N,G", [(1, 1, 1, 1, 1), (2, 2, 3, 4, 1), (1, 15, 5, 3, 1), (2, 16, 64, 16, 1), (3, 17, 65, 16, 1), (1, 33, 130, 5, 2),
                                       (2, 64, 12, 8, 4), (1, 65, 63, 17, 1), (2, 130, 66, 16, 3), (1, 250, 20, 64, 1), (2, 77, 260, 2, 2),
                                       (1, 129, 34, 24, 2), (4, 40, 48, 33, 1)])
def test_scan_matches_the_recurrence(dtype, B, T, D, N, G):
    c, _, dout, *_ = _case(B, T, D, N, G, dtype=dtype, seed=T + N)
    _check_scan(c, dout, None, None)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,T,D,N,G", [(5, 1, 7, 16, 1), (6, 16, 64, 16, 1), (7, 50, 33, 8, 3), (4, 200, 70, 16, 1), (3, 300, 20, 40, 2)])
def test_scan_ragged_behind_a_state(dtype, B, T, D, N, G):
    c, _, dout, state, _, lengths = _case(B, T, D, N, G, dtype=dtype, ragged=True, carry=True, seed=T)
    lengths[0], lengths[-1] = 0, T
    out, new, grads = _check_scan(c, dout, state, lengths)
    assert torch.equal(new[0], state[0])
    on = O.inside(B, T, lengths, "cuda")
    for t in (out, grads["du"], grads["ddt"], grads["dz"], grads["dB"], grads["dC"]):
        assert bool((t[~on] == 0).all())


@pytest.mark.parametrize("missing", ["D", "z", "dt_bias", "softplus", "all"])
def test_scan_optional_operands(missing):
    c, _, dout, state, _, lengths = _case(3, 90, 40, 16, dtype=torch.bfloat16, ragged=True, carry=True)
    for k in ("D", "z", "dt_bias"):
        if missing in (k, "all"):
            c[k] = None
    plain = missing in ("softplus", "all")
    if plain:
        c["dt"], c["dt_bias"] = c["dt"].abs() * 0.1, None if missing == "all" else c["dt_bias"].abs()
    _check_scan(c, dout, state, lengths, softplus=not plain)


def test_scan_without_chunks():
    # enough sequences and channels for every SIMD: the path that does not cut time (the small cases above all do, beyond 64 steps)
    c, _, dout, state, _, lengths = _case(18, 70, 1000, 16, dtype=torch.float32, ragged=True, carry=True)
    _check_scan(c, dout, state, lengths)


def test_scan_gradients_by_differences():
    """Along one direction through all inputs at once: the quotient's own error is the roundings of out over 2 h, and h^2 / 6 times
    the third derivative, estimated by the quotient at 2 h (a fourth-order quotient then leaves h^4 of it)."""
    from avsi_amd import ops
    c, _, dout, state, _, lengths = _case(2, 40, 24, 16, ragged=True, carry=True, seed=5)
    g = torch.Generator().manual_seed(6)
    v = {k: torch.randn(t.shape, generator=g).cuda() * (0.1 if k in ("A", "dt", "dt_bias") else 1.0) for k, t in c.items()}
    out, _, kept = ops.selective_scan(**c, state=state, lengths=lengths, keep=True)
    grads = dict(zip(NAMES, ops.selective_scan_bwd(dout, **c, kept=kept, state=state, lengths=lengths)))
    want = sum(float((grads["d" + k].double() * v[k]).sum()) for k in c)

    def at(h):
        o = ops.selective_scan(**{k: t + h * v[k] for k, t in c.items()}, state=state, lengths=lengths)[0]
        return float((o.double() * dout).sum())
    h = 2.0 ** -6
    q1, q2 = (at(h) - at(-h)) / (2 * h), (at(2 * h) - at(-2 * h)) / (4 * h)
    size = float((out.abs().double() * dout.abs()).sum())
    bound = 2 * 200 * O.U * size / h + abs(q1 - q2) / 8       # (4 q1 - q2) / 3 leaves well below an eighth of what it takes off
    assert abs((4 * q1 - q2) / 3 - want) <= bound + 1e-6 * abs(want)


def test_scan_strides_and_layouts():
    """Slices of wider buffers, time-major buffers, broadcast and unaligned operands give the bits that contiguous ones give."""
    from avsi_amd import ops
    c, _, dout, state, _, lengths = _case(3, 37, 33, 16, dtype=torch.bfloat16, ragged=True, carry=True)
    want = ops.selective_scan(**c, state=state, lengths=lengths, want_state=True, keep=True)
    wantg = ops.selective_scan_bwd(dout, **c, kept=want[2], state=state, lengths=lengths)

    def wide(t):
        buf = torch.full((*t.shape[:-1], t.shape[-1] + 5), float("nan"), dtype=t.dtype, device="cuda")
        buf[..., 3:3 + t.shape[-1]] = t
        return buf[..., 3:3 + t.shape[-1]]

    def time_major(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    for lay in (wide, time_major):
        d = {k: lay(t) if t.dim() >= 3 else t for k, t in c.items()}
        got = ops.selective_scan(**d, state=state, lengths=lengths, want_state=True, keep=True)
        assert all(torch.equal(a, b) for a, b in zip(got[:2], want))       # (rows of `kept` behind a length are not written)
        gotg = ops.selective_scan_bwd(lay(dout), **d, kept=got[2], state=state, lengths=lengths)
        assert all(torch.equal(a, b) for a, b in zip(gotg, wantg))
    # one z for all sequences, and B and C without an axis of groups
    d = dict(c, z=c["z"][:1].expand(3, -1, -1), B=c["B"][:, :, 0], C=c["C"][:, :, 0])
    got = ops.selective_scan(**d, state=state, lengths=lengths, keep=True)
    ref = ops.selective_scan(**dict(c, z=c["z"][:1].repeat(3, 1, 1)), state=state, lengths=lengths, keep=True)
    assert torch.equal(got[0], ref[0])
    g = ops.selective_scan_bwd(dout, **d, kept=got[2], state=state, lengths=lengths)
    assert g[3].shape == (3, 37, 16) and g[4].shape == (3, 37, 16)


def test_nothing_is_read_behind_a_length():
    from avsi_amd import ops
    c, v, dout, state, cstate, _ = _case(4, 100, 40, 16, dtype=torch.float16, carry=True)
    lengths = torch.tensor([0, 100, 33, 1], dtype=torch.int32, device="cuda")
    off = ~O.inside(4, 100, lengths, "cuda")

    def both(c, v, dout):
        s = ops.selective_scan(**c, state=state, lengths=lengths, want_state=True, keep=True)
        g = ops.selective_scan_bwd(dout, **c, kept=s[2], state=state, lengths=lengths)
        y = ops.causal_conv(**v, state=cstate, lengths=lengths, want_state=True)
        return list(s[:2]) + list(g) + list(y) + list(ops.causal_conv_bwd(dout, **v, state=cstate, lengths=lengths))
    want = both(c, v, dout)
    dirty = lambda t: t if t.dim() < 3 else torch.where(off.reshape(off.shape + (1,) * (t.dim() - 2)), float("nan"), t.float()).to(t.dtype)  # noqa: E731
    got = both({k: dirty(t) for k, t in c.items()}, {k: dirty(t) for k, t in v.items()}, dirty(dout))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # lengths outside 0 .. time are clamped
    wild = torch.tensor([-7, 2 ** 31 - 1, 33, 1], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.selective_scan(**c, state=state, lengths=wild)[0], want[0])
    assert torch.equal(ops.causal_conv(**v, state=cstate, lengths=wild)[0], want[10])


def test_masked_places_with_infinities():
    """A gate of -inf closes a channel to NaN (its definition: -inf times 0), and only that one; dt of -inf is a step of size zero."""
    from avsi_amd import ops
    c, *_ = _case(2, 20, 33, 16)
    want = ops.selective_scan(**c)[0]
    c2 = dict(c, dt=c["dt"].clone())
    c2["dt"][0, 5:, 7] = float("-inf")
    out, new, _ = ops.selective_scan(**c2, want_state=True)
    keep = torch.ones_like(want, dtype=torch.bool)
    keep[0, 5:, 7] = False
    assert torch.equal(out[keep], want[keep]) and bool(out.isfinite().all())
    first = ops.selective_scan(**{k: (t[:1, :5] if t.dim() > 2 else t) for k, t in c.items()}, want_state=True)[1]
    assert torch.equal(new[0, 7], first[0, 7])
    c3 = dict(c, u=c["u"].clone())
    c3["u"][1, 9, 4] = float("nan")
    out = ops.selective_scan(**c3)[0]
    bad = torch.zeros_like(want, dtype=torch.bool)
    bad[1, 9:, 4] = True
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], want[~bad])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_pieces_and_single_tokens_continue_a_prompt(dtype):
    """A prompt in two pieces and the rest token by token: held to the oracle of the whole sequence (its bound holds for every split)."""
    from avsi_amd import ops
    B, T, D = 3, 48, 37
    c, v, _, state, cstate, _ = _case(B, T, D, 16, G=1, dtype=dtype, carry=True, seed=11)
    val, err = O.scan(**_d(c), state=state.double())
    f, fe = O.conv_forward(*(v[k].double() for k in ("x", "w", "bias")), state=cstate.double())
    part = lambda kw, a, b: {k: (t[:, a:b] if t.dim() >= 3 else t) for k, t in kw.items()}                             # noqa: E731
    o1, s1, _ = ops.selective_scan(**part(c, 0, 20), state=state, want_state=True)
    o2, s2, _ = ops.selective_scan(**part(c, 20, 40), state=s1, want_state=True)
    y1, k1 = ops.causal_conv(**part(v, 0, 2), state=cstate, want_state=True)       # (shorter than the state: some of it stays)
    y2, k2 = ops.causal_conv(**part(v, 2, 40), state=k1, want_state=True)
    outs, ys = [o1, o2], [y1, y2]
    for t in range(40, T):
        one = {k: (x[:, t] if x.dim() >= 3 else x) for k, x in c.items()}
        outs.append(ops.selective_scan_step(**one, state=s2)[:, None])
        ys.append(ops.causal_conv_step(v["x"][:, t], v["w"], v["bias"], state=k2)[:, None])
    _near("out", torch.cat(outs, 1), val["out"], err["out"])
    _near("state", s2, val["state"], err["state"])
    _near("y", torch.cat(ys, 1), f["y"], fe["y"])
    assert torch.equal(k2, v["x"][:, -3:])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (3, 65, 16, 1), (5, 12, 5, 4), (2, 30, 64, 2), (300, 70, 16, 1), (7, 9, 33, 3)])
def test_step_matches_the_recurrence(dtype, B, D, N, G):
    from avsi_amd import ops
    c, _, _, state, _, _ = _case(B, 1, D, N, G, dtype=dtype, carry=True, seed=B)
    val, err = O.scan(**_d(c), state=state.double())
    one = {k: (t[:, 0] if t.dim() >= 3 else t) for k, t in c.items()}
    out = ops.selective_scan_step(**one, state=state)
    _near("out", out[:, None], val["out"], err["out"])
    _near("state", state, val["state"], err["state"])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,T,D,K,ragged,carry", [(1, 1, 1, 2, False, False), (2, 3, 7, 4, False, True), (3, 50, 64, 4, True, True), (1, 257, 130, 3, False, False),
                                                  (4, 33, 65, 8, True, True), (2, 90, 20, 5, True, False), (3, 1, 33, 4, True, True), (2, 1000, 9, 2, False, True),
                                                  (2, 40, 1100, 4, True, True)])
def test_conv_matches_its_formula(dtype, B, T, D, K, ragged, carry):
    from avsi_amd import ops
    for silu, with_bias in ((True, True), (False, False)):
        _, v, dy, _, state, lengths = _case(B, T, D, 1, K=K, dtype=dtype, ragged=ragged, carry=carry, seed=T)
        if not with_bias:
            v["bias"] = None
        dv, s64 = _d(v), None if state is None else state.double()
        f, fe = O.conv_forward(**dv, silu=silu, state=s64, lengths=lengths)
        y, new = ops.causal_conv(**v, silu=silu, state=state, lengths=lengths, want_state=True)
        _near("y", y, f["y"], fe["y"])
        assert torch.equal(new.double(), f["state"])
        val, err = O.conv_backward(dy.double(), **dv, silu=silu, state=s64, lengths=lengths)
        dx, dw, dbias = ops.causal_conv_bwd(dy, **v, silu=silu, state=state, lengths=lengths)
        _near("dx", dx, val["dx"], err["dx"])
        _near("dw", dw, val["dw"], err["dw"])
        if with_bias:
            _near("dbias", dbias, val["dbias"], err["dbias"])
        else:
            assert dbias is None
        only = ops.causal_conv_bwd(dy, **v, silu=silu, state=state, lengths=lengths, want_wgrad=False)
        assert torch.equal(only[0], dx) and only[1] is None and only[2] is None


def test_conv_strides():
    from avsi_amd import ops
    _, v, dy, _, state, lengths = _case(3, 37, 33, 1, dtype=torch.bfloat16, ragged=True, carry=True)
    want = ops.causal_conv(**v, state=state, lengths=lengths, want_state=True)
    wantb = ops.causal_conv_bwd(dy, **v, state=state, lengths=lengths)
    tm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)                                                      # noqa: E731
    buf = torch.zeros(3, 37, 40, dtype=torch.bfloat16, device="cuda")
    buf[..., 5:38] = v["x"]
    for x in (tm(v["x"]), buf[..., 5:38]):
        assert all(torch.equal(a, b) for a, b in zip(ops.causal_conv(x, v["w"], v["bias"], state=state, lengths=lengths, want_state=True), want))
        assert all(torch.equal(a, b) for a, b in zip(ops.causal_conv_bwd(tm(dy), x, v["w"], v["bias"], state=state, lengths=lengths), wantb))
    s1, s2 = state.clone(), state.clone()
    assert torch.equal(ops.causal_conv_step(buf[:, 3, 5:38], v["w"], v["bias"], state=s1),
                       ops.causal_conv_step(buf[:, 3, 5:38].contiguous(), v["w"], v["bias"], state=s2)) and torch.equal(s1, s2)


def test_empty_inputs():
    from avsi_amd import ops
    for B, T in ((0, 5), (3, 0)):
        c, v, dout, state, cstate, _ = _case(B, T, 6, 4, carry=True)
        out, new, kept = ops.selective_scan(**c, state=state, want_state=True, keep=True)
        assert out.shape == (B, T, 6) and torch.equal(new, state)
        g = dict(zip(NAMES, ops.selective_scan_bwd(dout, **c, kept=kept, state=state)))
        assert g["du"].shape == (B, T, 6) and all(bool((g[k] == 0).all()) for k in ("dA", "dD", "ddt_bias"))
        y, ks = ops.causal_conv(**v, state=cstate, want_state=True)
        assert y.shape == (B, T, 6) and torch.equal(ks, cstate)
        dx, dw, db = ops.causal_conv_bwd(dout, **v, state=cstate)
        assert dx.shape == (B, T, 6) and bool((dw == 0).all()) and bool((db == 0).all())
        new = ops.selective_scan(**c, want_state=True)[1]
        assert new.shape == (B, 6, 4) and bool((new == 0).all())
    c, v, _, state, cstate, _ = _case(0, 1, 6, 4, carry=True)
    assert ops.selective_scan_step(**{k: (t[:, 0] if t.dim() >= 3 else t) for k, t in c.items()}, state=state).shape == (0, 6)
    assert ops.causal_conv_step(v["x"][:, 0], v["w"], state=cstate).shape == (0, 6)


def test_graph_replays_and_side_streams():
    from avsi_amd import ops
    c, v, dout, state, cstate, lengths = _case(2, 200, 40, 16, dtype=torch.bfloat16, ragged=True, carry=True)

    def work():
        s = ops.selective_scan(**c, state=state, lengths=lengths, want_state=True, keep=True)
        y = ops.causal_conv(**v, state=cstate, lengths=lengths, want_state=True)
        return (list(s) + list(ops.selective_scan_bwd(dout, **c, kept=s[2], state=state, lengths=lengths)) + list(y)
                + list(ops.causal_conv_bwd(dout, **v, state=cstate, lengths=lengths)))

    def same(a, b):
        # (rows of `kept` behind a length are not written)
        return all(torch.equal(p, q) for i, (p, q) in enumerate(zip(a, b)) if i != 2)
    want = [t.clone() for t in work()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, want)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g1 = work()
    with torch.cuda.graph(other):
        g2 = work()
    for k in range(3):
        for t in (c["u"], v["x"], dout, state):
            t.mul_(-1.0 if k % 2 else 0.5)
        graph.replay()
        eager = [t.clone() for t in work()]
        other.replay()
        torch.cuda.synchronize()
        assert same(g1, eager) and same(g2, eager)


def test_step_in_a_graph_moves_the_state_on():
    from avsi_amd import ops
    c, v, _, state, cstate, _ = _case(4, 1, 50, 16, dtype=torch.bfloat16, carry=True)
    one = {k: (t[:, 0].contiguous() if t.dim() >= 3 else t) for k, t in c.items()}
    s1, k1, s2, k2 = state.clone(), cstate.clone(), state.clone(), cstate.clone()
    x = v["x"][:, 0].contiguous()
    ops.selective_scan_step(**one, state=s1.clone()), ops.causal_conv_step(x, v["w"], state=k1.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.selective_scan_step(**one, state=s1)
        y = ops.causal_conv_step(x, v["w"], state=k1)
    for _ in range(4):
        x.mul_(-0.5)
        one["u"].mul_(-0.5)
        graph.replay()
        o2, y2 = ops.selective_scan_step(**one, state=s2), ops.causal_conv_step(x, v["w"], state=k2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in ((out, o2), (y, y2), (s1, s2), (k1, k2)))
