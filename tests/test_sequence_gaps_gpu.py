"""A closed gate in both directions of the scan, the layer norm's backward pass on a stream beside others, and its gamma's gradient over
more than 2^31 values."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("dtype", [torch.float32, BF16, torch.float16], ids=str)
@pytest.mark.parametrize("T,D", [(20, 33), (200, 70)])
def test_a_gate_of_minus_infinity_closes_its_channel_only(dtype, T, D):
    """-inf times sigmoid(-inf) = 0 is NaN: in that output, in dz and dC of that step, in what reaches back from it (du, ddt of the channel
    and dB, up to that step) and in the channel's sums over time.  Everything else keeps its bits."""
    from avsi_amd import ops
    g = torch.Generator("cuda").manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")                                                         # noqa: E731
    N, b, t, ch = 16, 1, 11, 4
    c = {"u": r(2, T, D).to(dtype), "dt": (r(2, T, D) - 1).to(dtype), "A": -torch.exp(r(D, N)), "B": r(2, T, N).to(dtype),
         "C": r(2, T, N).to(dtype), "D": r(D), "z": r(2, T, D).to(dtype), "dt_bias": 0.3 * r(D)}
    dout = r(2, T, D).to(dtype)

    def run(c):
        out, new, kept = ops.selective_scan(**c, want_state=True, keep=True)
        return dict(zip(("out", "state", "du", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias"),
                        (out, new, *ops.selective_scan_bwd(dout, **c, kept=kept))))
    want = run(c)
    z = c["z"].clone()
    z[b, t, ch] = float("-inf")
    got = run(dict(c, z=z))
    bad = {k: torch.zeros_like(v, dtype=torch.bool) for k, v in want.items()}
    for k in ("out", "dz"):
        bad[k][b, t, ch] = True
    for k in ("du", "ddt"):
        bad[k][b, :t + 1, ch] = True
    bad["dB"][b, :t + 1] = True
    bad["dC"][b, t] = True
    for k in ("dA", "dD", "ddt_bias"):
        bad[k][ch] = True
    for k, v in got.items():
        assert bool(v[bad[k]].isnan().all()), k
        assert torch.equal(v[~bad[k]], want[k][~bad[k]]), k
    # one token
    one = {k: (v[:, t] if v.dim() == 3 else v) for k, v in c.items()}
    state = torch.zeros(2, 2, D, N, device="cuda")
    clean = ops.selective_scan_step(**one, state=state[0])
    closed = ops.selective_scan_step(**dict(one, z=z[:, t]), state=state[1])
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[b, ch] = True
    assert bool(closed[hit].isnan().all()) and torch.equal(closed[~hit], clean[~hit]) and torch.equal(state[0], state[1])


def test_layer_norm_backward_on_a_side_stream():
    from avsi_amd import ops
    x, dy = torch.randn(2, 500, 257, device="cuda").unbind(0)
    gamma = torch.randn(257, device="cuda")
    _, mean, rstd = ops.layer_norm(x, gamma)
    want = ops.layer_norm_bwd(dy, x, mean, rstd, gamma)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.layer_norm_bwd(dy, x, mean, rstd, gamma) for _ in range(3)]
    both = [ops.layer_norm_bwd(dy, x, mean, rstd, gamma) for _ in range(3)]        # (at the same time)
    torch.cuda.synchronize()
    for one in got + both:
        assert len(one) == 3 and all(torch.equal(a, b) for a, b in zip(one, want))


def test_gradient_of_gamma_over_more_than_two_to_the_31_values():
    if torch.cuda.mem_get_info()[0] < 30 * 2 ** 30:
        pytest.skip("needs 30 GiB of free memory")
    from avsi_amd import ops
    M, C = (1 << 21) + 5, 1032
    x, dy = torch.randn(2, M, C, device="cuda", dtype=BF16).unbind(0)
    gamma = torch.randn(C, device="cuda")
    _, mean, rstd = ops.layer_norm(x, gamma)
    dgamma = ops.layer_norm_bwd(dy, x, mean, rstd, gamma)[1]
    want, size = torch.zeros(2, C, dtype=torch.float64, device="cuda").unbind(0)
    for a in range(0, M, 1 << 17):
        k = slice(a, a + (1 << 17))
        terms = dy[k].double() * ((x[k].double() - mean[k, None].double()) * rstd[k, None].double())
        want += terms.sum(0)
        size += terms.abs().sum(0)
    # a term is off by two roundings; 512 workgroups add at most M / 512 + 1 of them one behind the other, then their 512 sums are added
    assert bool(((dgamma.double() - want).abs() <= (M // 512 + 1024 + 2) * 2.0 ** -24 * size).all())
    torch.cuda.empty_cache()
