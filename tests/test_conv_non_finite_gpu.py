"""Infinities and NaN in the inputs of the causal convolution reach the gradients of the taps that see them, and no others: behind a
sequence's end and a thread's run of steps nothing is multiplied by them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(B, T, D, K, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)                                                                        # noqa: E731
    return r(B, T, D).to(dtype).cuda(), r(B, T, D).to(dtype).cuda(), r(D, K).cuda(), r(D).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("B,T,D,K", [(1, 37, 64, 4), (2, 16, 3, 2), (3, 90, 65, 8), (2, 8, 130, 3)])
def test_the_last_input_belongs_to_one_tap(dtype, B, T, D, K):
    from avsi_amd import ops
    x, dy, w, bias = _case(B, T, D, K, T, dtype)
    want = ops.causal_conv_bwd(dy, x, w, bias, silu=False)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[-1, T - 1, 1] = bad
        dx, dw, dbias = ops.causal_conv_bwd(dy, y, w, bias, silu=False)
        assert torch.equal(dx, want[0]) and torch.equal(dbias, want[2])
        hit = torch.zeros_like(dw, dtype=torch.bool)
        hit[1, K - 1] = True
        assert torch.equal(dw[~hit], want[1][~hit])
        assert dw[1, K - 1].isnan() if bad != bad else float(dw[1, K - 1]) == bad * float(dy[-1, T - 1, 1].sign())


@pytest.mark.parametrize("ragged", [False, True])
def test_an_infinite_input_anywhere(ragged):
    """One infinite input per channel, each at another step: a tap's gradient is infinite with the sign of the output gradient that it
    meets there, or finite where that lies outside of the sequence."""
    from avsi_amd import ops
    T, K = 70, 4
    x, dy, w, _ = _case(1, T, T, K, 5, torch.float32)
    n = 61 if ragged else T
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda") if ragged else None
    want = ops.causal_conv_bwd(dy, x, w, silu=False, lengths=lengths)[1]
    y = x.clone()
    y[0].fill_diagonal_(float("inf"))
    dw = ops.causal_conv_bwd(dy, y, w, silu=False, lengths=lengths)[1]
    for p in range(T):
        for k in range(K):
            t = p + K - 1 - k                   # the step whose tap k is input p
            if p < n and t < n:
                assert float(dw[p, k]) == float(dy[0, t, p].sign()) * float("inf"), (p, k)
            else:
                assert float(dw[p, k]) == float(want[p, k]), (p, k)
