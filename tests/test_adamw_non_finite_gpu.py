"""8-bit moments: a block of v that has become infinite reads as NaN, all of it, and says so in the next step's weights; the moments of
m and the other blocks go on."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# (1 - beta2) g g with beta2 = 0.999: 9e35 for 3e19, inside the range; 1e39 for 1e21, beyond the largest float 3.4e38
@pytest.mark.parametrize("bad,nan_in", [(3e19, ""), (1e21, "v"), (float("inf"), "mv"), (float("nan"), "mv")])
def test_a_block_of_an_infinite_v_reads_as_nan(bad, nan_in):
    from avsi_amd import ops
    n = 1000
    g = torch.randn(n, generator=torch.Generator().manual_seed(3)).cuda()
    g[700:800] = 0
    w, w2 = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    plan, clean = ops.AdamwPlan([w], [g.clone()], bits=8), ops.AdamwPlan([w2], [g], bits=8)
    ops.adamw(clean, 1, 1e-3)
    plan._grads[0][600] = bad                        # the third block, values 512 .. 767
    ops.adamw(plan, 1, 1e-3)
    block = torch.zeros(n, dtype=torch.bool, device="cuda")
    block[512:768] = True
    read = lambda p, k: p.state[k].float() * p.state[k + "_scale"].repeat_interleave(256)                              # noqa: E731
    for k in ("m", "v"):
        got, want = read(plan, k)[:n], read(clean, k)[:n]
        assert torch.equal(got[~block], want[~block]), k
        assert bool(got[block].isnan().all() if k in nan_in else got[block].isfinite().all()), k
    plan._grads[0][600] = 0
    ops.adamw(plan, 2, 1e-3), ops.adamw(clean, 2, 1e-3)
    assert bool(w[block].isnan().all() if nan_in else w[block].isfinite().all()) and torch.equal(w[~block], w2[~block])
