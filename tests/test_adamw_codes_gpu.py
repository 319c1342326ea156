"""The moments of AdamW take one rounding per operation in the order of the formula, so a program that evaluates it in elementary float32
operations holds the very same moments, scales and codes, step after step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BLOCK = 256


def _encode(x, root):
    x = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    y = x * torch.where(top > 0, (1 / top) * 448, torch.zeros_like(top)).clamp(max=torch.finfo(torch.float32).max)
    if root:
        y = torch.where((x > 0) & (y < 2.0 ** -9), torch.full_like(y, 2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn), top[:, 0] * (1 / 448)


def _decode(code, scale, n):
    return (code.float() * scale[:, None]).reshape(-1)[:n]


@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_moments_equal_those_of_elementary_operations(bits, gdtype):
    from avsi_amd import ops
    b1, b2, scale = 0.9, 0.999, 0.3
    gen = torch.Generator(device="cuda").manual_seed(bits)
    sizes = [2_000_003, 300, 1]
    size = [torch.exp(2 * torch.randn(n, generator=gen, device="cuda")) for n in sizes]
    grads = [torch.empty(n, device="cuda", dtype=gdtype) for n in sizes]
    plan = ops.AdamwPlan([torch.zeros(n, device="cuda") for n in sizes], grads, bits=bits)
    m, v = [torch.zeros(n, device="cuda") for n in sizes], [torch.zeros(n, device="cuda") for n in sizes]
    for step in range(1, 9):
        for i, g in enumerate(grads):
            g.copy_(size[i] * torch.randn(sizes[i], generator=gen, device="cuda"))
        ops.adamw(plan, step, 1e-3, beta1=b1, beta2=b2, grad_scale=scale)
        for i, (n, o) in enumerate(zip(sizes, plan.offsets)):
            g = grads[i].float() * scale
            m[i] = b1 * m[i] + (1 - b1) * g
            v[i] = b2 * v[i] + (1 - b2) * g * g
            if bits == 32:
                assert torch.equal(plan.state["m"][o:o + n], m[i]) and torch.equal(plan.state["v"][o:o + n], v[i]), (step, i)
                continue
            for k, x, root in (("m", m[i], False), ("v", torch.sqrt(v[i]), True)):
                code, s = _encode(x, root)
                blocks = slice(o // BLOCK, o // BLOCK + len(s))
                assert torch.equal(plan.state[k + "_scale"][blocks], s), (step, i, k)
                assert torch.equal(plan.state[k][o:o + n].float(), code.float().reshape(-1)[:n]), (step, i, k)
                x = _decode(code, s, n)
                (m if k == "m" else v)[i] = x if k == "m" else x.square()
