"""The sequence operators at the calls that are easily got wrong: closed gates, long memories, narrow types, odd strides, repeated calls."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def normal(gpu, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return lambda *s, k=1.0, dtype=torch.float32: (torch.randn(*s, generator=g, device=gpu) * k).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,F", [(3996, 1000, 512), (300, 72, 4100), (4, 1024, 4096)])
def test_ff_same_bits_between_other_calls_and_how_far_from_64(gpu, dtype, M, K, F):
    """A pass gives the same bits at every call, other passes in between; and its 16-bit gradients are off by their own rounding and by that of dg and du, two
    independent errors of one size: sqrt 2 times the norm of the first alone (a twentieth for what both are sampled by)."""
    from videometamaterials_amd import gated_feed_forward
    n = normal(gpu, M)

    def inputs():
        return [n(M, K, dtype=dtype), *(n(F, K, k=K ** -0.5, dtype=dtype) for _ in range(2)), *(n(F, k=0.1, dtype=dtype) for _ in range(2))], n(M, F, dtype=dtype)

    def run(leaves, dh):
        leaves = [v.detach().requires_grad_() for v in leaves]
        h = gated_feed_forward(*leaves, activation="gelu")
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))
    (one, dh), (other, dh2) = inputs(), inputs()
    want = run(one, dh)
    for _ in range(4):
        run(other, dh2)
        assert all(torch.equal(a, b) for a, b in zip(run(one, dh), want))
    if dtype == torch.float32:
        return
    x, wg, wu, bg, bu = (v.double() for v in one)
    lin = torch.nn.functional.linear
    g, u = lin(x, wg, bg), lin(x, wu, bu)
    p = torch.special.ndtr(g)
    dg, du = dh.double() * u * (p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)), dh.double() * g * p
    exact = (g * p * u, dg @ wg + du @ wu, dg.t().contiguous() @ x, du.t().contiguous() @ x)
    for k, (got, w) in enumerate(zip(want, exact)):
        off, alone = float((got.double() - w).norm()), float((w.to(dtype).double() - w).norm())
        assert off < (1.05 if k == 0 else 1.05 * math.sqrt(2)) * alone, k
