"""Linear attention of bfloat16 streams rounds once, at the end: outputs and gradients are as far from the
float64 definition as that definition's own results are when rounded to bfloat16.

Tolerance: inside, every operand of a product carries at least 16 bits (2^-16 = 1.5e-5 of itself), so a
result of random sums is off by well under 1e-4 of its norm before it is rounded.  The rounding itself costs
r = 1.6e-3; sqrt(r^2 + (1e-4)^2) = 1.002 r, and 1.02 r is allowed."""
import pytest
import torch

from linear_attention_ref import attention, inputs

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _distance(a, b):
    return float((a.detach().double() - b.detach().double()).norm())


# widths of all four kernels; a row without and with another in front of it, shared heads, whole chunks and parts
@pytest.mark.parametrize("K,V", [(64, 64), (48, 37), (128, 128), (100, 80), (128, 64), (64, 128)])
@pytest.mark.parametrize("B,L,H,shared", [(2, 500, 4, False), (1, 1100, 6, True), (3, 128, 60, False)])
def test_one_rounding(cuda, B, L, H, shared, K, V):
    from ssm_mamba_b200 import linear_attention_fn
    q, k, v, g, gen = inputs(B, L, H, K, V, BF16, cuda, seed=K + V + L, heads=(H, H // 2, 2) if shared else (None,) * 3)
    s0 = torch.randn(B, H, K, V, generator=gen, device=cuda)
    xs = [x.detach().requires_grad_() for x in (q, k, v)]
    out = linear_attention_fn(*xs, g, initial_state=s0)
    ref = [x.detach().double().requires_grad_() for x in (q, k, v)]
    want, _ = attention(*ref, g, K ** -0.5, s0)
    dout = torch.randn(out.shape, generator=gen, device=cuda).to(BF16)
    got = (out, *torch.autograd.grad(out, xs, dout))
    want = (want, *torch.autograd.grad(want, ref, dout.double()))
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        rounding = _distance(b.to(BF16), b)
        assert _distance(a, b) <= 1.02 * rounding, (name, _distance(a, b) / float(b.norm()), rounding / float(b.norm()))
