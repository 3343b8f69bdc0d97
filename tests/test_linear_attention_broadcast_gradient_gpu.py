"""Gradients of sums: the incoming gradient has strides of zero and no element stride.  Values against the float64
definition (tests/linear_attention_ref.py, where the tolerances are derived)."""
import pytest
import torch

from linear_attention_ref import attention, check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(6, 6, 6), (6, 3, 2)])
@pytest.mark.parametrize("over", ["all", "channels", "tokens", "state"])
def test_gradient_of_a_sum(cuda, over, heads, dtype):
    from ssm_mamba_b200 import linear_attention_fn
    B, L, H, K, V = 2, 150, 6, 32, 40
    q, k, v, g, gen = inputs(B, L, H, K, V, dtype, cuda, seed=13, heads=heads)
    s0 = torch.randn(B, H, K, V, generator=gen, device=cuda)
    weight = torch.randn(B, L, H, V, generator=gen, device=cuda)
    weight = {"all": weight[:1, :1, :1, :1], "channels": weight[..., :1], "tokens": weight[:, :1]}.get(over)

    def loss(out, last):
        if over == "state":
            return last.sum()
        return (out * weight.to(out.dtype).expand_as(out)).sum() if over != "all" else out.sum()

    xs = [x.detach().requires_grad_() for x in (q, k, v, s0)]
    loss(*linear_attention_fn(*xs[:3], g, initial_state=xs[3], return_last_state=True)).backward()
    ref = [x.detach().double().requires_grad_() for x in (q, k, v, s0)]
    # the weights as the stream type has them
    if weight is not None:
        weight = weight.to(dtype)
    loss(*attention(*ref[:3], g, K ** -0.5, ref[3])).backward()
    for name, a, b in zip("qkvs", xs, ref):
        check(a.grad, torch.zeros_like(b) if b.grad is None else b.grad, "d" + name)     # none: q, of the state's sum
