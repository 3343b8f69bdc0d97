"""The bfloat16 linear-attention block on fixed inputs against the float64 restatement of
test_linear_block_gpu.py: output and gradients may be twice as far off as a composition whose stages are exact
inside and rounded to bfloat16.  Both round once at the same stages, so their errors are of one size; the factor of
two leaves room for the few first tokens that the norm after the attention makes ill-conditioned, where
the two errors are independent draws."""
import pytest
import torch

from test_linear_block_gpu import _error, _plain, _ref, _weights

pytestmark = pytest.mark.gpu

NAMES = ["norm_weight", "norm_bias", "qkv_weight", "gate_weight", "out_weight"]


@pytest.mark.parametrize("seed", range(4))
def test_as_near_as_the_roundings_allow(cuda, seed):
    from ssm_mamba_b200.linear_block import linear_block_forward
    w = _weights(cuda, torch.bfloat16)
    gen = torch.Generator(device=cuda).manual_seed(seed)
    hidden, dout = (torch.randn(2, 300, 96, generator=gen, device=cuda).bfloat16() for _ in range(2))
    params = [getattr(w, n).requires_grad_() for n in NAMES]

    def run(fn, leaves):
        out = fn(leaves)
        return [out, *torch.autograd.grad(out, leaves, dout.to(out.dtype))]

    fresh = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    got = run(lambda x: linear_block_forward(w, x[0]), [fresh(hidden)] + params)
    plain = run(lambda x: _plain(w, x[0], x[1:]), [fresh(hidden)] + params)
    want = run(lambda x: _ref(w, x[0], x[1:])[0], [hidden.double().requires_grad_()] +
               [p.detach().double().requires_grad_() for p in params])
    for n, a, b, c in zip(["out", "hidden"] + NAMES, got, want, plain):
        assert _error(a, b) <= 2 * _error(c, b), (n, _error(a, b), _error(c, b))
