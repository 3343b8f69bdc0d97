"""A linear-attention block (ssm_mamba_b200.linear_block) trained through a cache, against the float64
restatement of test_linear_block_gpu.py; tolerances as there (float32: 1e-5, gradients 5e-5)."""
import pytest
import torch

from test_linear_block_gpu import _near, _ref, _weights

pytestmark = pytest.mark.gpu

NAMES = ["norm_weight", "norm_bias", "qkv_weight", "gate_weight", "out_weight"]


def test_training_through_a_cache(cuda):
    """Two pieces of a sequence, one backward over both; the state between them is a constant."""
    from ssm_mamba_b200.linear_block import LinearBlockCache, linear_block_forward, linear_block_step
    w = _weights(cuda, torch.float32)
    gen = torch.Generator(device=cuda).manual_seed(7)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    pieces, douts = [rn(2, 150, 96), rn(2, 70, 96)], [rn(2, 150, 96), rn(2, 70, 96)]
    lengths = torch.tensor([150, 97], device=cuda)
    start = rn(2, 4, 32, 48)
    params = [getattr(w, n).requires_grad_() for n in NAMES]
    cache = LinearBlockCache(start.clone())
    xs = [p.clone().requires_grad_() for p in pieces]
    outs = [linear_block_forward(w, xs[0], lengths, cache), linear_block_forward(w, xs[1], None, cache)]
    assert not cache.state.requires_grad
    ref = [p.detach().double().requires_grad_() for p in params]
    rx = [p.double().requires_grad_() for p in pieces]
    want0, state = _ref(w, rx[0], ref, start, lengths)
    want1, end = _ref(w, rx[1], ref, state.detach())
    live = (torch.arange(150, device=cuda)[None] < lengths[:, None])[..., None].float()
    _near(outs[0] * live, want0 * live, 1e-5, "first")
    _near(outs[1], want1, 1e-5, "second")
    _near(cache.state, end, 1e-5, "state")
    got = torch.autograd.grad(outs, xs + params, [douts[0] * live, douts[1]])
    want = torch.autograd.grad([want0, want1], rx + ref, [(douts[0] * live).double(), douts[1].double()])
    for n, a, b in zip(["first", "second"] + NAMES, got, want):
        _near(a, b, 5e-5, n)
    # generation goes on in grad mode too
    token = rn(2, 96)
    before = cache.state.clone()
    linear_block_step(w, cache, token)
    with torch.no_grad():
        again = LinearBlockCache(before)
        linear_block_step(w, again, token)
    assert torch.equal(cache.state, again.state) and not cache.state.requires_grad


def test_a_cache_that_requires_a_gradient_is_refused(cuda):
    from ssm_mamba_b200.linear_block import LinearBlockCache, linear_block_forward
    w = _weights(cuda, torch.float32)
    hidden = torch.zeros(1, 5, 96, device=cuda)
    cache = LinearBlockCache.zeros(w, 1)
    cache.state.requires_grad_()
    with pytest.raises(ValueError, match="cache"):
        linear_block_forward(w, hidden, cache=cache)
    with torch.no_grad():
        linear_block_forward(w, hidden, cache=cache)
