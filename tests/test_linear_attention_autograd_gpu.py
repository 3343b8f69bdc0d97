"""What autograd sees of the linear-attention operators beyond their gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(cuda, seed=0, T=20):
    g = torch.Generator(device=cuda).manual_seed(seed)
    q, k, v = (torch.randn(2, T, 3, n, generator=g, device=cuda) for n in (16, 16, 24))
    return q, k, v, torch.tensor([-0.1, -0.5, 0.0], device=cuda), torch.randn(2, 3, 16, 24, generator=g, device=cuda)


def test_decode_step_counts_as_in_place_change(cuda):
    from ssm_mamba_b200 import linear_attention_fn, linear_attention_update
    q, k, v, g, state = _inputs(cuda)
    before = state._version
    linear_attention_update(state[1:], q[1:, 0], k[1:, 0], v[1:, 0], g)          # a view shares its base's version
    assert state._version > before
    x = q.clone().requires_grad_()
    out = linear_attention_fn(x, k, v, g, initial_state=state)                   # saves the state
    linear_attention_update(state, q[:, 0], k[:, 0], v[:, 0], g)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    with torch.inference_mode():
        fixed = state.clone()
        linear_attention_update(fixed, q[:, 0], k[:, 0], v[:, 0], g)
    linear_attention_update(fixed, q[:, 1], k[:, 1], v[:, 1], g)                 # has no version, and needs none
    for t in range(2):
        linear_attention_update(state, q[:, t], k[:, t], v[:, t], g)
    assert torch.equal(state, fixed)


def test_decode_step_has_no_silent_gradient(cuda):
    from ssm_mamba_b200 import linear_attention_fn, linear_attention_update
    q, k, v, g, state = _inputs(cuda)
    want = linear_attention_update(state.clone(), q[:, 0], k[:, 0], v[:, 0], g)
    for i in range(3):
        xs = [t[:, 0].clone() for t in (q, k, v)]
        xs[i].requires_grad_()
        new = state.clone()
        out = linear_attention_update(new, *xs, g)
        assert torch.equal(out, want) and not new.requires_grad
        with pytest.raises(RuntimeError, match="not differentiable"):
            out.sum().backward()
        with torch.no_grad():
            assert not linear_attention_update(new, *xs, g).requires_grad
    x = q.clone().requires_grad_()
    _, last = linear_attention_fn(x, k, v, g, initial_state=state, return_last_state=True)
    for s in (last, state.clone().requires_grad_()):
        before = s.detach().clone()
        with pytest.raises(ValueError, match="detach"):
            linear_attention_update(s, q[:, 0], k[:, 0], v[:, 0], g)
        assert torch.equal(s, before)                          # refused before it is written
        out = linear_attention_update(s.detach(), q[:, 0], k[:, 0], v[:, 0], g)
        with torch.no_grad():
            linear_attention_update(s, q[:, 0], k[:, 0], v[:, 0], g)
        assert not out.requires_grad and not torch.equal(s, before)


def test_log_decay_that_requires_a_gradient(cuda):
    """Refused where a gradient could be asked for, and a constant where none is."""
    from ssm_mamba_b200 import linear_attention_fn, linear_attention_update
    q, k, v, g, state = _inputs(cuda)
    want = linear_attention_fn(q, k, v, g, initial_state=state)
    one = linear_attention_update(state.clone(), q[:, 0], k[:, 0], v[:, 0], g)
    for p in (torch.nn.Parameter(g), torch.nn.Parameter(g.bfloat16().double())):
        for call in (lambda: linear_attention_fn(q, k, v, p, initial_state=state),
                     lambda: linear_attention_update(state.clone(), q[:, 0], k[:, 0], v[:, 0], p)):
            with pytest.raises(ValueError, match="log_decay"):
                call()
            with torch.no_grad():
                got = call()
            with torch.inference_mode():
                assert torch.equal(call(), got)
            if p.dtype == torch.float32:
                assert torch.equal(got, want if got.dim() == 4 else one)
