"""One decode step of linear attention (csrc/linattn_update.cu) against its definition in
float64.  Tolerances as in linear_attention_ref.py; the state, two float32 roundings from its
inputs, to 1e-6 (the decay's exp2 adds 2^-22)."""
import math

import pytest
import torch

from linear_attention_ref import check

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _ref(state, q, k, v, g, scale):
    H = g.numel()
    q, k, v = (x.double().repeat_interleave(H // x.shape[1], dim=1) for x in (q, k, v))
    new = torch.exp(g.double())[:, None, None] * state.double() + k[..., :, None] * v[..., None, :]
    return scale * torch.einsum("bhk,bhkv->bhv", q, new), new


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (1, 12, 64, 64), (3, 4, 128, 128), (2, 3, 33, 7), (2, 2, 1, 128),
                                  (5, 6, 16, 16), (2, 4, 100, 36), (2, 4, 128, 12), (3, 2, 80, 97), (70, 5, 48, 96)])
@pytest.mark.parametrize("shared", [False, True])
def test_step(cuda, size, dtype, shared):
    from ssm_mamba_b200 import linear_attention_update
    B, H, K, V = size
    gen = torch.Generator(device=cuda).manual_seed(H * K + V)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    J = 1 if shared else H
    # column blocks of one projection
    q, k, v = rn(B, H * K + J * K + J * V).to(dtype).split([H * K, J * K, J * V], dim=-1)
    q, k, v = q.unflatten(-1, (H, K)), k.unflatten(-1, (J, K)), v.unflatten(-1, (J, V))
    g = -torch.rand(H, generator=gen, device=cuda)
    if H > 1:
        g[0], g[1] = 0.0, -math.inf
    state = rn(B, H, K, V)
    for _ in range(3):
        want, new = _ref(state, q, k, v, g, K ** -0.5)
        out = linear_attention_update(state, q, k, v, g)
        assert out.dtype == dtype and out.shape == (B, H, V)
        check(out, want, "out")
        check(state, new, "state", rel=1e-6)


def test_state_views(cuda):
    """A state that is a slice of a larger cache, with odd strides, and nothing else written."""
    from ssm_mamba_b200 import linear_attention_update
    gen = torch.Generator(device=cuda).manual_seed(4)
    for V, off in ((64, 0), (64, 1), (30, 2)):
        cache = torch.randn(4, 6, 40, 80, generator=gen, device=cuda)
        before = cache.clone()
        state = cache[1:3, ::2, 4:36, off:off + V]
        q, k = (torch.randn(2, 3, 32, generator=gen, device=cuda) for _ in range(2))
        v = torch.randn(2, 3, V, generator=gen, device=cuda)
        g = torch.tensor([-0.1, -0.2, -0.3], device=cuda)
        want, new = _ref(state, q, k, v, g, 2.0)
        check(linear_attention_update(state, q, k, v, g, scale=2.0), want, "out")
        check(state, new, "state", rel=1e-6)
        before[1:3, ::2, 4:36, off:off + V] = cache[1:3, ::2, 4:36, off:off + V]
        assert torch.equal(before, cache)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_continues_a_prompt(cuda, dtype):
    """Prompt with lengths, then tokens one by one, equals the whole sequence at once."""
    from ssm_mamba_b200 import linear_attention_fn, linear_attention_update
    B, L, T, H, K, V = 3, 150, 6, 4, 64, 32
    gen = torch.Generator(device=cuda).manual_seed(6)
    q, k = (torch.randn(B, L, H, K, generator=gen, device=cuda).to(dtype) for _ in range(2))
    v = torch.randn(B, L, H, V, generator=gen, device=cuda).to(dtype)
    g = torch.tensor([-1.0, -0.1, -0.01, 0.0], device=cuda)
    lengths = torch.tensor([L - T, 0, 71], device=cuda)
    whole, end = linear_attention_fn(q, k, v, g, lengths=lengths + T, return_last_state=True)
    _, state = linear_attention_fn(q, k, v, g, lengths=lengths, return_last_state=True)
    rows = torch.arange(B, device=cuda)
    for i in range(T):
        at = lengths + i
        out = linear_attention_update(state, q[rows, at], k[rows, at], v[rows, at], g)
        check(out, whole[rows, at].double(), "token", rel=1e-5 if dtype == F32 else 6e-3)   # both sides rounded
    check(state, end.double(), "state", rel=2e-5)


def test_graph_and_empty(cuda):
    from ssm_mamba_b200 import linear_attention_update
    gen = torch.Generator(device=cuda).manual_seed(9)
    state = torch.randn(4, 8, 64, 64, generator=gen, device=cuda)
    q, k, v = (torch.randn(4, 8, 64, generator=gen, device=cuda).to(BF16) for _ in range(3))
    g = -torch.rand(8, generator=gen, device=cuda)
    s1, s2 = state.clone(), state.clone()
    outs = [linear_attention_update(s1, q, k, v, g) for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [linear_attention_update(s2, q, k, v, g) for _ in range(3)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(s1, s2) and all(torch.equal(a, b) for a, b in zip(outs, got))
    out = linear_attention_update(state[:0], q[:0], k[:0], v[:0], g)
    assert out.shape == (0, 8, 64)


def test_refusals(cuda):
    from ssm_mamba_b200 import linear_attention_update
    s = torch.zeros(2, 4, 16, 24, device=cuda)
    q, k, v = (torch.zeros(2, 4, n, device=cuda) for n in (16, 16, 24))
    g = torch.zeros(4, device=cuda)
    bad = [
        (TypeError, lambda: linear_attention_update(s, q.half(), k.half(), v.half(), g)),
        (TypeError, lambda: linear_attention_update(s, q, k, v.bfloat16(), g)),
        (ValueError, lambda: linear_attention_update(s, q, k, v, g.clone().requires_grad_())),
        (RuntimeError, lambda: linear_attention_update(s.bfloat16(), q, k, v, g)),
        (RuntimeError, lambda: linear_attention_update(s.transpose(2, 3), q, k, v, g)),
        (RuntimeError, lambda: linear_attention_update(s, q[:, :3], k, v, g)),
        (RuntimeError, lambda: linear_attention_update(s, q, k[..., :8], v, g)),
        (RuntimeError, lambda: linear_attention_update(s, q, k, v, g[:2])),
        (RuntimeError, lambda: linear_attention_update(s.cpu(), q.cpu(), k.cpu(), v.cpu(), g.cpu())),
        (RuntimeError, lambda: linear_attention_update(torch.zeros(1, 1, 129, 8, device=cuda),
                                                       *(torch.zeros(1, 1, n, device=cuda) for n in (129, 129, 8)), g[:1])),
    ]
    for err, call in bad:
        with pytest.raises(err):
            call()
