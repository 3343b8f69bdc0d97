"""Linear attention with a decay for each head (csrc/linattn_*.cu) against its definition in
float64 (tests/linear_attention_ref.py, where the tolerances are derived)."""
import math

import pytest
import torch

from linear_attention_ref import attention, check, inputs

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
SIZES = [(1, 1, 1, 1, 1), (2, 2, 3, 16, 16), (1, 63, 2, 64, 64), (2, 64, 2, 128, 128), (1, 65, 3, 33, 7),
         (2, 127, 2, 80, 96), (1, 128, 4, 64, 128), (2, 129, 1, 128, 64), (1, 300, 5, 100, 37), (2, 257, 2, 8, 120),
         (1, 700, 2, 128, 128), (3, 1000, 2, 64, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("init", [False, True])
def test_forward(cuda, size, dtype, init):
    from ssm_mamba_b200 import linear_attention_fn
    B, L, H, K, V = size
    q, k, v, g, gen = inputs(*size, dtype, cuda, seed=L + K)
    s0 = torch.randn(B, H, K, V, generator=gen, device=cuda) if init else None
    out, last = linear_attention_fn(q, k, v, g, initial_state=s0, return_last_state=True)
    ro, rl = attention(q, k, v, g, K ** -0.5, s0)
    assert out.dtype == dtype and last.dtype == F32
    check(out, ro, "out")
    check(last, rl, "last_state")
    assert torch.equal(linear_attention_fn(q, k, v, g, initial_state=s0), out)


# (heads of q, k, v) of 12
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads", [(12, 4, 4), (3, 3, 12), (12, 1, 6)])
def test_shared_heads_and_gradients(cuda, heads, dtype):
    from ssm_mamba_b200 import linear_attention_fn
    B, L, H, K, V = 2, 200, 12, 48, 64
    q, k, v, g, gen = inputs(B, L, H, K, V, dtype, cuda, seed=5, heads=heads)
    _grads(linear_attention_fn, (q, k, v, g), torch.randn(B, H, K, V, generator=gen, device=cuda), None, True, gen)


def _grads(fn, qkvg, s0, lengths, last, gen, scale=0.3):
    q, k, v, g = qkvg
    leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([s0.detach().requires_grad_()] if s0 is not None else [])
    init = leaves[3] if s0 is not None else None
    out, state = fn(*leaves[:3], g, scale=scale, initial_state=init, lengths=lengths, return_last_state=True)
    ref = [x.detach().double().requires_grad_() for x in leaves]
    ro, rs = attention(*ref[:3], g, scale, ref[3] if s0 is not None else None, lengths)
    dout = torch.randn(out.shape, generator=gen, device=out.device).to(out.dtype)
    dstate = torch.randn(state.shape, generator=gen, device=out.device)
    check(out, ro, "out")
    check(state, rs, "last_state")
    loss, rloss = (out * dout).sum(), (ro * dout.double()).sum()
    del loss
    got = torch.autograd.grad((out, state) if last else (out,), leaves, (dout, dstate) if last else (dout,))
    want = torch.autograd.grad(rloss + ((rs * dstate.double()).sum() if last else 0.0), ref)
    for name, a, b, x in zip(("dq", "dk", "dv", "dinitial_state"), got, want, leaves):
        assert a.dtype == x.dtype
        check(a, b, name)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("last", [False, True])
def test_gradients(cuda, size, dtype, last):
    from ssm_mamba_b200 import linear_attention_fn
    B, L, H, K, V = size
    q, k, v, g, gen = inputs(*size, dtype, cuda, seed=L + V)
    s0 = torch.randn(B, H, K, V, generator=gen, device=cuda) if last else None
    _grads(linear_attention_fn, (q, k, v, g), s0, None, last, gen)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L,lens", [(70, [70, 0, 1, 64]), (333, [0, 333, 129, 128]), (5, [5, 4, 0, 1]),
                                    (200, [-3, 500, 200, 63])])
def test_lengths(cuda, L, lens, dtype):
    """Padded tokens take no part, whatever they hold; a row without tokens keeps its state."""
    from ssm_mamba_b200 import linear_attention_fn
    B, H, K, V = len(lens), 3, 40, 72
    q, k, v, g, gen = inputs(B, L, H, K, V, dtype, cuda, seed=L)
    lengths = torch.tensor(lens, device=cuda)
    s0 = torch.randn(B, H, K, V, generator=gen, device=cuda)
    clean = _grads(linear_attention_fn, (q, k, v, g), s0, lengths, True, torch.Generator(device=cuda).manual_seed(1))
    pad = (torch.arange(L, device=cuda)[None] >= lengths.clamp(0, L)[:, None])[:, :, None, None]
    for bad in (math.nan, math.inf, -torch.finfo(dtype).max):
        dirty = [torch.where(pad, torch.tensor(bad, device=cuda, dtype=dtype), x).requires_grad_() for x in (q, k, v)]
        out, state = linear_attention_fn(*dirty, g, scale=0.3, initial_state=s0, lengths=lengths, return_last_state=True)
        gen1 = torch.Generator(device=cuda).manual_seed(1)
        dout = torch.randn(out.shape, generator=gen1, device=cuda).to(dtype)
        dstate = torch.randn(state.shape, generator=gen1, device=cuda)
        dout = torch.where(pad, torch.tensor(bad, device=cuda, dtype=dtype), dout)
        got = torch.autograd.grad((out, state), dirty, (dout, dstate))
        assert not out.masked_select(pad.expand_as(out)).any()
        for a, b, x in zip(got, clean, (q, k, v)):
            assert not a.masked_select(pad.expand_as(a)).any()
            check(a, b.double(), "gradient with padding", rel=1e-6)
    for b, n in enumerate(lens):
        if n <= 0:
            assert torch.equal(state[b], s0[b])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", [1024, 4097, 3000])
def test_long_rows_are_cut_into_segments(cuda, L, dtype):
    """Few heads: the row runs as segments whose states are folded; also with lengths that end
    inside, before and at the border of a segment."""
    from ssm_mamba_b200 import linear_attention_fn
    q, k, v, g, gen = inputs(1, L, 2, 64, 64, dtype, cuda, seed=L)
    s0 = torch.randn(1, 2, 64, 64, generator=gen, device=cuda)
    _grads(linear_attention_fn, (q, k, v, g), s0, None, True, gen)
    q, k, v, g, gen = inputs(4, L, 2, 32, 48, dtype, cuda, seed=L + 1, heads=(1, 2, 1))
    s0 = torch.randn(4, 2, 32, 48, generator=gen, device=cuda)
    lengths = torch.tensor([L, 0, L // 2 + 3, 512], device=cuda)
    _grads(linear_attention_fn, (q, k, v, g), s0, lengths, True, gen)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decays(cuda, dtype):
    """No decay, decays that leave nothing after one token, a decay of zero, a slight growth."""
    from ssm_mamba_b200 import linear_attention_fn
    decay = torch.tensor([0.0, -1e-6, -0.5, -20.0, -200.0, -3e38, -math.inf, 1e-3], device=cuda)
    q, k, v, g, gen = inputs(2, 333, 8, 32, 32, dtype, cuda, seed=3, decay=decay)
    s0 = torch.randn(2, 8, 32, 32, generator=gen, device=cuda)
    _grads(linear_attention_fn, (q, k, v, g), s0, None, True, gen)
    nan = decay.clone()
    nan[2] = math.nan
    out = linear_attention_fn(q, k, v, nan)
    assert torch.isnan(out[:, 1:, 2]).all() and torch.isfinite(out[:, :, [0, 1, 3, 4, 5, 6, 7]]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(cuda, dtype):
    """Head-major storage, unaligned bases, a channel stride that needs a copy, broadcast rows."""
    from ssm_mamba_b200 import linear_attention_fn
    B, L, H, K, V = 2, 150, 3, 32, 40
    g0 = torch.Generator(device=cuda).manual_seed(2)
    rn = lambda *s: torch.randn(*s, generator=g0, device=cuda).to(dtype)  # noqa: E731
    decay = torch.tensor([-0.01, -0.1, -1.0], device=cuda)
    q = rn(B, H, L, K).transpose(1, 2)                                    # head-major
    k = rn(B, L, H, K + 1)[..., 1:]                                       # odd head stride, unaligned base
    v = rn(B, L, V, H).transpose(2, 3)                                    # channel stride H
    _grads(linear_attention_fn, (q, k, v, decay), None, None, True, g0)
    q1 = rn(1, L, 1, K).expand(B, L, H, K)                                # one row, one head for all
    k1 = rn(B, 1, H, K).expand(B, L, H, K)                                # one token for all
    _grads(linear_attention_fn, (q1, k1, v, decay), None, None, True, g0)
    out = linear_attention_fn(q.detach().requires_grad_(), k, v, decay)
    out.sum().backward()                                                  # a gradient with zero strides


def test_multilinear_differences(cuda):
    """out is linear in each input, so a central difference of any size is its derivative:
    (f(x + d) - f(x - d)) / 2 = <df/dx, d> up to float32 rounding (1e-5 of the terms' size)."""
    from ssm_mamba_b200 import linear_attention_fn
    B, L, H, K, V = 2, 190, 3, 24, 40
    q, k, v, g, gen = inputs(B, L, H, K, V, F32, cuda, seed=11)
    s0 = torch.randn(B, H, K, V, generator=gen, device=cuda)
    xs = [x.contiguous() for x in (q, k, v)] + [s0]
    dout = torch.randn(B, L, H, V, generator=gen, device=cuda)
    dst = torch.randn(B, H, K, V, generator=gen, device=cuda)

    def loss(ys):
        out, st = linear_attention_fn(*ys[:3], g, initial_state=ys[3], return_last_state=True)
        return (out.double() * dout.double()).sum() + (st.double() * dst.double()).sum(), out, st

    leaves = [x.clone().requires_grad_() for x in xs]
    _, out, st = loss(leaves)
    grads = torch.autograd.grad((out, st), leaves, (dout, dst))
    for i, grad in enumerate(grads):
        d = torch.randn(xs[i].shape, generator=gen, device=cuda)
        up, down = (loss([x + s * d if j == i else x for j, x in enumerate(xs)]) for s in (1.0, -1.0))
        want = float((up[0] - down[0]) / 2)
        got = float((grad.double() * d.double()).sum())
        size = float((grad.double() * d.double()).norm())
        assert abs(got - want) <= 1e-4 * size, (i, got, want, size)


def test_no_tokens(cuda):
    from ssm_mamba_b200 import linear_attention_fn
    g = torch.tensor([-0.1, -0.2], device=cuda)
    s0 = torch.randn(3, 2, 8, 4, device=cuda).requires_grad_()
    q = torch.empty(3, 0, 2, 8, device=cuda)
    v = torch.empty(3, 0, 2, 4, device=cuda)
    out, last = linear_attention_fn(q, q, v, g, initial_state=s0, return_last_state=True)
    assert out.shape == (3, 0, 2, 4) and torch.equal(last, s0)
    (d,) = torch.autograd.grad(last, s0, torch.ones_like(last))
    assert torch.equal(d, torch.ones_like(s0))


def test_deterministic_streams_and_graphs(cuda):
    """Equal bits on another stream and from a captured graph."""
    from ssm_mamba_b200 import linear_attention_fn
    q, k, v, g, gen = inputs(1, 2000, 4, 64, 64, BF16, cuda, seed=8, heads=(4, 2, 2))
    dout = torch.randn(1, 2000, 4, 64, generator=gen, device=cuda).to(BF16)

    def step():
        xs = [x.detach().requires_grad_() for x in (q, k, v)]
        out, last = linear_attention_fn(*xs, g, return_last_state=True)
        return (out.detach(), last.detach(), *torch.autograd.grad(out, xs, dout))

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(cuda):
    from ssm_mamba_b200 import linear_attention_fn
    q, k, v, g, _ = inputs(2, 10, 4, 16, 24, BF16, cuda)
    bad = [
        (TypeError, lambda: linear_attention_fn(q.half(), k.half(), v.half(), g)),
        (TypeError, lambda: linear_attention_fn(q, k.float(), v, g)),
        (ValueError, lambda: linear_attention_fn(q, k, v, g.clone().requires_grad_())),
        (TypeError, lambda: linear_attention_fn(q, k, v, g, initial_state=torch.zeros(2, 4, 16, 24, device=cuda).half())),
        (RuntimeError, lambda: linear_attention_fn(q.cpu(), k.cpu(), v.cpu(), g.cpu())),
        (RuntimeError, lambda: linear_attention_fn(q, k, v, g.cpu())),
        (RuntimeError, lambda: linear_attention_fn(q, k[..., :8], v, g)),
        (RuntimeError, lambda: linear_attention_fn(q, k[:, :5], v, g)),
        (RuntimeError, lambda: linear_attention_fn(q, k, v[:, :, :3], g)),
        (RuntimeError, lambda: linear_attention_fn(q[0], k[0], v[0], g)),
        (RuntimeError, lambda: linear_attention_fn(q, k, v, g[:3])),
        (RuntimeError, lambda: linear_attention_fn(q, k, v, g, initial_state=torch.zeros(2, 4, 24, 16, device=cuda))),
        (RuntimeError, lambda: linear_attention_fn(q, k, v, g, lengths=torch.ones(3, device=cuda, dtype=torch.int64))),
        (RuntimeError, lambda: linear_attention_fn(*(torch.zeros(1, 4, 1, 129, device=cuda),) * 3, g[:1])),
    ]
    for err, call in bad:
        with pytest.raises(err):
            call()
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    out = linear_attention_fn(*x, g)
    (dq,) = torch.autograd.grad(out, x[0], torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()                # no second derivative
