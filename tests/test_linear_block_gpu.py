"""A residual linear-attention block (ssm_mamba_b200.linear_block) against a float64 torch
restatement: output, gradients, prompt-to-decode hand-over, decoding from a CUDA graph.
Relative 2-norm tolerances: float32 1e-5 and gradients 5e-5 (two norms and two projections
multiply the operators' 1e-5); bfloat16 1e-2 (seven roundings of 1.7e-3, one after each stage,
and 4e-3 of the attention).

The norm after the attention makes some gradients ill-conditioned whatever computes them: the first
token's output is (q . k) v, whose direction does not depend on q . k, so the gradient with respect to
q . k is a small difference divided by it.  With q . k near zero the roundings of the stages alone
move the gradient of hidden by 2% and more (one random input in twelve in bfloat16), so gradients are
allowed twice the error of a torch composition with the same roundings on top."""
import pytest
import torch
import torch.nn.functional as F

from linear_attention_ref import attention

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _weights(dev, dtype, model=96, q_heads=4, k_heads=2, v_heads=2, dk=32, dv=48, heads=4):
    from ssm_mamba_b200.linear_block import LinearBlockWeights
    g = torch.Generator(device=dev).manual_seed(3)
    r = lambda *s, sc=0.1: (torch.randn(*s, device=dev, generator=g) * sc)  # noqa: E731
    return LinearBlockWeights(
        norm_weight=1 + r(model), norm_bias=r(model),
        qkv_weight=r(q_heads * dk + k_heads * dk + v_heads * dv, model).to(dtype),
        gate_weight=r(heads * dv, model).to(dtype), out_weight=r(model, heads * dv).to(dtype),
        log_decay=-torch.exp2(-8.0 * torch.arange(1, heads + 1, device=dev, dtype=F32) / heads),
        q_heads=q_heads, k_heads=k_heads, v_heads=v_heads, dk=dk, dv=dv)


def _ref(w, hidden, params, state=None, lengths=None):
    nw, nb, qkv, gate, out = params
    norm = lambda t: F.layer_norm(t, (t.shape[-1],))  # noqa: E731
    x = norm(hidden) * nw + nb
    q, k, v = w.split(F.linear(x, qkv))
    o, last = attention(q, k, v, w.log_decay, w.dk ** -0.5, state, lengths)
    return hidden + F.linear(norm(o).flatten(-2) * F.silu(F.linear(x, gate)), out), last


def _plain(w, hidden, params):
    """The block with every stage exact inside and rounded to the stream type."""
    nw, nb, qkv, gate, out = params
    norm = lambda t: F.layer_norm(t.double(), (t.shape[-1],))  # noqa: E731
    x = (norm(hidden) * nw + nb).to(hidden.dtype)
    q, k, v = (t.double() for t in w.split(F.linear(x, qkv)))
    o, _ = attention(q, k, v, w.log_decay, w.dk ** -0.5, None, None)
    o = norm(o.to(hidden.dtype)).to(hidden.dtype)
    return hidden + F.linear(o.flatten(-2) * F.silu(F.linear(x, gate)), out)


def _error(a, b):
    return float((a.detach().double() - b.detach().double()).norm() / b.detach().double().norm())


def _near(a, b, rel, name=""):
    err = _error(a, b)
    assert err <= rel, (name, err)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forward_and_gradients(cuda, dtype):
    from ssm_mamba_b200.linear_block import linear_block_forward
    w = _weights(cuda, dtype)
    hidden = torch.randn(2, 300, 96, device=cuda).to(dtype)
    names = ["norm_weight", "norm_bias", "qkv_weight", "gate_weight", "out_weight"]
    for n in names:
        getattr(w, n).requires_grad_()
    h = hidden.clone().requires_grad_()
    out = linear_block_forward(w, h)
    dout = torch.randn_like(out)
    got = torch.autograd.grad(out, [h] + [getattr(w, n) for n in names], dout)
    ref = [hidden.double().requires_grad_()] + [getattr(w, n).detach().double().requires_grad_() for n in names]
    want_out, _ = _ref(w, ref[0], ref[1:])
    want = torch.autograd.grad(want_out, ref, dout.double())
    _near(out, want_out, 1e-5 if dtype == F32 else 1e-2, "out")
    again = [hidden.clone().requires_grad_()] + [getattr(w, n) for n in names]
    rounded = torch.autograd.grad(_plain(w, again[0], again[1:]), again, dout)
    for n, a, b, c in zip(["hidden"] + names, got, want, rounded):
        _near(a, b, (5e-5 if dtype == F32 else 2e-2) + 2 * _error(c, b), n)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prompt_then_decode(cuda, dtype):
    from ssm_mamba_b200.decode import GraphedStep
    from ssm_mamba_b200.linear_block import LinearBlockCache, linear_block_forward, linear_block_step
    w = _weights(cuda, dtype)
    params = [p.double() for p in (w.norm_weight, w.norm_bias, w.qkv_weight, w.gate_weight, w.out_weight)]
    lengths = torch.tensor([130, 5, 0], device=cuda)
    hidden = torch.randn(3, 140, 96, device=cuda).to(dtype)
    cache = LinearBlockCache.zeros(w, 3)
    with torch.no_grad():
        out = linear_block_forward(w, hidden, lengths, cache)
        want, last = _ref(w, hidden.double(), params, lengths=lengths)
        live = torch.arange(140, device=cuda)[None] < lengths[:, None]
        _near(out[live], want[live], 1e-5 if dtype == F32 else 1e-2)
        _near(cache.state, last, 1e-5 if dtype == F32 else 1e-2)
        step = GraphedStep(lambda t: linear_block_step(w, cache, t), [hidden[:, 0].contiguous()], preserve=[cache.state])
        rows = torch.arange(3, device=cuda)
        for i in range(4):
            token = hidden[rows, lengths + i].contiguous()
            got = step(token).clone()
            want, _ = _ref(w, hidden.double(), params, lengths=lengths + i + 1)
            _near(got, want[rows, lengths + i], 1e-5 if dtype == F32 else 1e-2, i)
