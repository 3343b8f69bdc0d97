"""How far a NaN or an infinity in one element reaches: not finite where the definition has neither number
nor zero for it, up to 127 tokens further, and nowhere else (the docstring of linear_attention_fn)."""
import math

import pytest
import torch

from linear_attention_ref import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 96)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["q", "k", "v"])
def test_reach(cuda, where, bad, K, V, dtype):
    from ssm_mamba_b200 import linear_attention_fn
    B, L, H, b, t, h, c = 2, 700, 3, 1, 333, 2, 5
    q, k, v, g, gen = inputs(B, L, H, K, V, dtype, cuda, seed=3)
    dout = torch.randn(B, L, H, V, generator=gen, device=cuda).to(dtype)

    def run(q, k, v):
        xs = [x.detach().clone().requires_grad_() for x in (q, k, v)]
        out, last = linear_attention_fn(*xs, g, return_last_state=True)
        return (out.detach(), last.detach(), *torch.autograd.grad(out, xs, dout))

    clean = run(q, k, v)
    dirty = [x.clone() for x in (q, k, v)]
    x = dirty["qkv".index(where)]
    x[b, t, h, c] = bad
    got = run(*dirty)
    for name, a, r in zip(("out", "last_state", "dq", "dk", "dv"), got, clean):
        assert torch.equal(a[0], r[0]), name                                       # the other batch row
        heads = a[1].transpose(0, 1) if name != "last_state" else a[1]
        rheads = r[1].transpose(0, 1) if name != "last_state" else r[1]
        assert torch.equal(heads[:2], rheads[:2]), name                            # the other heads
    out, last = got[0][b, :, h], got[1][b, h]
    rout, rlast = clean[0][b, :, h], clean[1][b, h]
    if where == "q":
        assert torch.equal(last, rlast) and not torch.isfinite(out[t]).any()
        rows = torch.arange(L, device=cuda) != t
        assert torch.equal(out[rows], rout[rows])
    else:
        column = (slice(None), c) if where == "v" else (c,)
        assert not torch.isfinite(last[column]).any()
        assert torch.equal(out[:t - 127], rout[:t - 127])
        late = out[t:t + 100, c] if where == "v" else out[t:t + 100]
        assert not torch.isfinite(late).any()
