"""Rows of many chunks cut into few segments (bfloat16 streams): the state of a segment is a sum over all of
its tokens, held and added in float32 with rounding.

k and v have a positive mean, so the sums grow without cancelling and an error of one sign in each addition
would show.  Tolerances of linear_attention_ref.py: states 1e-5.  Within a chunk the tensor core adds 40
products at the sum's full size, each cut off by at most 2^-23 of it and by half of that on average (2.4e-6); the
additions of chunks and segments round to nearest (2^-24 each, of either sign).  Outputs: the rounding to
bfloat16 and that error, 1.02 times the rounding alone."""
import pytest
import torch

from linear_attention_ref import check

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _by_chunks(q, k, v, g, scale, dout=None, chunk=1024):
    """(out, last state) in float64 by the recurrence over chunks, one batch row."""
    q, k, v = (x[0].double().transpose(0, 1) for x in (q, k, v))               # (H, L, d)
    H, L, K = k.shape
    t = torch.arange(chunk, device=q.device, dtype=torch.float64)
    g = g.double()[:, None, None]
    near = torch.where(t[:, None] >= t[None], torch.exp(g * (t[:, None] - t[None]).clamp(min=0)), 0.0)
    state = torch.zeros(H, K, v.shape[2], device=q.device, dtype=torch.float64)
    outs = []
    for i in range(0, L, chunk):
        a, b, c = q[:, i:i + chunk], k[:, i:i + chunk], v[:, i:i + chunk]
        n = a.shape[1]
        outs.append(((a @ b.transpose(1, 2)) * near[:, :n, :n]) @ c + torch.exp(g[:, 0] * (t[:n] + 1))[..., None] * (a @ state))
        state = torch.exp(g * n) * state + (b * torch.exp(g[:, 0] * (n - 1 - t[:n]))[..., None]).transpose(1, 2) @ c
    return scale * torch.cat(outs, dim=1).transpose(0, 1)[None], state[None]


@pytest.mark.parametrize("K,V", [(64, 64), (128, 128), (128, 48)])
@pytest.mark.parametrize("log_decay", [0.0, -1e-5, -1e-3])
def test_state_of_long_segments(cuda, K, V, log_decay):
    from ssm_mamba_b200 import linear_attention_fn
    L, H, scale = 200_000, 2, 2.0 ** -20
    gen = torch.Generator(device=cuda).manual_seed(K + V)
    q = torch.randn(1, L, H, K, generator=gen, device=cuda).to(BF16)
    k, v = ((1 + torch.randn(1, L, H, n, generator=gen, device=cuda)).to(BF16) for n in (K, V))
    g = torch.tensor([log_decay, log_decay / 2], device=cuda)
    xs = [x.requires_grad_() for x in (q, k, v)]
    out, last = linear_attention_fn(*xs, g, scale=scale, return_last_state=True)
    want, end = _by_chunks(q.detach(), k.detach(), v.detach(), g, scale)
    check(last, end, "last_state")
    d = (out.double() - want).norm()
    assert d <= 1.02 * (want.to(BF16).double() - want).norm(), float(d / want.norm())
    # dv_t = scale sum_{s >= t} w^(s - t) (k_t . q_s) dout_s: the same recurrence from the last token on
    dout = (1 + torch.randn(1, L, H, V, generator=gen, device=cuda)).to(BF16)
    with torch.no_grad():
        q += 1                                       # of one sign too
    out = linear_attention_fn(*xs, g, scale=scale)
    (dv,) = torch.autograd.grad(out, xs[2], dout)
    want = _by_chunks(k.detach().flip(1), q.detach().flip(1), dout.flip(1), g, scale)[0].flip(1)
    d = (dv.double() - want).norm()
    assert d <= 1.02 * (want.to(BF16).double() - want).norm(), float(d / want.norm())
