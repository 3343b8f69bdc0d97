"""Linear attention with a decay for each head in float64, from its definition as one masked
product (differentiable through autograd), and the checks that its tests share.

Tolerances, as relative 2-norm errors, from the arithmetic of each stream type:
  * float32: 1e-5.  Products and sums in float32 (2^-24 each, sums of up to a few thousand
    terms of random sign) and decays from exp2 (2^-22): a few 1e-7, times the cancellation of
    sums whose terms are larger than they are.
  * bfloat16 outputs: 4e-3.  Rounding a result to bfloat16 costs 1.7e-3 (2^-9 over a mantissa
    spread evenly); the decayed scores and the state are rounded once more as operands of the
    matrix products, each on its own part of the output: at most sqrt(3) * 1.7e-3 = 2.9e-3.
  * float32 states of bfloat16 streams: 1e-5, as float32 (the products of bfloat16 inputs are
    exact and their decays are carried in more than 16 bits).
Every element is held to 40 times that of the larger of its magnitude and the result's root
mean square.
"""
import torch

REL = {torch.float32: 1e-5, torch.bfloat16: 4e-3}


def attention(q, k, v, log_decay, scale, initial_state=None, lengths=None):
    """(out (B, L, H, V), last_state (B, H, K, V)) in float64."""
    H, L = log_decay.numel(), q.shape[1]
    q, k, v = (x.double().repeat_interleave(H // x.shape[2], dim=2).transpose(1, 2) for x in (q, k, v))
    g = log_decay.double()[:, None, None]
    t = torch.arange(L, device=q.device, dtype=torch.float64)
    n = torch.full((q.shape[0],), L, device=q.device, dtype=torch.int64) if lengths is None else lengths.clamp(0, L)
    live = (t[None] < n[:, None])[:, None, :, None]
    q, k, v = (torch.where(live, x, 0.0) for x in (q, k, v))

    def power(dist):                      # exp(g * dist), 1 at a distance of zero, 0 below it
        d = dist.clamp(min=0)
        return torch.where(dist < 0, 0.0, torch.where(d == 0, 1.0, torch.exp(g * d.clamp(min=1))))

    out = ((q @ k.transpose(-1, -2)) * power(t[:, None] - t[None, :])[None]) @ v
    ends = torch.stack([power((n_b - 1 - t)[None, :])[:, 0] for n_b in n])            # (B, H, L)
    last = (k * ends[..., None]).transpose(-1, -2) @ v
    if initial_state is not None:
        s0 = initial_state.double()
        out = out + power(t[None, :] + 1).transpose(-1, -2)[None] * (q @ s0)
        last = last + torch.stack([power(n_b.double().reshape(1, 1))[:, 0] for n_b in n])[..., None] * s0
    out = torch.where(live, out * scale, 0.0)
    return out.transpose(1, 2), last


def check(got, want, name, rel=None):
    rel = REL[got.dtype] if rel is None else rel
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)} vs {tuple(want.shape)}"
    got, want = got.detach().double(), want.detach().double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    norm = want.norm()
    err = (got - want).norm()
    assert err <= rel * norm + 1e-30, f"{name}: relative error {float(err / norm):.3g} above {rel:.3g}"
    rms = norm / max(1, want.numel()) ** 0.5
    worst = ((got - want).abs() / want.abs().clamp(min=float(rms) + 1e-30)).max() if want.numel() else 0.0
    assert worst <= 40 * rel, f"{name}: an element is {float(worst):.3g} off"


def inputs(B, L, H, K, V, dtype, dev, seed=0, heads=(None, None, None), decay=None):
    """Column blocks of one projection, and decays from fast to slow."""
    g = torch.Generator(device=dev).manual_seed(seed)
    G, J, M = (H if n is None else n for n in heads)
    qkv = torch.randn(B, L, G * K + J * K + M * V, generator=g, device=dev).to(dtype)
    q, k, v = qkv.split([G * K, J * K, M * V], dim=-1)
    if decay is None:
        decay = -torch.exp2(-8.0 * torch.arange(1, H + 1, device=dev, dtype=torch.float32) / H)
    return q.unflatten(-1, (G, K)), k.unflatten(-1, (J, K)), v.unflatten(-1, (M, V)), decay, g
