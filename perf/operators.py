"""Measured cases of the linear-attention and layer-norm operators.

Each case is one call pattern of a hybrid Mamba / linear-attention stack:
  prefill   linear_attention_fn over whole prompts, no gradient, with the state that decoding
            continues from
  train     linear_attention_fn and its backward
  step      linear_attention_update, one token per sequence, the state updated in place
  norm      layer_norm_fn without a gradient
  normgrad  layer_norm_fn and its backward, weight and bias included
`own` selects this repository's kernels; otherwise the same results come from elementary torch
operations in float32.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def _attn(name, op, dtype, batch, seqlen, heads, dk, dv, q_heads=0, kv_heads=0, init=False, ragged=False):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "seqlen": seqlen, "heads": heads,
            "q_heads": q_heads or heads, "kv_heads": kv_heads or heads, "dk": dk, "dv": dv,
            "init": init, "ragged": ragged}


def _norm(name, op, dtype, rows, dim):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "dim": dim}


def listed():
    return [
        # a short prompt in float32, as a unit test or a small model runs it: latency
        _attn("prefill_short_fp32", "prefill", "fp32", 2, 256, 4, 16, 16),
        # prompts of the 2.8B-width benchmark (4 x 2048 tokens, 5120 channels as 40 heads of 128)
        _attn("prefill_prompts", "prefill", "bf16", 4, 2048, 40, 128, 128),
        # one very long sequence (131072 tokens, 5120 channels): batch 1, few rows to fill the GPU with
        _attn("prefill_long", "prefill", "bf16", 1, 131072, 40, 128, 128),
        # a served batch of prompts of different lengths, keys and values shared by groups of
        # query heads, continued from an earlier state
        _attn("prefill_ragged_shared", "prefill", "bf16", 7, 1531, 24, 64, 64, 24, 8, True, True),
        # training step of the 130M-width layer (8 x 2048 tokens, 1536 channels as 12 heads of 128)
        _attn("train_layer", "train", "bf16", 8, 2048, 12, 128, 128),
        # the same width in float32, 24 heads of 64
        _attn("train_fp32", "train", "fp32", 2, 1024, 24, 64, 64),
        # training on padded sequences, one query/key head per two value heads, odd sizes,
        # truncated back-propagation through time (a gradient into the initial state)
        _attn("train_ragged_odd", "train", "bf16", 3, 1000, 10, 80, 96, 5, 5, True, True),
        # one sequence decoding: latency
        _attn("step_single", "step", "bf16", 1, 1, 12, 64, 64),
        # the decode batch of the benchmark (64 sequences, 5120 channels as 40 heads of 128)
        _attn("step_batch", "step", "bf16", 64, 1, 40, 128, 128),
        # the norm in front of a decode step (64 rows of the 2.8B model width)
        _norm("norm_decode", "norm", "bf16", 64, 2560),
        # the norm of a training step (8 x 2048 tokens of the 130M model width)
        _norm("normgrad_layer", "normgrad", "bf16", 16384, 768),
        # a long batch in float32 with a width that is no multiple of a vector
        _norm("normgrad_odd_fp32", "normgrad", "fp32", 32768, 2565),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "train", "train", "step", "norm", "normgrad"])
    dtype = "bf16" if rng.random() < 0.7 else "fp32"
    if op in ("norm", "normgrad"):
        dim = _log_int(rng, 33, 8192)
        if rng.random() < 0.6:
            dim = max(80, dim // 80 * 80)
        rows = _log_int(rng, 1, max(1, min(131072, (1 << 28) // dim)))
        return {"op": op, "dtype": dtype, "rows": rows, "dim": dim}
    dims = [16, 32, 64, 64, 80, 96, 128, 128, 37, 100]
    dk, dv = rng.choice(dims), rng.choice(dims)
    group = rng.choice([1, 1, 1, 2, 4])
    heads = group * _log_int(rng, 1, 64 // group)
    q_heads, kv_heads = heads, heads
    if group > 1 and rng.random() < 0.5:
        kv_heads = heads // group
    elif group > 1:
        q_heads = kv_heads = heads // group
    if op == "step":
        batch, seqlen = _log_int(rng, 1, 128), 1
        batch = min(batch, max(1, (1 << 26) // (heads * dk * dv)))
    else:
        most = (1 << 27) // (heads * max(dk, dv)) // (4 if op == "train" else 1)
        seqlen = _log_int(rng, 1, min(65536, most))
        batch = _log_int(rng, 1, max(1, min(32, most // seqlen)))
    return {"op": op, "dtype": dtype, "batch": batch, "seqlen": seqlen, "heads": heads, "q_heads": q_heads,
            "kv_heads": kv_heads, "dk": dk, "dv": dv, "init": rng.random() < 0.5,
            "ragged": op != "step" and batch > 1 and rng.random() < 0.5}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _inputs(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] in ("norm", "normgrad"):
        rows, dim = case["rows"], case["dim"]
        # a residual stream: rows of different scale, a few channels with an offset
        x = (rn(rows, dim) * (1.0 + rn(rows, 1).abs()) + 0.5 * rn(1, dim)).to(dt)
        s = {"x": x, "weight": 1.0 + 0.1 * rn(dim), "bias": 0.1 * rn(dim), "eps": 1e-5}
        if case["op"] == "normgrad":
            s["dy"] = rn(rows, dim).to(dt)
            for n in ("x", "weight", "bias"):
                s[n].requires_grad_()
        return s
    B, L, H, G, J, K, V = (case[n] for n in ("batch", "seqlen", "heads", "q_heads", "kv_heads", "dk", "dv"))
    v_heads = H if G < H else J      # q and k shared by groups of value heads, or k and v by groups of query heads
    # q, k and v are column blocks of one projection's output
    qkv = rn(B, L, G * K + J * K + v_heads * V).to(dt)
    q, k, v = qkv.split([G * K, J * K, v_heads * V], dim=-1)
    s = {"q": q.unflatten(-1, (G, K)), "k": k.unflatten(-1, (J, K)), "v": v.unflatten(-1, (v_heads, V)),
         # fixed geometric decay rates, the slowest over some 250 tokens
         "log_decay": -torch.exp2(-8.0 * torch.arange(1, H + 1, device=dev, dtype=torch.float32) / H),
         "scale": K ** -0.5, "initial_state": None, "lengths": None}
    if case["init"]:
        s["initial_state"] = rn(B, H, K, V)
    if case["ragged"]:
        lengths = torch.randint((L + 1) // 2, L + 1, (B,), generator=gen, device=dev)
        lengths[0] = L
        s["lengths"] = lengths
    if case["op"] == "step":
        s["state"] = 3.0 * rn(B, H, K, V)
        for n in ("q", "k", "v"):
            s[n] = s[n][:, 0]
    if case["op"] == "train":
        s["dout"] = rn(B, L, H, V).to(dt)
        for n in ("q", "k", "v"):
            s[n] = s[n].detach().requires_grad_()
        if case["init"]:
            s["initial_state"].requires_grad_()
    return s


def prepare(case, seed):
    return {"op": case["op"], **_inputs(case, seed)}


# ---------------------------------------------------------------------------------------
# plain forms: float32, elementary operations
# ---------------------------------------------------------------------------------------
def _heads(x, H):
    """(B, L, h, D) -> (B, H, L, D) float32, each head repeated for its group."""
    return x.detach().float().repeat_interleave(H // x.shape[2], dim=2).transpose(1, 2)


def _chunked(q, k, v, g, state):
    """sum_{s <= t} exp(g (t - s)) (q_t . k_s) v_s + exp(g (t + 1)) q_t state, and the state after the
    last token; q, k (B, H, L, K), v (B, H, L, V), g (H,), state (B, H, K, V)."""
    B, H, L, K = q.shape
    V = v.shape[-1]
    C = min(L, 128 if L <= 16384 else 256)
    N = -(-L // C)
    pad = (0, 0, N * C - L, 0)            # zeros in front: they leave the state as it is ...
    q, k, v = (torch.nn.functional.pad(x, pad).reshape(B, H, N, C, -1) for x in (q, k, v))
    i = torch.arange(C, device=q.device, dtype=torch.float32)
    dist = i[:, None] - i[None, :]
    near = torch.where(dist >= 0, torch.exp(g[:, None, None] * dist.clamp(min=0)), 0.0)
    out = ((q @ k.transpose(-1, -2)) * near[None, :, None]) @ v
    added = (k * torch.exp(g[:, None] * (C - 1 - i))[None, :, None, :, None]).transpose(-1, -2) @ v
    n = torch.arange(N + 1, device=q.device, dtype=torch.float32)
    far = n[:, None] - 1 - n[None, :N]    # chunks between the end of chunk j and the start of chunk i
    carry = torch.where(far >= 0, torch.exp(g[:, None, None] * C * far.clamp(min=0)), 0.0)
    starts = (carry[None] @ added.reshape(B, H, N, K * V)).reshape(B, H, N + 1, K, V)
    # ... but not an initial state, so its decay starts at the first real token
    first = N * C - L
    age = (n * C - first).clamp(min=0)
    starts = starts + torch.exp(g[:, None] * age)[None, :, :, None, None] * state[:, :, None]
    row = torch.where(n[:N, None] * C >= first, i[None] + 1, i[None] + 1 - first)
    out = out + (q * torch.exp(g[:, None, None] * row.clamp(min=0))[None, ..., None]) @ starts[:, :, :N]
    return out.reshape(B, H, N * C, V)[:, :, N * C - L:], starts[:, :, N]


def _masked(x, lengths):
    if lengths is None:
        return x
    at = torch.arange(x.shape[2], device=x.device)
    return torch.where((at[None] < lengths[:, None])[:, None, :, None], x, 0.0)


def _to_right(x, lengths):
    """Every row's tokens moved to the end, zeros in front."""
    if lengths is None:
        return x
    L = x.shape[2]
    at = torch.arange(L, device=x.device)[None] - (L - lengths[:, None])
    got = torch.gather(x, 2, at.clamp(min=0)[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3]))
    return torch.where((at >= 0)[:, None, :, None], got, 0.0)


def _plain_attention(s):
    H = s["log_decay"].numel()
    g, lengths = s["log_decay"], s["lengths"]
    q, k, v = (_masked(_heads(s[n], H), lengths) for n in ("q", "k", "v"))
    B, _, L, K = q.shape
    V = v.shape[-1]
    zero = torch.zeros(B, H, K, V, device=q.device)
    init = zero if s["initial_state"] is None else s["initial_state"].detach()
    out, last = _chunked(q, k, v, g, init)
    out = _masked(out * s["scale"], lengths).transpose(1, 2).to(s["q"].dtype)
    if s["op"] == "prefill":
        if lengths is not None:           # the state after each row's own last token
            left = (L - lengths).float()
            _, last = _chunked(*(_to_right(x, lengths) for x in (q, k, v)), g, zero)
            last = last + torch.exp(g[None] * (L - left)[:, None])[..., None, None] * init
        return {"out": out, "last_state": last}
    do = _masked(s["dout"].float().transpose(1, 2), lengths)
    dq, _ = _chunked(do, v, k, g, init.transpose(-1, -2))
    flip = (x.flip(2) for x in (q, k, v, do))
    q, k, v, do = flip
    dv, _ = _chunked(k, q, do, g, zero)
    dk, first = _chunked(v, do, q, g, zero.transpose(-1, -2))
    dk, dv = dk.flip(2), dv.flip(2)
    got = {"out": out}
    for n, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        x = _masked(x * s["scale"], lengths).transpose(1, 2)
        h = s[n[1]].shape[2]
        got[n] = x.unflatten(2, (h, H // h)).sum(3).to(s["q"].dtype)
    if s["initial_state"] is not None:
        got["dinit"] = s["scale"] * torch.exp(g)[None, :, None, None] * first.transpose(-1, -2)
    return got


def _plain_step(s):
    H = s["log_decay"].numel()
    q, k, v = (s[n].float().repeat_interleave(H // s[n].shape[1], dim=1) for n in ("q", "k", "v"))
    s["state"].mul_(torch.exp(s["log_decay"])[None, :, None, None]).add_(k[..., None] * v[..., None, :])
    out = s["scale"] * (q[..., None, :] @ s["state"])[..., 0, :]
    return {"out": out.to(s["q"].dtype), "state": s["state"]}


def _plain_norm(s):
    x, w, b = s["x"].detach().float(), s["weight"].detach(), s["bias"].detach()
    c = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(c.square().mean(-1, keepdim=True) + s["eps"])
    h = c * r
    y = (h * w + b).to(s["x"].dtype)
    if s["op"] == "norm":
        return y
    dy = s["dy"].float()
    e = dy * w
    dx = r * (e - e.mean(-1, keepdim=True) - h * (e * h).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dy * h).sum(0), "dbias": dy.sum(0)}


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    s = state
    if not own:
        return {"prefill": _plain_attention, "train": _plain_attention, "step": _plain_step,
                "norm": _plain_norm, "normgrad": _plain_norm}[s["op"]](s)
    from ssm_mamba_b200 import layer_norm_fn, linear_attention_fn, linear_attention_update
    if s["op"] == "prefill":
        out, last = linear_attention_fn(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"],
                                        initial_state=s["initial_state"], lengths=s["lengths"],
                                        return_last_state=True)
        return {"out": out, "last_state": last}
    if s["op"] == "train":
        out = linear_attention_fn(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"],
                                  initial_state=s["initial_state"], lengths=s["lengths"])
        leaves = [s["q"], s["k"], s["v"]] + ([s["initial_state"]] if s["initial_state"] is not None else [])
        got = torch.autograd.grad(out, leaves, s["dout"])
        return {"out": out.detach(), **dict(zip(("dq", "dk", "dv", "dinit"), got))}
    if s["op"] == "step":
        out = linear_attention_update(s["state"], s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"])
        return {"out": out, "state": s["state"]}
    if s["op"] == "norm":
        return layer_norm_fn(s["x"], s["weight"], s["bias"], eps=s["eps"])
    y = layer_norm_fn(s["x"], s["weight"], s["bias"], eps=s["eps"])
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("norm", "normgrad"):
        rows, dim = case["rows"], case["dim"]
        grad = case["op"] == "normgrad"      # x, y; then x, dy, dx again
        return {"bytes": rows * dim * e * (4 if grad else 2) + dim * 4 * (4 if grad else 2),
                "flops": rows * dim * (20 if grad else 7)}
    B, L, H, G, J, K, V = (case[n] for n in ("batch", "seqlen", "heads", "q_heads", "kv_heads", "dk", "dv"))
    v_heads = H if G < H else J
    tokens = B * L
    qkv, out, state = tokens * (G * K + J * K + v_heads * V) * e, tokens * H * V * e, B * H * K * V * 4
    if case["op"] == "step":
        return {"bytes": qkv + out + 2 * state, "flops": 5 * B * H * K * V}
    # the recurrence: a product and a sum for each state element when it is written and when it is read
    flops = 4 * tokens * H * K * V
    if case["op"] == "prefill":
        return {"bytes": qkv + out + state * (2 if case["init"] else 1), "flops": flops}
    return {"bytes": 2 * qkv + 2 * out + state * (2 if case["init"] else 0), "flops": 3.5 * flops}


# ---------------------------------------------------------------------------------------
# the definition, in 64 bits, token by token
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("norm", "normgrad"):
        s = _inputs(case, seed)
        x, w, b = (s[n].detach().double() for n in ("x", "weight", "bias"))
        var, mean = torch.var_mean(x, dim=-1, keepdim=True, unbiased=False)
        h = (x - mean) / torch.sqrt(var + s["eps"])
        if case["op"] == "norm":
            return h * w + b
        dy = s["dy"].double()
        dh = dy * w
        D = x.shape[-1]
        dx = (D * dh - dh.sum(-1, keepdim=True) - h * (dh * h).sum(-1, keepdim=True)) / (D * torch.sqrt(var + s["eps"]))
        return {"y": h * w + b, "dx": dx, "dweight": (dy * h).sum(0), "dbias": dy.sum(0)}
    B, L, H, K, V = (case[n] for n in ("batch", "seqlen", "heads", "dk", "dv"))
    passes = 3 if case["op"] == "train" else 1
    if L * passes * max(60e-6, B * H * K * V * 8 * 8 / 4e12) > 18:
        return None
    s = _inputs(case, seed)
    decay = torch.exp(s["log_decay"].double())[:, None, None]

    def head(x, t):
        x = x.detach()[:, t] if case["op"] != "step" else x
        return x.double().repeat_interleave(H // x.shape[1], dim=1)

    if case["op"] == "step":
        q, k, v = (head(s[n], 0) for n in ("q", "k", "v"))
        new = decay * s["state"].double() + k[..., :, None] * v[..., None, :]
        return {"out": s["scale"] * torch.einsum("bhk,bhkv->bhv", q, new), "state": new}
    lengths = s["lengths"]
    init = s["initial_state"]
    S = torch.zeros(B, H, K, V, dtype=torch.float64, device="cuda") if init is None else init.detach().double().clone()
    live = None if lengths is None else (torch.arange(L, device="cuda")[:, None] < lengths[None]).double()[..., None, None]
    train = case["op"] == "train"
    out = torch.zeros(B, L, H, V, dtype=torch.float64, device="cuda")
    dq, dk = (torch.zeros(B, L, H, K, dtype=torch.float64, device="cuda") for _ in range(2)) if train else (None, None)
    dv = torch.zeros_like(out) if train else None
    for t in range(L):
        k, v = head(s["k"], t), head(s["v"], t)
        new = decay * S + k[..., :, None] * v[..., None, :]
        S = new if live is None else torch.where(live[t][..., None] > 0, new, S)
        out[:, t] = (head(s["q"], t)[..., None, :] @ S)[..., 0, :]
        if train:
            dq[:, t] = (S @ s["dout"][:, t].double()[..., :, None])[..., 0]
    live = 1.0 if live is None else live.transpose(0, 1)
    out = out * (s["scale"] * live)
    if not train:
        return {"out": out, "last_state": S}
    R = torch.zeros_like(S)
    for t in range(L - 1, -1, -1):
        do = s["dout"][:, t].double() if lengths is None else s["dout"][:, t].double() * live[:, t]
        R = decay * R + head(s["q"], t)[..., :, None] * do[..., None, :]
        dv[:, t] = (head(s["k"], t)[..., None, :] @ R)[..., 0, :]
        dk[:, t] = (R @ head(s["v"], t)[..., :, None])[..., 0]
    got = {"out": out}
    for n, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        h = s[n[1]].shape[2]
        got[n] = (x * (s["scale"] * live)).unflatten(2, (h, H // h)).sum(3)
    if init is not None:
        got["dinit"] = s["scale"] * decay * R
    return got
