"""Linear attention of bfloat16 streams with more rows than SMs, whose chunks the CTAs share (a row's state
goes from one CTA to the next), and rows cut into segments, at the widths of every kernel: against the
definition in float64 (tests/linear_attention_ref.py, where the tolerances are derived)."""
import pytest
import torch

from linear_attention_ref import attention, check, inputs

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
WIDTHS = [(128, 128), (48, 100), (100, 48), (64, 64)]


def _step(q, k, v, g, s0, lengths, dout, dlast):
    from ssm_mamba_b200 import linear_attention_fn
    xs = [x.detach().requires_grad_() for x in (q, k, v, s0)]
    out, last = linear_attention_fn(*xs[:3], g, initial_state=xs[3], lengths=lengths, return_last_state=True)
    return (out.detach(), last.detach(), *torch.autograd.grad((out, last), xs, (dout, dlast)))


def _reference(q, k, v, g, s0, lengths, dout, dlast):
    """Row by row over its own tokens, so that one long row among short ones stays affordable."""
    B, L, H = dout.shape[:3]
    got = [torch.zeros(t.shape, device=t.device, dtype=torch.float64) for t in (dout, s0, q, k, v, s0)]
    for b in range(B):
        n = L if lengths is None else int(lengths[b].clamp(0, L))
        xs = [x[b:b + 1, :n].detach().double().requires_grad_() for x in (q, k, v)]
        xs.append(s0[b:b + 1].detach().double().requires_grad_())
        if n == 0:
            got[1][b], got[5][b] = s0[b], dlast[b]
            continue
        out, last = attention(*xs[:3], g, q.shape[3] ** -0.5, xs[3])
        grads = torch.autograd.grad((out, last), xs, (dout[b:b + 1, :n].double(), dlast[b:b + 1].double()))
        got[0][b, :n], got[1][b], got[5][b] = out[0].detach(), last[0].detach(), grads[3][0]
        for i in range(3):
            got[2 + i][b, :n] = grads[i][0]
    return got


def _compare(got, want):
    for name, a, b in zip(("out", "last_state", "dq", "dk", "dv", "dinitial_state"), got, want):
        check(a, b, name)


def _case(cuda, B, L, H, K, V, seed, heads=(None, None, None)):
    q, k, v, g, gen = inputs(B, L, H, K, V, BF16, cuda, seed=seed, heads=heads)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    return q, k, v, g, rn(B, H, K, V), rn(B, L, H, V).to(BF16), rn(B, H, K, V)


def _sms(cuda):
    return torch.cuda.get_device_properties(cuda).multi_processor_count


@pytest.mark.parametrize("K,V", WIDTHS)
@pytest.mark.parametrize("ragged", [False, True])
def test_more_rows_than_sms(cuda, K, V, ragged):
    H = _sms(cuda) // 2 + 6
    H += H % 2
    q, k, v, g, s0, dout, dlast = _case(cuda, 2, 600, H, K, V, K + V, heads=(H, H // 2, H))
    lengths = torch.tensor([471, 600], device=cuda) if ragged else None
    _compare(_step(q, k, v, g, s0, lengths, dout, dlast), _reference(q, k, v, g, s0, lengths, dout, dlast))


@pytest.mark.parametrize("K,V", WIDTHS)
def test_one_long_row_among_short_ones(cuda, K, V):
    """The long rows run through a dozen CTAs, each of which waits for the one before; rows without
    tokens stand between the others."""
    B, L, H = _sms(cuda) // 2 + 6, 3000, 2
    q, k, v, g, s0, dout, dlast = _case(cuda, B, L, H, K, V, K * V)
    lengths = torch.arange(B, device=cuda) % 7 * 20
    lengths[B // 3], lengths[B - 1] = L, 1500
    _compare(_step(q, k, v, g, s0, lengths, dout, dlast), _reference(q, k, v, g, s0, lengths, dout, dlast))


@pytest.mark.parametrize("K,V", WIDTHS)
@pytest.mark.parametrize("lengths", [None, [4097, 2051]])
def test_segments(cuda, K, V, lengths):
    q, k, v, g, s0, dout, dlast = _case(cuda, 2, 4097, 2, K, V, K + 2 * V, heads=(2, 1, 2))
    lengths = None if lengths is None else torch.tensor(lengths, device=cuda)
    _compare(_step(q, k, v, g, s0, lengths, dout, dlast), _reference(q, k, v, g, s0, lengths, dout, dlast))


@pytest.mark.parametrize("K,V", WIDTHS)
def test_outputs_that_no_tma_can_store(cuda, K, V):
    """Rows of out and of the gradients that start off 16 bytes, among NaN that stays."""
    from ssm_mamba_b200 import capi
    H = _sms(cuda) + 3
    q, k, v, g, s0, dout, dlast = _case(cuda, 1, 300, H, K, V, 9)
    want = _reference(q, k, v, g, s0, None, dout, dlast)
    room = [torch.full((1, 300, H, n + 3), float("nan"), device=cuda, dtype=BF16) for n in (V, K, K, V)]
    out, dq, dk, dv = (r[..., 1:-2] for r in room)
    last, ds = torch.empty_like(s0), torch.empty_like(s0)
    scale = K ** -0.5
    capi.call_linear_attn(capi.fill_linear_attn(q, k, v, g, scale, initial_state=s0, out=out, last_state=last))
    capi.call_linear_attn(capi.fill_linear_attn(q, k, v, g, scale, initial_state=s0, dout=dout, dlast_state=dlast, dq=dq,
                                                dk=dk, dv=dv, dinitial_state=ds), backward=True)
    assert capi.check_device_error() == 0
    _compare((out, last, dq, dk, dv, ds), want)
    for r in room:
        assert torch.isnan(r[..., 0]).all() and torch.isnan(r[..., -2:]).all()


@pytest.mark.parametrize("K,V", WIDTHS)
def test_graph_and_streams(cuda, K, V):
    """Equal bits from a captured graph, and from two streams that run at once."""
    H = _sms(cuda) + 12
    args = _case(cuda, 1, 700, H, K, V, 4)
    args = (*args[:5], torch.tensor([650], device=cuda), *args[5:])
    want = _step(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([_step(*args) for _ in range(3)])
    torch.cuda.synchronize()
    for a in got[0] + got[1]:
        assert all(torch.equal(x, y) for x, y in zip(a, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(*args)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
