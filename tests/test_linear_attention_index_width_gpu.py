"""Rows so long that the elements of their padding pass 2^31, all of which are written as zeros, and heads so
many that the elements of 16 tokens do.

Through the C ABI, with tensors whose tokens share memory so that nothing large is allocated: tokens of the
outputs have a stride of zero (all of them write the same values), those of the inputs one that overlaps."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _run(cuda, dtype, L, batch, K, V, step):
    from ssm_mamba_b200 import capi
    x = torch.ones(L * step + batch * 8 + 128, device=cuda, dtype=dtype)
    q, k, v = (x.as_strided((batch, L, 1, n), (8, step, 8, 1)) for n in (K, K, V))
    room = torch.full((batch, V + 2), math.nan, device=cuda, dtype=dtype)
    out = room[:, 1:-1].as_strided((batch, L, 1, V), (V + 2, 0, V + 2, 1))
    lengths = torch.zeros(batch, device=cuda, dtype=torch.int64)
    last = torch.full((batch, 1, K, V), math.nan, device=cuda)
    capi.call_linear_attn(capi.fill_linear_attn(q, k, v, torch.tensor([-0.1], device=cuda), 1.0, length=lengths, out=out,
                                                last_state=last))
    assert capi.check_device_error() == 0
    assert torch.isnan(room[:, 0]).all() and torch.isnan(room[:, -1]).all()
    assert not room[:, 1:-1].any() and not last.any()


def _sms(cuda):
    return torch.cuda.get_device_properties(cuda).multi_processor_count


def test_float32(cuda):
    _run(cuda, torch.float32, 1 << 26, 2 * _sms(cuda), 1, 1, 0)          # one segment per row, 32 columns of work


def test_bfloat16(cuda):
    _run(cuda, torch.bfloat16, 1 << 24, _sms(cuda) + 1, 8, 128, 8)       # rows shared between CTAs, single elements


def test_gradients_of_many_shared_heads(cuda):
    """With a decay of zero and inputs of one every head's gradient of v is one, and the sum over two of
    them two (17 GB of workspace for the heads' gradients)."""
    from ssm_mamba_b200 import capi
    H, V = 2 * 1_060_000, 127
    one = torch.ones(V, device=cuda)
    q, v, dout = (one.as_strided((1, 16, h, n), (0, 0, 0, 1)) for h, n in ((H, 1), (H // 2, V), (H, V)))
    room = torch.full((V + 2,), math.nan, device=cuda)
    dv = room[1:-1].as_strided((1, 16, H // 2, V), (0, 0, 0, 1))
    dq, dk = (torch.empty(1, 16, H, 1, device=cuda) for _ in range(2))
    decay = torch.full((H,), -math.inf, device=cuda)
    capi.call_linear_attn(capi.fill_linear_attn(q, q, v, decay, 1.0, dout=dout, dq=dq, dk=dk, dv=dv), backward=True)
    assert torch.isnan(room[0]) and torch.isnan(room[-1])
    assert (room[1:-1] == 2).all() and (dq == V).all() and (dk == V).all()
