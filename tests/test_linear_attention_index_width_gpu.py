"""Rows so long that the elements of their padding pass 2^31: all of them are written as zeros.

Through the C ABI, with tensors whose tokens share memory so that nothing large is allocated: tokens of the
output have a stride of zero (all of them write the same zeros), those of the inputs one that overlaps."""
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
