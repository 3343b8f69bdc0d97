"""One very long row among short ones, more rows than SMs (bfloat16 streams): the row's CTAs run one after the
other, and the last of them waits seconds for the state of the one before it.  Such a wait is no failure.

Through the C ABI with tensors whose rows overlap, so that 480,000 chunks fit into 1 GB: token t of
batch row b is row t + b of one buffer.  The outputs overlap in the same way and are not looked at."""
import ctypes

import pytest
import torch

from linear_attention_ref import attention, check

pytestmark = pytest.mark.gpu


def test_wait_of_seconds_for_another_ctas_state(cuda):
    from ssm_mamba_b200 import capi
    B, L, D = torch.cuda.get_device_properties(cuda).multi_processor_count + 2, 480_000 * 128, 8
    gen = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(L + B, D, generator=gen, device=cuda, dtype=torch.bfloat16)
    out = torch.empty_like(x)
    decay = torch.tensor([-1.0], device=cuda)
    lengths = torch.arange(B, device=cuda) % 200
    lengths[0] = L
    last = torch.zeros(B, 1, D, D, device=cuda)
    rows = x.as_strided((B, L, 1, D), (D, D, D, 1))
    args = capi.fill_linear_attn(rows, rows, rows, decay, 1.0, length=lengths, last_state=last,
                                 out=out.as_strided((B, L, 1, D), (D, D, D, 1)))
    assert capi.lib().ssm_linear_attn_workspace_size(ctypes.byref(args), 0) > 0      # the states that CTAs hand on
    capi.call_linear_attn(args)
    assert capi.check_device_error() == 0
    for b in (0, 1, 100, 150 % B):
        n = int(lengths[b])
        t = x[b + max(0, n - 150):b + n][None, :, None]         # what came before has decayed to e^-150
        if n == 0:
            assert not last[b].any()
        else:
            check(last[b:b + 1], attention(t, t, t, decay, 1.0)[1], f"row {b}")
