"""A decode step refuses a state whose elements share memory: several CTAs would read, change and write
the same place at once."""
import ctypes

import pytest

from linear_attention_ref import check
from ssm_mamba_b200 import capi


@pytest.mark.parametrize("strides", [(0, 128, 8), (512, 0, 8), (512, 128, 0), (0, 0, 0), (511, 128, 8), (512, 127, 8),
                                     (512, 128, 7), (8, 16, 32), (128, -128, 8)])
def test_refused(strides):
    """(batch, heads, dk) strides of a (3, 4, 16, 8) state; refused on the host, before anything is launched."""
    a = capi.LinearAttnUpdateArgs()
    a.batch, a.heads, a.dk, a.dv, a.q_heads, a.k_heads, a.v_heads = 3, 4, 16, 8, 4, 4, 4
    a.q = a.k = a.v = a.log_decay = a.state = a.out = 16
    a.state_batch_stride, a.state_head_stride, a.state_k_stride = strides
    assert capi.lib().ssm_linear_attn_update(ctypes.byref(a), None) == capi.SSM_ERR_INVALID
    assert b"share memory" in capi.lib().ssm_last_error()


@pytest.mark.gpu
def test_views(cuda):
    import torch
    from ssm_mamba_b200 import linear_attention_update
    gen = torch.Generator(device=cuda).manual_seed(2)
    q, k = (torch.randn(3, 4, 16, generator=gen, device=cuda) for _ in range(2))
    v, g = torch.randn(3, 4, 8, generator=gen, device=cuda), torch.tensor([-0.1, -0.2, -0.3, 0.0], device=cuda)
    one = torch.randn(1, 4, 16, 8, generator=gen, device=cuda)
    for bad in (one.expand(3, 4, 16, 8), one[:, :1].expand(3, 4, 16, 8), one[:, :, :1].expand(1, 4, 16, 8).expand(3, -1, -1, -1),
                torch.zeros(3 * 512, device=cuda).as_strided((3, 4, 16, 8), (512, 128, 4, 1))):
        with pytest.raises(RuntimeError, match="share memory"):
            linear_attention_update(bad, q, k, v, g)
    start = one.expand(3, 4, 16, 8).contiguous()
    want = start.clone()
    out = linear_attention_update(want, q, k, v, g)
    room = torch.zeros(16, 6, 7, 20, device=cuda)
    for state in (start.transpose(0, 1).contiguous().transpose(0, 1),                      # head-major
                  start.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3),              # dk-major
                  room[:, ::2, 1:5, 3:11].permute(1, 2, 0, 3)):                            # a part of a larger cache
        state.copy_(start)
        # the order of the output's sums goes by the width of the accesses, that of the state's elements does not
        check(linear_attention_update(state, q, k, v, g), out.double(), "out")
        assert torch.equal(state, want)
    # dimensions of one element may have any stride
    s1 = start[:1].as_strided((1, 4, 16, 8), (0, 128, 8, 1))
    linear_attention_update(s1, q[:1], k[:1], v[:1], g)
    assert torch.equal(s1, want[:1])
