"""Every tensor of a call is on one device (two GPUs needed)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_state_on_another_device_is_refused(cuda):
    from ssm_mamba_b200 import linear_attention_fn
    q, k, v = (torch.zeros(1, 8, 2, 16, device=cuda) for _ in range(3))
    g = torch.zeros(2, device=cuda)
    state = torch.zeros(1, 2, 16, 16, device="cuda:1")
    with pytest.raises(RuntimeError, match="device"):
        linear_attention_fn(q, k, v, g, initial_state=state)
    _, last = linear_attention_fn(q, k, v, g, initial_state=state.to(cuda), return_last_state=True)
    assert last.device == q.device
