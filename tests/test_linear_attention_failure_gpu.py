"""Failure detection of the tensor-core linear attention without a GPU fault: every wait is bounded
(0.1 to 4 s); the first that runs out sets the device error word and ends the others of its CTA, so
that the kernel returns and the context stays usable.  The SSM_TEST_WITHHOLD_TMA hook makes the first
wait run out: no load is issued, so none is in flight when the CTAs leave."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [2, 170])       # a CTA per row; rows shared between CTAs
def test_wait_that_runs_out(cuda, monkeypatch, heads):
    from ssm_mamba_b200 import linear_attention_fn
    from ssm_mamba_b200._ext import _C
    g = torch.Generator(device=cuda).manual_seed(heads)
    q, k, v = torch.randn(3, 1, 300, heads, 64, generator=g, device=cuda).bfloat16()
    decay = torch.full((heads,), -0.1, device=cuda)
    want = linear_attention_fn(q, k, v, decay)
    assert _C.check_device_error() == 0
    monkeypatch.setenv("SSM_TEST_WITHHOLD_TMA", "1")
    linear_attention_fn(q, k, v, decay)
    assert _C.check_device_error() == 1            # a wait ran out; read and cleared
    assert _C.check_device_error() == 0
    monkeypatch.delenv("SSM_TEST_WITHHOLD_TMA")
    assert torch.equal(linear_attention_fn(q, k, v, decay), want)
    assert _C.check_device_error() == 0
