"""Linear attention and layer norm have no forward-mode derivative: a tangent is refused, not dropped,
whichever input carries it and whether or not one requires a gradient."""
import pytest
import torch
from torch.autograd import forward_ad


def _refuses(dev):
    from ssm_mamba_b200 import layer_norm_fn, linear_attention_fn, linear_attention_update
    ones = lambda *s: torch.ones(*s, device=dev)  # noqa: E731
    calls = [
        (linear_attention_fn, [ones(1, 4, 2, 8), ones(1, 4, 2, 8), ones(1, 4, 2, 8), -ones(2), None, ones(1, 2, 8, 8)]),
        (linear_attention_update, [ones(1, 2, 8, 8), ones(1, 2, 8), ones(1, 2, 8), ones(1, 2, 8), -ones(2)]),
        (layer_norm_fn, [ones(3, 8), ones(8), ones(8)]),
    ]
    for fn, args in calls:
        for i, a in enumerate(args):
            if a is None:
                continue
            with forward_ad.dual_level():
                dual = [forward_ad.make_dual(a, torch.ones_like(a)) if j == i else x for j, x in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fn(*dual)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    fn(*dual)


def test_tangents_are_refused():
    _refuses(torch.device("cpu"))            # before the device is looked at


@pytest.mark.gpu
def test_tangents_are_refused_gpu(cuda):
    _refuses(cuda)
