"""The backward of layer norm leaves one partial row of dweight and dbias per CTA, and runs no CTA without a
row: what it writes of the workspace goes by the rows that a CTA takes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


# bfloat16 vectors of up to 768 and every row of up to 512: four rows to a CTA, else one
@pytest.mark.parametrize("dtype,dim,offset,per_cta", [
    (torch.bfloat16, 640, 0, 4), (torch.bfloat16, 768, 0, 4), (torch.bfloat16, 640, 1, 1), (torch.bfloat16, 776, 0, 1),
    (torch.bfloat16, 512, 0, 4), (torch.float32, 512, 0, 4), (torch.float32, 640, 0, 1)])
@pytest.mark.parametrize("rows", [1, 3, 4, 37])
def test_partial_rows(cuda, dtype, dim, offset, per_cta, rows):
    from ssm_mamba_b200 import capi
    gen = torch.Generator(device=cuda).manual_seed(dim + rows)
    room = torch.randn(2, rows, dim + 8, generator=gen, device=cuda).to(dtype)
    x, dy = room[0, :, offset:offset + dim], room[1, :, offset:offset + dim]
    w = torch.randn(dim, generator=gen, device=cuda)
    mean = x.float().mean(1)
    rstd = torch.rsqrt(x.float().var(1, unbiased=False) + 1e-5)
    dx = torch.empty(rows, dim, device=cuda, dtype=dtype)
    dw, db = torch.empty(dim, device=cuda), torch.empty(dim, device=cuda)
    args = capi.fill_layer_norm(x, 1e-5, w, mean=mean, rstd=rstd, dy=dy, dx=dx, dweight=dw, dbias=db)
    ws = torch.full((64, 2, dim), math.nan, device=cuda)
    capi.call_layer_norm_bwd(args, workspace=ws.view(torch.uint8).view(-1))
    ctas = -(-rows // per_cta)
    assert torch.isfinite(ws[:ctas]).all() and torch.isnan(ws[ctas:]).all()
    h = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    for got, want in ((dw, (dy.double() * h).sum(0)), (db, dy.double().sum(0))):
        assert (got.double() - want).norm() <= 2e-6 * want.norm()
