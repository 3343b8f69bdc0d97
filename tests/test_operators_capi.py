"""The C ABI of linear attention and layer norm: struct layouts against the header and host-side
refusals (no GPU), and on the GPU the entry points through ctypes, workspaces included."""
import ctypes
import os
import subprocess

import pytest

from ssm_mamba_b200 import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_header(tmp_path):
    structs = {"ssm_linear_attn_args": capi.LinearAttnArgs, "ssm_linear_attn_update_args": capi.LinearAttnUpdateArgs,
               "ssm_layer_norm_args": capi.LayerNormArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ssm_b200.h"', "int main(void){"]
    for cs, py in structs.items():
        lines.append(f'printf("{cs} %zu\\n", sizeof({cs}));')
        lines += [f'printf("{cs}.{f} %zu\\n", offsetof({cs}, {f}));' for f, _ in py._fields_]
    (tmp_path / "probe.c").write_text("\n".join(lines + ["return 0;}"]))
    exe = tmp_path / "probe"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "probe.c"), "-o", str(exe)])
    got = dict(line.split() for line in subprocess.check_output([str(exe)], text=True).splitlines())
    for cs, py in structs.items():
        assert int(got[cs]) == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert int(got[f"{cs}.{f}"]) == getattr(py, f).offset, f


def _attn(**kw):
    a = capi.LinearAttnArgs()
    a.batch, a.seqlen, a.heads, a.dk, a.dv, a.q_heads, a.k_heads, a.v_heads = 1, 8, 4, 16, 16, 4, 2, 1
    a.q = a.k = a.v = a.log_decay = a.out = 16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(batch=0), b"positive"), (dict(seqlen=0), b"positive"), (dict(heads=0), b"positive"),
    (dict(dk=129), b"1 to 128"), (dict(dv=0), b"1 to 128"), (dict(k_heads=3), b"divide"), (dict(q_heads=0), b"divide"),
    (dict(dtype=2), b"dtype"), (dict(q=None), b"required"), (dict(log_decay=None), b"required"),
    (dict(out=None), b"out is required"), (dict(batch=1 << 25, heads=4), b"2^24"),
    (dict(seqlen=(1 << 30) + 1), b"2^30")])
def test_attention_refusals(change, word):
    lib = capi.lib()
    assert lib.ssm_linear_attn_fwd(ctypes.byref(_attn(**change)), None, 0, None) == capi.SSM_ERR_INVALID
    assert word in lib.ssm_last_error(), lib.ssm_last_error()


def test_other_refusals():
    lib = capi.lib()
    for f in (lib.ssm_linear_attn_fwd, lib.ssm_linear_attn_bwd):
        assert f(None, None, 0, None) == capi.SSM_ERR_INVALID
    assert lib.ssm_linear_attn_bwd(ctypes.byref(_attn()), None, 0, None) == capi.SSM_ERR_INVALID
    assert b"dout" in lib.ssm_last_error()
    assert lib.ssm_linear_attn_workspace_size(ctypes.byref(_attn(dk=0)), 0) == 0 and lib.ssm_last_error()
    assert lib.ssm_linear_attn_update(None, None) == capi.SSM_ERR_INVALID
    u = capi.LinearAttnUpdateArgs()
    u.batch, u.heads, u.dk, u.dv, u.q_heads, u.k_heads, u.v_heads = 1, 4, 16, 200, 4, 4, 4
    assert lib.ssm_linear_attn_update(ctypes.byref(u), None) == capi.SSM_ERR_INVALID
    assert b"1 to 128" in lib.ssm_last_error()
    u.dv = 16
    assert lib.ssm_linear_attn_update(ctypes.byref(u), None) == capi.SSM_ERR_INVALID
    assert b"required" in lib.ssm_last_error()
    assert lib.ssm_layer_norm_fwd(None, None) == capi.SSM_ERR_INVALID
    n = capi.LayerNormArgs()
    assert lib.ssm_layer_norm_fwd(ctypes.byref(n), None) == capi.SSM_ERR_INVALID
    n.rows, n.dim = 2, 8
    assert lib.ssm_layer_norm_fwd(ctypes.byref(n), None) == capi.SSM_ERR_INVALID
    n.x = n.y = n.mean = 16
    assert lib.ssm_layer_norm_fwd(ctypes.byref(n), None) == capi.SSM_ERR_INVALID
    assert b"together" in lib.ssm_last_error()
    assert lib.ssm_layer_norm_bwd(ctypes.byref(n), None, 0, None) == capi.SSM_ERR_INVALID
    assert b"required" in lib.ssm_last_error()
    n.dtype = 9
    assert lib.ssm_layer_norm_bwd_workspace_size(ctypes.byref(n)) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("L", [200, 3000])
def test_attention_through_ctypes(cuda, L):
    import torch
    from linear_attention_ref import attention, check, inputs
    q, k, v, g, gen = inputs(2, L, 4, 64, 32, torch.bfloat16, cuda, seed=L, heads=(4, 2, 2))
    out = torch.empty(2, L, 4, 32, device=cuda, dtype=torch.bfloat16)
    last = torch.empty(2, 4, 64, 32, device=cuda)
    capi.call_linear_attn(capi.fill_linear_attn(q, k, v, g, 0.5, out=out, last_state=last))
    ref = [x.detach().double().requires_grad_() for x in (q, k, v)]
    ro, rl = attention(*ref, g, 0.5)
    check(out, ro, "out")
    check(last, rl, "last_state")
    dout = torch.randn(out.shape, generator=gen, device=cuda).bfloat16()
    got = [torch.empty(x.shape, device=cuda, dtype=x.dtype) for x in (q, k, v)]
    args = capi.fill_linear_attn(q, k, v, g, 0.5, dout=dout, dq=got[0], dk=got[1], dv=got[2])
    capi.call_linear_attn(args, backward=True)
    for a, b in zip(got, torch.autograd.grad(ro, ref, dout.double())):
        check(a, b, "gradient")
    # a workspace that is too small, or not aligned, is refused before anything is launched
    need = capi.lib().ssm_linear_attn_workspace_size(ctypes.byref(args), 1)
    assert need > 0
    ws = torch.empty(need + 512, dtype=torch.uint8, device=cuda)
    for p, n in ((None, need), (ws.data_ptr(), need - 1), (ws.data_ptr() + 8, need)):
        assert capi.lib().ssm_linear_attn_bwd(ctypes.byref(args), p, n, None) == capi.SSM_ERR_WORKSPACE
    assert capi.check_device_error() == 0


@pytest.mark.gpu
def test_norm_and_step_through_ctypes(cuda):
    import torch
    x, dy = (torch.randn(300, 640, device=cuda) for _ in range(2))
    w, b = torch.randn(640, device=cuda), torch.randn(640, device=cuda)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(300, device=cuda), torch.empty(300, device=cuda)
    dw, db = torch.empty_like(w), torch.empty_like(b)
    capi.call_layer_norm_fwd(capi.fill_layer_norm(x, 1e-5, w, b, y=y, mean=mean, rstd=rstd))
    args = capi.fill_layer_norm(x, 1e-5, w, mean=mean, rstd=rstd, dy=dy, dx=dx, dweight=dw, dbias=db)
    capi.call_layer_norm_bwd(args)
    xs = [t.double().requires_grad_() for t in (x, w, b)]
    ry = torch.nn.functional.layer_norm(xs[0], (640,), xs[1], xs[2])
    for got, want in zip((y, dx, dw, db), (ry, *torch.autograd.grad(ry, xs, dy.double()))):
        assert (got.double() - want).norm() <= 2e-6 * want.norm()
    assert capi.lib().ssm_layer_norm_bwd(ctypes.byref(args), None, 0, None) == capi.SSM_ERR_WORKSPACE
    state = torch.randn(2, 3, 16, 8, device=cuda)
    q, k, v = (torch.randn(2, 3, n, device=cuda) for n in (16, 16, 8))
    g, out = torch.tensor([-0.1, -0.5, 0.0], device=cuda), torch.empty(2, 3, 8, device=cuda)
    new = torch.exp(g.double())[:, None, None] * state.double() + k.double()[..., None] * v.double()[..., None, :]
    capi.call_linear_attn_update(capi.fill_linear_attn_update(state, q, k, v, g, 0.25, out))
    assert (state.double() - new).norm() <= 1e-6 * new.norm()
    want = 0.25 * torch.einsum("bhk,bhkv->bhv", q.double(), new)
    assert (out.double() - want).norm() <= 1e-5 * want.norm()
