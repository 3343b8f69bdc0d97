"""Layer norm forward and backward (csrc/layer_norm.cu) against the formula in float64.
Relative 2-norm tolerances: float32 results 2e-6 (sums of up to 2^15 terms in float32, rsqrt
2^-22), bfloat16 results 2.5e-3 (one rounding: 1.7e-3); every element to 40 times that of the
larger of its magnitude and the result's root mean square."""
import math

import pytest
import torch

from linear_attention_ref import check

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
REL = {F32: 2e-6, BF16: 2.5e-3}


def _norm(x, w, b, eps):
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    y = (x - mean) / torch.sqrt(var + eps)
    y = y if w is None else y * w
    return y if b is None else y + b


def _both(x, w, b, eps, dy, rel=None):
    from ssm_mamba_b200 import layer_norm_fn
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    y = layer_norm_fn(*(next(it) if t is not None else None for t in (x, w, b)), eps=eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    got = torch.autograd.grad(y, leaves, dy)
    ref = [t.detach().double().requires_grad_() for t in leaves]
    it = iter(ref)
    ry = _norm(*(next(it) if t is not None else None for t in (x, w, b)), eps)
    want = torch.autograd.grad(ry, ref, dy.double())
    check(y, ry, "y", rel=rel or REL[x.dtype])
    for n, a, r, t in zip(("dx", "d1", "d2"), got, want, leaves):
        assert a.dtype == t.dtype and a.shape == t.shape
        check(a, r, n, rel=rel or REL[a.dtype])
    return y, got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 8), (3, 7), (5, 256), (7, 257), (600, 512), (33, 520), (2000, 768),
                                      (9, 769), (64, 1024), (5, 1025), (3, 2048), (700, 2049), (31, 2560), (17, 2565),
                                      (9, 4096), (5, 4097), (1300, 5120), (3, 8192), (3, 8193), (130, 16384), (2, 20001)])
def test_forward_backward(cuda, rows, dim, dtype):
    gen = torch.Generator(device=cuda).manual_seed(rows * 7 + dim)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    x = (rn(rows, dim) * (1 + rn(rows, 1).abs()) + rn(1, dim)).to(dtype)
    # gradients through a division by the spread: rows of one element have none (dx = 0)
    _both(x, 1 + 0.1 * rn(dim), rn(dim), 1e-5, rn(rows, dim).to(dtype)) if dim > 1 else _one(x, rn(1), rn(1))


def _one(x, w, b):
    from ssm_mamba_b200 import layer_norm_fn
    x = x.detach().requires_grad_()
    y = layer_norm_fn(x, w, b)
    assert torch.equal(y, b.to(x.dtype).expand_as(y))
    y.sum().backward()
    assert not x.grad.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [640, 333, 9000])
@pytest.mark.parametrize("affine", ["none", "weight", "bias"])
def test_without_weight_or_bias(cuda, dim, affine, dtype):
    gen = torch.Generator(device=cuda).manual_seed(dim)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    _both(rn(40, dim).to(dtype), rn(dim) if affine == "weight" else None, rn(dim) if affine == "bias" else None,
          1e-3, rn(40, dim).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_shapes(cuda, dtype):
    gen = torch.Generator(device=cuda).manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda).to(dtype)  # noqa: E731
    w, b = rn(96).float(), rn(97).float()[1:]                        # an unaligned bias
    _both(rn(2, 5, 3, 96), w, b, 1e-5, rn(2, 5, 3, 96))
    _both(rn(4, 6, 200)[..., 8:104], w, b, 1e-5, rn(4, 6, 96))       # a column block
    _both(rn(4, 6, 200)[..., 7:103], w, b, 1e-5, rn(4, 6, 96))       # an unaligned one
    _both(rn(6, 4, 96).transpose(0, 1), w, b, 1e-5, rn(4, 6, 96))    # rows in another order
    _both(rn(4, 96, 6).transpose(1, 2), w, b, 1e-5, rn(4, 96, 6).transpose(1, 2))
    _both(rn(96), w, b, 1e-5, rn(96))                                # one row
    _both(rn(4, 6, 96), w, b, 1e-5, rn(1, 1, 96).expand(4, 6, 96))   # a broadcast gradient


def test_bf16_parameters(cuda):
    """Parameters of the stream type get gradients of their type."""
    from ssm_mamba_b200 import layer_norm_fn
    x = torch.randn(50, 128, device=cuda).to(BF16)
    w, b = (torch.randn(128, device=cuda).to(BF16).requires_grad_() for _ in range(2))
    dy = torch.randn(50, 128, device=cuda).to(BF16)
    got = torch.autograd.grad(layer_norm_fn(x, w, b), (w, b), dy)
    ref = [t.detach().double().requires_grad_() for t in (w, b)]
    want = torch.autograd.grad(_norm(x.double(), *ref, 1e-5), ref, dy.double())
    for a, r in zip(got, want):
        assert a.dtype == BF16
        check(a, r, "parameter gradient", rel=REL[BF16])


def test_large_offset_and_special_values(cuda):
    """A mean far above the spread (the variance is a second pass, not a difference of
    squares: 1e4 offsets cost 1e4 * 2^-24 of the spread), constant rows, rows with NaN or inf."""
    from ssm_mamba_b200 import layer_norm_fn
    gen = torch.Generator(device=cuda).manual_seed(5)
    for dim in (300, 2000, 9000):
        x = torch.randn(20, dim, generator=gen, device=cuda) + 1e4
        check(layer_norm_fn(x), _norm(x.double(), None, None, 1e-5), "offset", rel=2e-3)
        x = torch.randn(6, dim, generator=gen, device=cuda)
        x[1], x[2, 3], x[4, 5] = 3.0, math.nan, math.inf
        x = x.requires_grad_()
        w = torch.ones(dim, device=cuda, requires_grad=True)
        y = layer_norm_fn(x, w)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        for t in (y, dx):
            assert torch.isnan(t[2]).all() and torch.isnan(t[4]).any() and torch.isfinite(t[[0, 1, 3, 5]]).all()
        assert not y[1].any()


def test_differences(cuda):
    """The gradient against central differences of the float32 forward: step 1e-2 leaves a
    third-order term of about 1e-4 of the derivative and a rounding of 1e-7 / 1e-2 = 1e-5."""
    from ssm_mamba_b200 import layer_norm_fn
    gen = torch.Generator(device=cuda).manual_seed(8)
    rn = lambda *s: torch.randn(*s, generator=gen, device=cuda)  # noqa: E731
    xs, dy, h = [rn(12, 200), rn(200), rn(200)], rn(12, 200), 1e-2
    leaves = [t.clone().requires_grad_() for t in xs]
    grads = torch.autograd.grad(layer_norm_fn(*leaves), leaves, dy)
    for i, grad in enumerate(grads):
        d = rn(*xs[i].shape)
        up, down = (layer_norm_fn(*[t + s * h * d if j == i else t for j, t in enumerate(xs)]) for s in (1, -1))
        want = float(((up.double() - down.double()) * dy.double()).sum()) / (2 * h)
        size = float((grad.double() * d.double()).norm())
        assert abs(float((grad.double() * d.double()).sum()) - want) <= 2e-3 * size, i


def test_empty_deterministic_graph(cuda):
    from ssm_mamba_b200 import layer_norm_fn
    w, b = torch.randn(64, device=cuda, requires_grad=True), torch.randn(64, device=cuda, requires_grad=True)
    x = torch.empty(0, 3, 64, device=cuda, requires_grad=True)
    y = layer_norm_fn(x, w, b)
    assert y.shape == (0, 3, 64)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == x.shape and not dw.any() and not db.any()
    for dim in (768, 3000, 5000, 9000):
        x = torch.randn(3000, dim, device=cuda).to(BF16)
        dy = torch.randn(3000, dim, device=cuda).to(BF16)
        w = torch.randn(dim, device=cuda)

        def step():
            xs = [x.detach().requires_grad_(), w.detach().requires_grad_()]
            y = layer_norm_fn(*xs)
            return (y.detach(), *torch.autograd.grad(y, xs, dy))

        want = step()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            assert all(torch.equal(a, r) for a, r in zip(step(), want))
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, r) for a, r in zip(got, want))


def test_refusals(cuda):
    from ssm_mamba_b200 import layer_norm_fn
    x, w = torch.zeros(4, 8, device=cuda), torch.ones(8, device=cuda)
    for err, call in [(TypeError, lambda: layer_norm_fn(x.half())), (RuntimeError, lambda: layer_norm_fn(x, w[:4])),
                      (RuntimeError, lambda: layer_norm_fn(x, w, w.cpu())), (RuntimeError, lambda: layer_norm_fn(x.cpu())),
                      (RuntimeError, lambda: layer_norm_fn(torch.zeros(4, 0, device=cuda))),
                      (ValueError, lambda: layer_norm_fn(torch.zeros((), device=cuda)))]:
        with pytest.raises(err):
            call()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 131, 776, 1023, 1602, 2565, 3500, 4104, 6143, 8191])
def test_many_rows_between_nans(cuda, dim, dtype):
    """Several rows per CTA, x and its gradient at different offsets from 16 bytes, NaN on either
    side of every row."""
    gen = torch.Generator(device=cuda).manual_seed(dim)

    def among_nans(at):
        t = torch.full((4000, dim + 16), math.nan, device=cuda, dtype=dtype)
        t[:, at:at + dim] = torch.randn(4000, dim, generator=gen, device=cuda)
        return t[:, at:at + dim]

    w, b = (torch.randn(dim, generator=gen, device=cuda) for _ in range(2))
    for at in ((8, 16), (5, 2)):
        _both(among_nans(at[0]), w, b, 1e-5, among_nans(at[1]))
