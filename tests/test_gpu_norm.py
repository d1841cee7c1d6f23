"""Layer norm against its definition in 64 bits.

Bounds, with u half a step of x's type and e = 2^-24: the kernel's sums over d take at most
32 additions in a thread and 10 across threads, so with the few operations around them
  y:  u |y| + 64 e (|xh w| + |w| + |b|)   (|w|: the mean's and the base's part of xh)
  dx: u |dx| + 64 e rstd (|a| + mean |a| + |xh| mean |a xh| + mean |a| |xh|), a = dy w
  dw, db: the rows of a block one after another and the blocks in order, (rows + 64) e times
  the sum of magnitudes (|dy| (|xh| + 1) for dw)."""

import math

import pytest
import torch

from param_decomp_amd import _lib as L
from param_decomp_amd import ops
from param_decomp_amd.norms import layer_norm

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E = 2.0**-24


def _inputs(device, shape, dtype, seed=0, offset=0.5, spread=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    d = shape[-1]
    x = (torch.randn(shape, device=device, generator=g) * spread + offset).to(dtype)
    dy = torch.randn(shape, device=device, generator=g).to(dtype)
    return x, dy, 1 + 0.3 * torch.randn(d, device=device, generator=g), 0.2 * torch.randn(d, device=device, generator=g)


def _definition(x, dy, w, b, eps):
    d = x.shape[-1]
    u = torch.finfo(x.dtype).eps / 2
    x, dy = x.double().reshape(-1, d), dy.double().reshape(-1, d)
    W = torch.ones(d, dtype=F64, device=x.device) if w is None else w.double()
    B = torch.zeros(d, dtype=F64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    y = xh * W + B
    a = dy * W
    m = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    dx = rstd * (a - m(a) - xh * m(a * xh))
    rows = x.shape[0]
    val = [y, dx, (dy * xh).sum(0), dy.sum(0)]
    tol = [u * y.abs() + 64 * E * ((xh * W).abs() + W.abs() + B.abs()),
           u * dx.abs() + 64 * E * rstd * (a.abs() + m(a.abs()) + xh.abs() * m((a * xh).abs()) + m(a.abs()) * xh.abs()),
           (rows + 64) * E * (dy.abs() * (xh.abs() + 1)).sum(0), (rows + 64) * E * dy.abs().sum(0)]
    return val, [t + 1e-30 for t in tol]


def _check(got, val, tol, names=("y", "dx", "dweight", "dbias")):
    for x, v, t, name in zip(got, val, tol, names):
        if x is None:
            continue
        off = (x.double().reshape(v.shape) - v).abs()
        assert torch.isfinite(x.float()).all(), name
        assert (off <= t).all(), f"{name}: {(off / t).max().item():.3g} of the bound"


def _run(x, dy, w, b, eps=1e-5):
    leaves = [t if t is None else t.detach().clone().requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, eps=eps)
    grads = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    return (y.detach(), *[None if t is None else next(grads) for t in leaves])


WIDTHS = [1, 2, 7, 8, 64, 100, 257, 504, 512, 520, 768, 1000, 1023, 1024, 1032, 2040, 2048, 2056, 4095, 4096, 4104, 5000,
          8192, 8200, 16384, 16385, 20000]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", WIDTHS)
def test_widths(device, dtype, d):
    for rows in (1, 5, 37):
        x, dy, w, b = _inputs(device, (rows, d), dtype, seed=d + rows)
        _check(_run(x, dy, w, b), *_definition(x, dy, w, b, 1e-5))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows, d", [(2049, 64), (4100, 200), (1300, 768), (3001, 2048), (700, 4096), (531, 8192),
                                     (600, 12000), (40, 17000), (5000, 33)])
def test_many_rows(device, dtype, rows, d):
    x, dy, w, b = _inputs(device, (rows, d), dtype, seed=rows)
    got = _run(x, dy, w, b)
    _check(got, *_definition(x, dy, w, b, 1e-5))
    for p, q in zip(got, _run(x, dy, w, b)):  # the same bits a second time
        assert torch.equal(p, q)
    assert torch.equal(layer_norm(x, w, b), got[0])


@pytest.mark.parametrize("affine", ["weight", "bias", "none"])
def test_affine_parts(device, affine):
    x, dy, w, b = _inputs(device, (70, 384), BF16, seed=1)
    w, b = w if affine == "weight" else None, b if affine == "bias" else None
    _check(_run(x, dy, w, b), *_definition(x, dy, w, b, 1e-5))


def test_leading_axes_strides_and_alignment(device):
    x, dy, w, b = _inputs(device, (3, 5, 8, 96), F32, seed=2)
    got = _run(x, dy, w, b)
    assert got[0].shape == x.shape and got[1].shape == x.shape
    _check(got, *_definition(x, dy, w, b, 1e-5))
    # a transposed view, columns of a wider tensor, a start that is not 16-byte aligned
    flat = torch.cat([x.flatten()[:1], x.flatten()])[1:].view(-1, 96)
    wide = torch.cat([x.reshape(-1, 96), x.reshape(-1, 96)], 1)[:, 96:]
    swapped = x.reshape(-1, 96).t().contiguous().t()
    for t in (flat, wide, swapped):
        same = _run(t, dy.reshape(-1, 96), w, b)
        _check(same, *_definition(t, dy.reshape(-1, 96), w, b, 1e-5))
    xv = flat.detach().requires_grad_()  # the unaligned leaf itself
    y = layer_norm(xv, w, b)
    (dx,) = torch.autograd.grad(y, xv, dy.reshape(-1, 96).t().contiguous().t())
    val, tol = _definition(flat, dy.reshape(-1, 96), w, b, 1e-5)
    _check((y.detach(), dx), val, tol)


@pytest.mark.parametrize("d", [300, 3000, 20000])
def test_offset_far_above_the_spread(device, d):
    """x = 1000 + a spread of 1 (exact multiples of 2^-10): no digits of the spread are lost."""
    x, dy, w, b = _inputs(device, (9, d), F32, seed=3)
    x = (x * 1024).round() / 1024 + 1000
    assert torch.equal(x * 1024, (x * 1024).round())
    _check(_run(x, dy, w, b), *_definition(x, dy, w, b, 1e-5))


def test_constant_rows_and_one_column(device):
    x = torch.full((4, 100), 3.25, device=device)
    _, dy, w, b = _inputs(device, (4, 100), F32, seed=4)
    got = _run(x, dy, w, b)
    assert torch.equal(got[0], b.expand(4, 100))
    _check(got, *_definition(x, dy, w, b, 1e-5))


def test_rows_with_nan_or_infinities_stay_alone(device):
    for d in (200, 3000, 17000):
        x, dy, w, b = _inputs(device, (12, d), F32, seed=5)
        want = _run(x, dy, w, b)
        for bad in (math.nan, math.inf):
            xb = x.clone()
            xb[7, d // 2] = bad
            got = _run(xb, dy, w, b)
            keep = torch.arange(12, device=device) != 7
            assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])
            assert torch.isnan(got[0][7]).any() and torch.isnan(got[1][7]).all()
            assert torch.equal(got[3], want[3])


def test_no_rows(device):
    x, dy, w, b = _inputs(device, (0, 96), BF16)
    y, dx, dw, db = _run(x, dy, w, b)
    assert y.shape == (0, 96) and dx.shape == (0, 96)
    assert (dw == 0).all() and (db == 0).all()


def test_only_some_gradients(device):
    x, dy, w, b = _inputs(device, (50, 640), BF16, seed=6)
    full = _run(x, dy, w, b)
    for i, leaf in enumerate((x, w, b)):
        args = [x, w, b]
        args[i] = leaf.clone().requires_grad_()
        (g,) = torch.autograd.grad(layer_norm(*args), args[i], dy)
        assert torch.equal(g, full[i + 1])
    stats = ops.layer_norm_fwd(x, w, b, want_stats=True)[1]
    assert ops.layer_norm_bwd(x, dy, w, stats, want_dx=False, want_dweight=False, want_dbias=False) == (None, None, None)


def test_gradient_is_the_difference_of_the_definition(device):
    x, dy, w, b = _inputs(device, (20, 130), F32, seed=7)
    got = _run(x, dy, w, b)[1:]
    gen = torch.Generator(device=device).manual_seed(1)
    dirs = [torch.randn(t.shape, dtype=F64, device=device, generator=gen) for t in (x, w, b)]

    def loss(t):
        X, W, B = (v.double() + t * r for v, r in zip((x, w, b), dirs))
        c = X - X.mean(-1, keepdim=True)
        return float(((c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * W + B) * dy.double()).sum())

    want = (loss(1e-5) - loss(-1e-5)) / 2e-5
    have = sum(float((g.double() * r).sum()) for g, r in zip(got, dirs))
    size = sum(float((g.double().abs() * r.abs()).sum()) for g, r in zip(got, dirs))
    assert abs(want - have) <= 1e-5 * size


def test_stream_and_graph(device):
    static = _inputs(device, (333, 768), BF16, seed=0)

    def calls(x, dy, w, b):
        y, stats = ops.layer_norm_fwd(x, w, b, want_stats=True)
        return (y, *ops.layer_norm_bwd(x, dy, w, stats))

    want = calls(*static)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(device=device)
    with torch.cuda.stream(side):
        got = calls(*static)
    side.synchronize()
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls(*static)
    for i in range(3):
        for dst, src in zip(static, _inputs(device, (333, 768), BF16, seed=i + 1)):
            dst.copy_(src)
        for t in got:
            t.fill_(float("nan"))
        graph.replay()
        want = calls(*static)
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert torch.equal(p, q)


def test_mixed_devices_are_refused(device):
    with pytest.raises(L.PDError, match="weight is on cpu"):
        layer_norm(torch.zeros(2, 8, device=device), torch.ones(8))
