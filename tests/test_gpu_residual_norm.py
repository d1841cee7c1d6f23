"""The norms around a residual branch against the formula in 64 bits.

Tolerances: a mean of d squares is summed in fp32 over chains of at most 64 additions, so 1 / rms is off by at
most 40 2^-24 of itself; with the products behind it a value is off by 64 2^-24 of the magnitudes that are
added, and by half a step of the type it is stored in. y and the gradients are compared for the stream as the
kernel stored it (a neighbouring bf16 is within the stream's own tolerance and changes them by more than their
fp32 roundings). Sums over rows: as many 2^-24 of the sum of magnitudes as there are rows, and 64."""

import pytest
import torch

from param_decomp_amd import _lib as L
from param_decomp_amd import ops
from param_decomp_amd.norms import residual_norm, rms_norm

pytestmark = pytest.mark.gpu

F64, BF16, F32 = torch.float64, torch.bfloat16, torch.float32
U = 2.0**-24
HALF = {BF16: 2.0**-8, F32: U}
EPS = 1e-6
TYPES = [(BF16, BF16), (F32, BF16), (F32, F32)]


def _within(name, a, want, mag, terms=64):
    bound = terms * U * mag + HALF[a.dtype] * (want.abs() + terms * U * mag) + 1e-38
    err = (a.double() - want).abs()
    assert (err <= bound).all(), (name, float((err - bound).max()), float((err / bound).max()))


def _case(device, rows, d, types, gate=None, post=True, seed=0, gate_dtype=F32):
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    c = dict(x=rnd(rows, d).to(types[0]), branch=(rnd(rows, d) * 0.7).to(types[1]), post=1 + 0.2 * rnd(d) if post else None,
             gate=None, pre=1 + 0.2 * rnd(d), gh=rnd(rows, d).to(types[0]), gy=rnd(rows, d).to(types[1]))
    if gate is not None:
        c["gate"] = (0.3 + 0.5 * rnd(*((d,) if gate == 0 else (gate, d)))).to(gate_dtype)
    return c


def _check(c, scale=0.7, zero_centered=False, post_norm=None):
    post_norm = c["post"] is not None if post_norm is None else post_norm
    names = [n for n in ("x", "branch", "post", "gate", "pre") if c[n] is not None]
    leaves = [c[n].detach().clone().requires_grad_() for n in names]
    t = dict(zip(names, leaves))
    h, y = residual_norm(t["x"], t["branch"], post_norm=post_norm, post_weight=t.get("post"), gate=t.get("gate"), pre_weight=t.get("pre"),
                         scale=scale, zero_centered=zero_centered, eps=EPS)
    grads = dict(zip(names, torch.autograd.grad((h, y), leaves, (c["gh"], c["gy"]))))
    plain = residual_norm(c["x"], c["branch"], post_norm=post_norm, post_weight=c["post"], gate=c["gate"], pre_weight=c["pre"],
                          scale=scale, zero_centered=zero_centered, eps=EPS)
    assert torch.equal(plain[0], h) and torch.equal(plain[1], y)
    assert h.dtype == c["x"].dtype and y.dtype == c["branch"].dtype
    x, b, gh, gy = (c[n].double() for n in ("x", "branch", "gh", "gy"))
    rows, d = x.shape
    off = 1.0 if zero_centered else 0.0
    one = torch.ones(d, dtype=F64, device=x.device)
    post = one if c["post"] is None else c["post"].double() + off
    pre = one if c["pre"] is None else c["pre"].double() + off
    G = scale * (one[None] if c["gate"] is None else c["gate"].double().view(-1, d))
    of = torch.arange(rows, device=x.device) // (rows // G.shape[0])
    rb = (b.square().mean(-1, keepdim=True) + EPS).rsqrt() if post_norm else 1.0
    bh = b * rb
    n = bh * post
    want = x + G[of] * n
    _within("stream", h, want, x.abs() + (G[of] * n).abs())
    hs = h.detach().double()
    rh = (hs.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hh = hs * rh
    _within("y", y, hh * pre, (hh * pre).abs())
    a = gy * pre
    m = (a * hh).mean(-1, keepdim=True)
    dx = gh + rh * (a - hh * m)
    mx = gh.abs() + rh * (a.abs() + hh.abs() * (a * hh).abs().mean(-1, keepdim=True))
    _within("dx", grads["x"], dx, mx)
    u, mu = dx * G[of] * post, mx * (G[of] * post).abs()
    db, mb = (rb * (u - bh * (u * bh).mean(-1, keepdim=True)), rb * (mu + bh.abs() * (mu * bh.abs()).mean(-1, keepdim=True))) \
        if post_norm else (u, mu)
    # sums over a row of terms that are themselves off by 64 roundings
    _within("dbranch", grads["branch"], db, mb, 160)
    if c["pre"] is not None:
        _within("dpre", grads["pre"], (gy * hh).sum(0), (gy * hh).abs().sum(0), rows + 64)
    if c["post"] is not None:
        _within("dpost", grads["post"], (dx * G[of] * bh).sum(0), (mx * (G[of] * bh).abs()).sum(0), rows + 128)
    if c["gate"] is not None:
        z = torch.zeros_like(G)
        dg, mg = z.index_add(0, of, scale * dx * n), z.index_add(0, of, abs(scale) * mx * n.abs())
        _within("dgate", grads["gate"].view(-1, d), dg, mg, rows // G.shape[0] + 128)


@pytest.mark.parametrize("d", [1, 7, 8, 33, 64, 100, 128, 200, 256, 500, 512, 513, 768, 1000, 1024, 2000, 2048, 4095, 4096, 5000,
                               8192, 9001, 16384])
@pytest.mark.parametrize("types", TYPES)
def test_widths(device, d, types):
    _check(_case(device, 37, d, types, gate=0, seed=d))
    _check(_case(device, 5, d, types, gate=5, post=False, seed=d, gate_dtype=types[1]))


@pytest.mark.parametrize("rows, gate", [(1, 1), (1, 0), (2, 2), (6, 3), (64, 4), (1000, 8), (1000, 500), (4000, 1), (4000, 2), (9000, 3),
                                        (5003, 0), (3, None), (20000, 20000), (20000, 10000)])
@pytest.mark.parametrize("d", [40, 200, 768])
def test_rows_and_gates(device, rows, gate, d):
    for i, types in enumerate(TYPES):
        _check(_case(device, rows, d, types, gate, seed=rows, gate_dtype=BF16 if i == 1 else F32))


@pytest.mark.parametrize("rows, gate", [(1, 1), (6, 3), (300, 300), (1000, 500), (600, 2), (2000, 1000), (700, 1), (700, 0)])
def test_gates_of_wide_rows(device, rows, gate):
    """Whose sums over rows are formed apart from the rows' own gradients."""
    for i, types in enumerate(TYPES):
        _check(_case(device, rows, 4104, types, gate, seed=rows, gate_dtype=BF16 if i == 1 else F32))


def test_without_weights_and_around_zero(device):
    c = _case(device, 50, 96, (BF16, BF16), gate=5)
    c["pre"] -= 1
    c["post"] -= 1
    _check(c, zero_centered=True)
    c["pre"] = c["post"] = None
    _check(c, post_norm=True, zero_centered=True)
    _check(c, post_norm=False, scale=-2.0)


def test_axes_strides_and_gates_of_sequences(device):
    c = _case(device, 60, 48, (BF16, BF16), gate=3)
    want = residual_norm(c["x"], c["branch"], gate=c["gate"], pre_weight=c["pre"])
    wide = torch.cat([c["x"], c["x"]], -1).view(3, 20, 96)[..., :48]  # rows 96 apart
    for gate in (c["gate"], c["gate"][:, None]):
        got = residual_norm(wide, c["branch"].view(3, 20, 48), gate=gate, pre_weight=c["pre"])
        for a, b in zip(got, want):
            assert a.shape == (3, 20, 48) and torch.equal(a.view(60, 48), b)
    gate = c["gate"].clone().requires_grad_()
    h, y = residual_norm(wide, c["branch"].view(3, 20, 48), gate=gate[:, None], pre_weight=c["pre"])
    (d,) = torch.autograd.grad(h.sum(), gate)
    assert d.shape == gate.shape


@pytest.mark.parametrize("d", [300, 5000])
def test_one_result_alone_and_one_gradient_alone(device, d):
    c = _case(device, 70, d, (BF16, BF16), gate=7)
    names = ("x", "branch", "post", "gate", "pre")
    leaves = [c[n].requires_grad_() for n in names]
    call = lambda ls: residual_norm(ls[0], ls[1], post_weight=ls[2], gate=ls[3], pre_weight=ls[4], scale=0.7)  # noqa: E731
    both = torch.autograd.grad(call(leaves), leaves, (c["gh"], c["gy"]))
    zero_h = torch.autograd.grad(call(leaves), leaves, (torch.zeros_like(c["gh"]), c["gy"]))
    zero_y = torch.autograd.grad(call(leaves), leaves[:4], (c["gh"], torch.zeros_like(c["gy"])))
    for a, b in zip(zero_h, torch.autograd.grad(call(leaves)[1], leaves, c["gy"])):
        assert torch.equal(a, b)
    for a, b in zip(zero_y, torch.autograd.grad(call(leaves)[0], leaves[:4], c["gh"])):
        assert torch.equal(a, b)
    for i in range(5):
        one = [t.detach() for t in leaves]
        one[i] = one[i].requires_grad_()
        (d,) = torch.autograd.grad(call(one), [one[i]], (c["gh"], c["gy"]))
        assert torch.equal(d, both[i])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", [(1, 8), (9, 100), (3, 5, 768), (300, 2048)])
def test_rms_norm(device, types, shape):
    c = _case(device, 1, shape[-1], types, seed=3)
    g = torch.Generator(device=device).manual_seed(4)
    x = torch.randn(*shape, device=device, generator=g).to(types[0]).requires_grad_()
    w = c["pre"].clone().requires_grad_()
    gy = torch.randn(*shape, device=device, generator=g).to(types[1])
    y = rms_norm(x, w, dtype=types[1], eps=EPS)
    assert y.dtype == types[1] and torch.equal(y, rms_norm(x.detach(), w.detach(), dtype=types[1], eps=EPS))
    dx, dw = torch.autograd.grad(y, (x, w), gy)
    X, W, GY = x.detach().double().view(-1, shape[-1]), w.detach().double(), gy.double().view(-1, shape[-1])
    r = (X.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh, a = X * r, GY * W
    _within("y", y.detach().view_as(X), xh * W, (xh * W).abs())
    _within("dx", dx.view_as(X), r * (a - xh * (a * xh).mean(-1, keepdim=True)), r * (a.abs() + xh.abs() * (a * xh).abs().mean(-1, keepdim=True)))
    _within("dw", dw, (GY * xh).sum(0), (GY * xh).abs().sum(0), X.shape[0] + 64)


def test_no_rows(device):
    x = torch.zeros(0, 64, device=device, requires_grad=True)
    w = torch.ones(64, device=device, requires_grad=True)
    p = torch.ones(64, device=device, requires_grad=True)
    h, y = residual_norm(x, x.detach(), post_weight=p, pre_weight=w)
    assert h.shape == y.shape == (0, 64)
    for d in torch.autograd.grad((h, y), (w, p), (torch.zeros_like(h), torch.zeros_like(y)), allow_unused=True):
        assert d is None or not d.any()


def test_rows_far_from_one(device):
    """Squares past fp32's range, rows of zeros, and infinities and NaN that stay in their rows."""
    for types in TYPES:
        c = _case(device, 12, 300, types, seed=9)
        clean = residual_norm(c["x"], c["branch"], post_weight=c["post"], pre_weight=c["pre"])
        c["branch"][2] *= 2.0**100
        c["x"][3] *= 2.0**100
        c["x"][4] = 0
        c["branch"][4] = 0
        h, y = residual_norm(c["x"], c["branch"], post_weight=c["post"], pre_weight=c["pre"])
        b = c["branch"].double()
        n = b / (b.square().mean(-1, keepdim=True) + EPS).sqrt() * c["post"].double()
        _within("stream", h, c["x"].double() + n, c["x"].double().abs() + n.abs())
        hs = h.double()
        want = hs / (hs.square().mean(-1, keepdim=True) + EPS).sqrt() * c["pre"].double()
        _within("y", y, want, want.abs())
        assert not h[4].any() and not y[4].any()
        c["x"][5, 7], c["branch"][6, 1] = float("nan"), float("inf")
        h, y = residual_norm(c["x"], c["branch"], post_weight=c["post"], pre_weight=c["pre"])
        rest = [0, 1, 7, 8, 9, 10, 11]
        assert torch.equal(h[rest], clean[0][rest]) and torch.equal(y[rest], clean[1][rest])
        assert torch.isnan(y[5]).all() and torch.isnan(h[6, 1])


def test_twice_the_same(device):
    c = _case(device, 3000, 640, (BF16, BF16), gate=3)
    run = lambda: ops.residual_norm_bwd(c["x"], c["branch"], st, c["gh"], c["gy"], post_weight=c["post"], gate=c["gate"],  # noqa: E731
                                        pre_weight=c["pre"])
    _, _, st = ops.residual_norm_fwd(c["x"], c["branch"], post_weight=c["post"], gate=c["gate"], pre_weight=c["pre"], want_stats=True)
    first = run()
    for _ in range(3):
        for a, b in zip(first, run()):
            assert torch.equal(a, b)


def test_refusals(device):
    c = _case(device, 6, 16, (BF16, BF16))
    with pytest.raises(L.PDError):
        residual_norm(c["x"], c["branch"].cpu())
    with pytest.raises(L.PDError):
        residual_norm(c["x"], c["branch"], pre_weight=c["pre"].cpu())
    h, y, st = ops.residual_norm_fwd(c["x"], c["branch"], want_stats=True)
    for bad in (dict(d_y=y[:5]), dict(d_stream=h.float()), dict(stats=st[:, :1])):
        kw = dict(dict(stats=st, d_stream=h, d_y=y), **bad)
        with pytest.raises(L.PDError):
            ops.residual_norm_bwd(h, c["branch"], kw["stats"], kw["d_stream"], kw["d_y"])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("d", [8, 300, 768, 5000, 9000])
@pytest.mark.parametrize("eps", [0.0, 1e-38])
def test_rows_whose_squares_vanish(device, types, d, eps):
    """Rows whose squares are below fp32's numbers, where eps does not hide them, beside ordinary ones."""
    c = _case(device, 9, d, types, seed=d)
    for r, e in ((1, -70), (2, -90), (3, -115), (5, -64)):
        c["branch"][r] *= 2.0**e
    for r, e in ((3, -100), (4, -80), (6, -66)):
        c["x"][r] *= 2.0**e
    c["post"][:] = 2.0**-60  # so that streams may be small too
    c["branch"][6] *= 2.0**-70
    h, y = residual_norm(c["x"], c["branch"], post_weight=c["post"], pre_weight=c["pre"], eps=eps)
    b = c["branch"].double()
    n = b * (b.square().mean(-1, keepdim=True) + eps).rsqrt() * c["post"].double()
    _within("stream", h, c["x"].double() + n, c["x"].double().abs() + n.abs())
    hs = h.double()
    want = hs * (hs.square().mean(-1, keepdim=True) + eps).rsqrt() * c["pre"].double()
    _within("y", y, want, want.abs())
    for x in (c["x"], c["branch"].to(types[0])):
        x, w, gy = x.clone().requires_grad_(), c["pre"].clone().requires_grad_(), c["gy"]
        y = rms_norm(x, w, dtype=types[1], eps=eps)
        X, W, GY = x.detach().double(), w.detach().double(), gy.double()
        r = (X.square().mean(-1, keepdim=True) + eps).rsqrt()
        xh, a = X * r, GY * W
        _within("rms", y.detach(), xh * W, (xh * W).abs())
        dx, dw = torch.autograd.grad(y, (x, w), gy)
        _within("dx", dx, r * (a - xh * (a * xh).mean(-1, keepdim=True)), r * (a.abs() + xh.abs() * (a * xh).abs().mean(-1, keepdim=True)))
        _within("dw", dw, (GY * xh).sum(0), (GY * xh).abs().sum(0), 9 + 64)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", [(20000, 768), (6001, 4096), (40, 16384), (100000, 33), (1, 1)])
def test_rms_norm_of_many_and_of_wide_rows(device, types, shape):
    g = torch.Generator(device=device).manual_seed(5)
    x = torch.randn(*shape, device=device, generator=g).to(types[0]).requires_grad_()
    w = (1 + 0.2 * torch.randn(shape[1], device=device, generator=g)).requires_grad_()
    gy = torch.randn(*shape, device=device, generator=g).to(types[1])
    y = rms_norm(x, w, dtype=types[1], eps=EPS)
    dx, dw = torch.autograd.grad(y, (x, w), gy)
    X, W, GY = x.detach().double(), w.detach().double(), gy.double()
    r = (X.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh, a = X * r, GY * W
    _within("y", y.detach(), xh * W, (xh * W).abs())
    _within("dx", dx, r * (a - xh * (a * xh).mean(-1, keepdim=True)), r * (a.abs() + xh.abs() * (a * xh).abs().mean(-1, keepdim=True)))
    _within("dw", dw, (GY * xh).sum(0), (GY * xh).abs().sum(0), shape[0] + 64)


@pytest.mark.parametrize("rows, d, gate", [(900, 8192, 3), (700, 5000, 700), (300, 9001, 1), (5000, 40, 5000)])
def test_twice_the_same_in_other_plans(device, rows, d, gate):
    c = _case(device, rows, d, (BF16, BF16), gate=gate)
    kw = dict(post_weight=c["post"], gate=c["gate"], pre_weight=c["pre"])
    h, _, st = ops.residual_norm_fwd(c["x"], c["branch"], want_stats=True, **kw)
    first = ops.residual_norm_bwd(h, c["branch"], st, c["gh"], c["gy"], **kw)
    for _ in range(3):
        for a, b in zip(first, ops.residual_norm_bwd(h, c["branch"], st, c["gh"], c["gy"], **kw)):
            assert torch.equal(a, b)
