"""Routing by scores against the definition in 64 bits: the choice is equal, weights and gradients within
their roundings (a score, its exponential and a sum of at most 64 of them: 64 roundings of 2^-24, those of
an exponent's argument up to 16 included; bf16 gradients half a step more)."""

import pytest
import torch

from param_decomp_amd import _lib as L
from param_decomp_amd import ops
from param_decomp_amd.routed import experts

pytestmark = pytest.mark.gpu

U = 2.0**-24
INF = float("inf")


def _expected(x, k, scoring="softmax", bias=None, n_groups=1, top_groups=None, renormalize=True, scale=1.0):
    x = x.double()
    T, E = x.shape
    s = torch.softmax(x, -1) if scoring == "softmax" else torch.sigmoid(x)
    masked = x == -INF
    s = torch.where(masked & ~torch.isnan(s), torch.zeros_like(s), s)
    key = x if bias is None and (n_groups == 1 or top_groups in (None, n_groups)) else s if bias is None else s + bias.double()
    key = torch.where(torch.isnan(key), torch.full_like(key, INF), key)
    key = torch.where(masked, torch.full_like(key, -INF), key)
    if top_groups not in (None, n_groups):
        best = key.view(T, n_groups, -1).sort(-1, descending=True).values[..., :2]
        score = torch.where(best > -INF, best, torch.zeros_like(best)).sum(-1).masked_fill((best == -INF).all(-1), -INF)
        keep = score.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
        ok = torch.zeros(T, n_groups, dtype=torch.bool, device=x.device).scatter_(1, keep, True).repeat_interleave(E // n_groups, 1)
        # what groups leave out comes behind what is masked inside them
        order = torch.where(ok, key, torch.full_like(key, -INF)).sort(dim=-1, descending=True, stable=True).indices
        idx = torch.stack([o[ok[r, o]][:k] for r, o in enumerate(order)]) if T else order[:, :k]
    else:
        idx = key.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    c = s.gather(1, idx)
    if renormalize:
        l = x.gather(1, idx) if scoring == "softmax" else torch.nn.functional.logsigmoid(x.gather(1, idx))
        c = torch.softmax(l, -1)
        c = torch.where((l == -INF).all(-1, keepdim=True), torch.zeros_like(c), c)
    elif scoring == "softmax":
        c = torch.where(masked.all(-1, keepdim=True), torch.zeros_like(c), c)
    return c * scale, idx


def _check(device, x, k, seed=0, **kw):
    w, idx = experts.route_scores(x, k, **kw)
    want, at = _expected(x, k, **kw)
    assert torch.equal(idx.long(), at)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32
    assert ((w.double() - want).abs() <= 64 * U * want.abs() + 1e-37).all()
    # gradients, through 64-bit autograd at the same choice
    g = torch.randn(w.shape, device=device, generator=torch.Generator(device=device).manual_seed(seed))
    leaf = x.clone().requires_grad_()
    (d,) = torch.autograd.grad(experts.route_scores(leaf, k, **kw)[0], leaf, g)
    y = x.double().requires_grad_()
    scale, renorm = kw.get("scale", 1.0), kw.get("renormalize", True)
    if kw.get("scoring", "softmax") == "softmax":
        c = torch.softmax(y.gather(1, at) if renorm else y, -1)
        c = c if renorm else c.gather(1, at)
    else:
        c = torch.softmax(torch.nn.functional.logsigmoid(y.gather(1, at)), -1) if renorm else torch.sigmoid(y).gather(1, at)
    (r,) = torch.autograd.grad(c * scale, y, g.double())
    mag = abs(scale) * (g.double().abs() * c.detach()).sum(-1, keepdim=True) + abs(scale) * g.double().abs().amax(-1, keepdim=True)
    half = 2.0**-8 if x.dtype == torch.bfloat16 else U
    s = torch.softmax(y.detach(), -1) if kw.get("scoring", "softmax") == "softmax" else torch.sigmoid(y.detach())
    near = torch.zeros_like(r).scatter_(1, at, c.detach()) + (s if not renorm else 0)
    assert ((d.double() - r).abs() <= 64 * U * mag * (near + 1e-30) + half * r.abs() + 1e-37).all()
    if not (kw.get("scoring", "softmax") == "softmax" and not renorm):
        out = torch.ones_like(x, dtype=torch.bool).scatter_(1, at, False)
        assert not d[out].any()


def _x(device, T, E, dtype, seed=0, scale=1.5):
    return (torch.randn(T, E, device=device, generator=torch.Generator(device=device).manual_seed(seed)) * scale).to(dtype)


KINDS = [dict(), dict(renormalize=False), dict(scoring="sigmoid"), dict(scoring="sigmoid", renormalize=False, scale=2.5)]


@pytest.mark.parametrize("E, k", [(1, 1), (2, 2), (7, 3), (8, 8), (42, 8), (63, 5), (64, 64), (65, 6), (128, 8), (129, 9), (200, 16),
                                  (256, 8), (384, 6), (512, 10), (600, 40), (1024, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_choice_weights_and_gradients(device, E, k, dtype):
    for i, kind in enumerate(KINDS):
        for bias in (False, True):
            kw = dict(kind, bias=torch.randn(E, device=device, generator=torch.Generator(device=device).manual_seed(E)) * 0.2 if bias else None)
            _check(device, _x(device, 67, E, dtype, E + i), k, **kw)


@pytest.mark.parametrize("E, groups, top, k", [(8, 8, 3, 2), (16, 4, 2, 8), (42, 6, 2, 5), (64, 64, 9, 9), (72, 9, 4, 8), (128, 8, 3, 16),
                                               (160, 8, 3, 6), (256, 8, 4, 8), (256, 32, 5, 8), (384, 6, 1, 7), (512, 2, 1, 12),
                                               (1024, 64, 7, 30), (256, 8, 8, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_groups(device, E, groups, top, k, dtype):
    for i, kind in enumerate(KINDS):
        for bias in (False, True):
            b = torch.randn(E, device=device, generator=torch.Generator(device=device).manual_seed(E)) * 0.3 - 0.5 if bias else None
            _check(device, _x(device, 45, E, dtype, E + i), k, **dict(kind, bias=b, n_groups=groups, top_groups=top))


@pytest.mark.parametrize("T", [1, 2, 31, 1000, 4097])
def test_rows(device, T):
    _check(device, _x(device, T, 96, torch.float32, T), 7, scoring="sigmoid")


def test_no_rows(device):
    w, idx = experts.route_scores(torch.zeros(0, 16, device=device), 3)
    assert w.shape == idx.shape == (0, 3)
    x = torch.zeros(0, 16, device=device, requires_grad=True)
    (d,) = torch.autograd.grad(experts.route_scores(x, 3)[0].sum(), x)
    assert d.shape == (0, 16)


@pytest.mark.parametrize("E, k", [(16, 4), (128, 8), (256, 8), (300, 20), (1024, 64)])
def test_equal_scores_go_to_the_lower_index(device, E, k):
    for dtype in (torch.float32, torch.bfloat16):
        zeros = torch.zeros(9, E, device=device, dtype=dtype)
        few = (_x(device, 200, E, torch.float32, 3) * 2).round().div(4).to(dtype)
        bias = (torch.arange(E, device=device) % 3).float() / 4
        for x in (zeros, few):
            for kind in KINDS:
                _check(device, x, k, **kind)
                _check(device, x, k, **dict(kind, bias=bias))
                _check(device, x, k, **dict(kind, bias=bias, n_groups=4, top_groups=2))
                _check(device, x, k, **dict(kind, n_groups=4, top_groups=2))


def test_scores_closer_than_fp32_tells_apart(device):
    """Scores a few 2^-30 apart, on both sides of the last place chosen, in every order of index."""
    E, k = 128, 8
    g = torch.Generator(device=device).manual_seed(5)
    for base in (4.0, 9.0, -3.0):
        x = torch.full((64, E), -6.0, device=device)
        for r in range(64):
            at = torch.randperm(E, device=device, generator=g)[:12]
            x[r, at] = base + torch.arange(12, device=device) * 2.0**-20
        for kind in KINDS:
            _check(device, x, k, **kind)
            _check(device, x, k, **dict(kind, bias=torch.full((E,), 0.37, device=device)))
            _check(device, x, k, **dict(kind, n_groups=8, top_groups=6))


def test_masked_experts(device):
    E = 64
    for dtype in (torch.float32, torch.bfloat16):
        x = _x(device, 40, E, dtype, 6)
        x[:, 5:20] = -INF
        x[0] = -INF           # nothing left
        x[1, :-3] = -INF      # fewer left than are chosen
        x[2, 1:] = -INF
        for i, kind in enumerate(KINDS):
            for kw in (dict(), dict(bias=torch.linspace(-1, 1, E, device=device)), dict(n_groups=8, top_groups=3)):
                w, idx = experts.route_scores(x, 6, **kind, **kw)
                want, at = _expected(x, 6, **kind, **kw)
                assert torch.equal(idx.long(), at)
                assert ((w.double() - want).abs() <= 64 * U * want.abs()).all()
                assert not w[0].any() and torch.isfinite(w).all()
                leaf = x.clone().requires_grad_()
                (d,) = torch.autograd.grad(experts.route_scores(leaf, 6, **kind, **kw)[0].sum(), leaf)
                assert torch.isfinite(d).all() and not d[0].any() and not d[x == -INF].any()


def test_a_nan_shows_and_stays_in_its_row(device):
    for dtype in (torch.float32, torch.bfloat16):
        x = _x(device, 10, 40, dtype, 7)
        clean = experts.route_scores(x, 4, scoring="sigmoid")
        x[3, 17] = float("nan")
        for kind in KINDS:
            for kw in (dict(), dict(bias=torch.zeros(40, device=device)), dict(n_groups=4, top_groups=2)):
                w, idx = experts.route_scores(x, 4, **kind, **kw)
                assert torch.isnan(w[3]).any() and torch.isfinite(w[[0, 1, 2, 4, 5]]).all()
                assert ((idx >= 0) & (idx < 40)).all() and len(set(idx[3].tolist())) == 4
        w, idx = experts.route_scores(x, 4, scoring="sigmoid")
        assert torch.equal(idx[4:], clean[1][4:]) and torch.equal(w[4:], clean[0][4:])


def test_sigmoids_that_underflow_together(device):
    x = torch.full((3, 16), -200.0, device=device)
    x[:, 3:6] = torch.tensor([-150.0, -149.0, -151.0], device=device)
    _check(device, x, 3, scoring="sigmoid")


def test_extreme_biases(device):
    for b in (1e4, 1e30):
        bias = torch.linspace(-b, b, 64, device=device)
        _check(device, _x(device, 20, 64, torch.float32, 8), 5, scoring="sigmoid", bias=bias)


def test_strided_logits_and_the_routed_jobs(device):
    wide = _x(device, 50, 96, torch.bfloat16, 9)
    a = experts.route_scores(wide[:, 16:58], 8)
    b = experts.route_scores(wide[:, 16:58].contiguous(), 8)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # softmax, renormalised: what route_tokens gives
    _, idx, w = experts.route_tokens(wide[:, 16:58].float(), 8)
    assert torch.equal(idx, a[1]) and ((w - a[0]).abs() <= 64 * U).all()
    jobs = experts.routed_jobs(a[1], 42)
    assert int(jobs.group_sizes.sum()) == 400


def test_refusals(device):
    x = _x(device, 4, 16, torch.float32)
    with pytest.raises(L.PDError):
        experts.route_scores(x, 2, bias=torch.zeros(16))
    with pytest.raises(L.PDError):
        ops.route_scores_fwd(x.t(), 2)
    _, idx = ops.route_scores_fwd(x, 2)
    with pytest.raises(L.PDError):
        ops.route_scores_bwd(x, idx, torch.zeros(4, 2))


def _apart(E, n):
    """n experts, each in a lane of its own and at another place of it (or, where E is small, the last n)."""
    return torch.arange(n) * 9 if E >= 64 else torch.arange(E - n, E)


@pytest.mark.parametrize("E, masked, groups", [(8, 6, 1), (8, 1, 1), (8, 7, 1), (8, 5, 2), (42, 5, 1), (42, 5, 6), (64, 8, 1), (64, 8, 8),
                                               (100, 6, 1), (100, 6, 4), (600, 12, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_bias_does_not_bring_masked_experts_back(device, E, masked, groups, dtype):
    """Masked experts whose words differ, a bias in their favour, and k below, at and above the number that is left."""
    gone = _apart(E, masked).to(device)
    bias = torch.linspace(-0.2, 0.2, E, device=device)
    bias[gone] += 0.9
    x = _x(device, 30, E, dtype, E + masked)
    x[:, gone] = -INF
    for kind in KINDS:
        for top in sorted({groups, groups - 1 or 1}):
            size = E // groups
            for k in {1, 2, E - masked - 1, E - masked, E - masked + 1, E}:
                if not 1 <= k <= min(64, size * top):
                    continue
                kw = dict(kind, bias=bias, n_groups=groups, top_groups=top)
                w, idx = experts.route_scores(x, k, **kw)
                want, at = _expected(x, k, **kw)
                assert torch.equal(idx.long(), at), (kind, top, k)
                assert ((w.double() - want).abs() <= 64 * U * want.abs() + 1e-37).all()
                leaf = x.clone().requires_grad_()
                (d,) = torch.autograd.grad(experts.route_scores(leaf, k, **kw)[0].sum(), leaf)
                assert torch.isfinite(d).all() and not d[x == -INF].any()


def test_one_masked_expert_beside_a_live_one(device):
    x = torch.full((1, 8), -INF, device=device)
    x[0, :2] = torch.tensor([1.0, -1.0])
    bias = torch.tensor([0, 0, 0.9, 0.9, 0.9, 0.9, 0.9, 0.9], device=device)
    w, idx = experts.route_scores(x, 2, scoring="sigmoid", bias=bias)
    assert idx.tolist() == [[0, 1]] and (w > 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equal_scores_of_unequal_logits(device, dtype):
    """Scores that are one number in 64 bits (saturated sigmoids, exponentials of logits next to zero): inside groups the
    lower index is first, wherever the experts lie in their lanes."""
    E, groups = 64, 8
    for places in ([0, 9, 2, 11], [0, 8, 2, 10], [7, 6, 5, 4], [15, 14, 1, 0], [3, 11, 6, 5]):
        for a, b, kind in ((40.0, 41.0, dict(scoring="sigmoid")), (300.0, 38.0, dict(scoring="sigmoid", renormalize=False)),
                           (0.0, 1e-20, dict()), (1e-20, -1e-20, dict(renormalize=False))):
            x = _x(device, 2, E, torch.float32, 11, 0.1) - 6
            x[0, places] = torch.tensor([a, b, a, b], device=device)
            x[1, places] = torch.tensor([b, a, b, a], device=device)
            for k in (1, 2, 3, 4, 6):
                _check(device, x.to(dtype), k, **dict(kind, n_groups=groups, top_groups=2))


@pytest.mark.parametrize("E, k", [(8, 2), (42, 8), (256, 8), (600, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_an_index_that_a_row_holds_twice(device, E, k, dtype):
    """A choice of the caller's own: what its places give is added."""
    x = _x(device, 50, E, dtype, E)
    g = torch.Generator(device=device).manual_seed(k)
    at = torch.randint(E, (50, k), device=device, generator=g)
    at[::2, 1] = at[::2, 0]
    at[::4] = at[::4, :1]
    dw = torch.randn(50, k, device=device, generator=g)
    for sigmoid in (False, True):
        for renorm in (False, True):
            d = ops.route_scores_bwd(x, at.int(), dw, sigmoid=sigmoid, renormalize=renorm, scale=1.5)
            y = x.double().requires_grad_()
            s = torch.sigmoid(y) if sigmoid else torch.softmax(y, -1)
            chosen = y.gather(1, at)  # renormalised from these alone: 64-bit roundings of the others are no gradient
            c = torch.softmax(torch.nn.functional.logsigmoid(chosen) if sigmoid else chosen, -1) if renorm else s.gather(1, at)
            (want,) = torch.autograd.grad(1.5 * c, y, dw.double())
            # each place: 64 roundings of its two terms; k of them are added, and those of the row's sum with them
            per = 1.5 * c.detach() * (dw.double().abs() + (c.detach() * dw.double().abs()).sum(-1, keepdim=True))
            mag = torch.zeros_like(want).scatter_add(1, at, per) + s.detach() * per.sum(-1, keepdim=True) * (not renorm)
            half = 2.0**-8 if dtype == torch.bfloat16 else U
            bound = (64 + k) * U * mag + half * (want.abs() + (64 + k) * U * mag) + 1e-37
            assert ((d.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_of_sigmoids_that_leave_fp32_beside_others(device, dtype):
    """Scores below fp32 whose share of the chosen ones' sum is not, beside masked experts. A logarithm is off by a few
    2^-24 of itself, and a weight by as much: 110 is the largest here."""
    x = torch.full((6, 24), -INF, device=device)
    for r, v in enumerate(([-33.75, -89.5], [-40.0, -90.0, -102.5], [-13.5, -95.0, -88.0], [-99.5, -26.875], [-31.75, -101.0, -31.0], [-60.0, -110.0])):
        x[r, 7:7 + 5 * len(v):5] = torch.tensor(v, device=device)
    x = x.to(dtype)
    for k in (2, 3, 8):
        w, idx = experts.route_scores(x, k, scoring="sigmoid", scale=1.5)
        want, at = _expected(x, k, scoring="sigmoid", scale=1.5)
        assert torch.equal(idx.long(), at) and (want[:, :2] > 1e-37).all()
        assert ((w.double() - want).abs() <= (64 + 2 * 110) * U * want).all()
