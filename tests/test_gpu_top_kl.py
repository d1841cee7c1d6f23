"""KL to a teacher's top logits against its definition in 64 bits.

Bounds, with u half a step of the gradient's type and e = 2^-24: a sum of exponentials takes
at most 512 additions a thread holds in turn (a few more across threads), each exponential
an error of a few e and e times its exponent's size, so log q of an entry is off by
g = (600 + 4 range) e, range the row's spread of logits / temperature:
  kl:   g (P + rest) + 4 e |kl|;  dz: u |dz| + s (P q + p [+ rest q / S_r]) (2 g)."""

import math

import pytest
import torch

from param_decomp_amd import _lib as L
from param_decomp_amd import losses, ops

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E = 2.0**-24


def _inputs(device, rows, V, k, dtype, tau=1.0, seed=0, top_dtype=None):
    g = torch.Generator(device=device).manual_seed(seed)
    clean = torch.empty(rows, V, device=device).exponential_(generator=g) * 1.6
    top = clean.topk(k, -1)
    values = top.values.to(top_dtype or dtype)
    lse = torch.maximum(torch.logsumexp(clean / tau, -1), torch.logsumexp(values.float() / tau, -1))
    z = (clean + torch.randn(rows, V, device=device, generator=g) * 0.7).to(dtype)
    w = torch.rand(rows, device=device, generator=g) + 0.1
    return z, values, top.indices.to(torch.int32), lse, w


def _definition(z, top, idx, lse, tau, w):
    """(kl, grad), (bounds) row by row in 64 bits; entries outside [0, V) are absent."""
    rows, V = z.shape
    u = torch.finfo(z.dtype).eps / 2
    Z, t, at = z.double() / tau, top.double() / tau, idx.long()
    ok = (at >= 0) & (at < V)
    logq = torch.log_softmax(Z, -1)
    t = t.masked_fill(~ok, -math.inf)
    at = at.clamp(0, V - 1)
    logp = t - (torch.logsumexp(t, -1, keepdim=True) if lse is None else lse.double()[:, None])
    p = torch.where(ok, logp.exp(), torch.zeros_like(t))
    target = torch.zeros_like(Z).scatter_add_(1, at, p)
    listed = torch.zeros_like(Z).scatter_add_(1, at, ok.double()) > 0
    term = torch.where(p > 0, p * (logp - logq.gather(1, at)), torch.zeros_like(p))
    kl = term.sum(-1)
    P = p.sum(-1, keepdim=True)
    rest = torch.zeros_like(P)
    share = torch.zeros_like(Z)
    if lse is not None:
        rest = 1 - P
        rest = torch.where((rest < 2.0**-20) | listed.all(-1, keepdim=True), torch.zeros_like(rest), rest)
        qr = logq.masked_fill(listed, -math.inf)
        lr = torch.logsumexp(qr, -1, keepdim=True)
        kl = kl + torch.where(rest > 0, rest * (rest.log() - lr), torch.zeros_like(rest))[:, 0]
        share = torch.where(rest > 0, rest * (qr - lr).exp(), torch.zeros_like(qr))
    s = w.double()[:, None] / tau
    grad = s * ((P + rest) * logq.exp() - target - share)
    finite = torch.where(torch.isfinite(Z), Z, torch.zeros_like(Z))
    g = (600 + 4 * (finite.amax(-1, keepdim=True) - finite.amin(-1, keepdim=True))) * E
    tk = (g * (P + rest))[:, 0] + 4 * E * kl.abs()
    tg = u * grad.abs() + s * 2 * g * ((P + rest) * logq.exp() + target + share)
    return (kl, grad), (tk + 1e-30, tg + 1e-30)


def _check(got, val, tol):
    for x, v, t, name in zip(got, val, tol, ("kl", "grad")):
        off = (x.double().reshape(v.shape) - v).abs()
        assert torch.isfinite(x.float()).all(), name
        assert (off <= t).all(), f"{name}: {(off / t).max().item():.3g} of the bound"


def _both(z, top, idx, lse, tau, w):
    """One call, and the autograd pair: the same bits."""
    fused = ops.top_logits_kl(z, top, idx, clean_lse=lse, temperature=tau, row_weight=w, want_grad=True)
    leaf = z.detach().requires_grad_()
    kl = losses.top_logits_position_kl(leaf, top, idx, clean_lse=lse, temperature=tau)
    (grad,) = torch.autograd.grad(kl, leaf, w)
    assert torch.equal(kl.detach(), fused[0]) and torch.equal(grad, fused[1])
    return fused


SIZES = [(1, 1, 1), (3, 2, 1), (4, 7, 7), (5, 8, 3), (2, 9, 4), (6, 100, 10), (3, 1000, 64), (3, 4089, 16), (2, 4096, 1),
         (3, 4097, 200), (2, 16381, 33), (2, 16385, 128), (3, 50277, 64), (2, 65536, 300), (2, 65537, 20),
         (2, 131072, 128), (2, 131073, 1024), (2, 200001, 50)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows, V, k", SIZES)
def test_sizes(device, dtype, rest, rows, V, k):
    for tau in (1.0, 1.7):
        z, top, idx, lse, w = _inputs(device, rows, V, k, dtype, tau, seed=V + k)
        args = (z, top, idx, lse if rest else None, tau, w)
        _check(_both(*args), *_definition(*args))


def test_largest_vocabulary(device):
    z, top, idx, lse, w = _inputs(device, 1, 1 << 19, 1024, BF16, seed=1)
    args = (z, top, idx, lse, 1.0, w)
    _check(_both(*args), *_definition(*args))


@pytest.mark.parametrize("rest", [False, True])
def test_many_rows(device, rest):
    z, top, idx, lse, w = _inputs(device, 3000, 301, 17, BF16, seed=3)
    args = (z, top, idx, lse if rest else None, 1.0, w)
    got = _both(*args)
    _check(got, *_definition(*args))
    for x, y in zip(got, _both(*args)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("rest", [False, True])
def test_padding_any_order_and_repeats(device, rest):
    """Absent entries (negative and past the vocabulary), entries in any order, 64-bit
    indices, and indices listed more than once (their p adds up)."""
    z, top, idx, lse, w = _inputs(device, 40, 600, 24, F32, seed=4)
    order = torch.randperm(24, device=device)
    top, idx = top[:, order].contiguous(), idx[:, order].contiguous().long()
    idx[::2, 3] = -1
    idx[1::3, 7] = 600
    idx[2, 5] = 1 << 40
    idx[5] = -100  # no entry at all
    idx[6, 1:] = -1  # one entry
    idx[9, 4], idx[9, 11], idx[9, 20] = idx[9, 2], idx[9, 2], idx[9, 6]
    idx[10] = idx[10, :1]
    top[9] -= 2.0  # repeated entries keep their mass below one
    top[10] = lse[10] - 4.0
    args = (z, top, idx, lse if rest else None, 1.0, w)
    got = _both(*args)
    if not rest:  # nothing listed: no loss (the definition's 0 / 0)
        assert got[0][5] == 0 and (got[1][5] == 0).all()
        keep = torch.arange(40, device=device) != 5
        args = (z[keep], top[keep], idx[keep], None, 1.0, w[keep])
        got = [t[keep] for t in got]
    _check(got, *_definition(*args))


def test_listed_entries_of_no_mass(device):
    z, top, idx, lse, w = _inputs(device, 8, 200, 10, F32, seed=5)
    top[:, 4:] = -math.inf
    for l in (None, lse):
        args = (z, top, idx, l, 1.0, w)
        _check(_both(*args), *_definition(*args))


def test_everything_listed_meets_the_full_kl(device):
    z, _, _, _, w = _inputs(device, 16, 300, 5, F32, seed=6)
    clean = torch.randn(16, 300, device=device) * 2
    top = clean.topk(300, -1)
    lse = torch.logsumexp(clean, -1)
    full = losses.categorical_kl_from_logits(z, clean)
    for l in (None, lse):
        kl = losses.top_logits_kl(z, top.values, top.indices, clean_lse=l)
        # both sides carry 32-bit sums of 300 exponentials
        assert abs(float(kl) - float(full)) <= 700 * E * (1 + abs(float(full)))
        args = (z, top.values, top.indices, l, 1.0, w)
        _check(_both(*args), *_definition(*args))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rest", [False, True])
def test_masked_vocabulary(device, dtype, rest):
    """Entries at -inf, and at the type's lowest value, have no mass and no gradient."""
    for low in (-math.inf, torch.finfo(dtype).min):
        z, top, idx, lse, w = _inputs(device, 6, 900, 8, dtype, seed=7)
        z[:, 600:] = low
        top, idx = z[:, :600].float().topk(8, -1)
        lse = torch.logsumexp(z[:, :600].float(), -1) + 0.01
        got = _both(z, top, idx.to(torch.int32), lse if rest else None, 1.0, w)
        assert (got[1][:, 600:] == 0).all()
        args = (z[:, :600].contiguous(), top, idx, lse if rest else None, 1.0, w)
        val, tol = _definition(*args)
        _check((got[0], got[1][:, :600]), val, tol)


def test_all_listed_entries_far_below_the_rest(device):
    """q of the listed entries underflows as a difference of sums; as a sum of their own
    it does not. And the rest's far below the listed ones."""
    z, top, idx, lse, w = _inputs(device, 4, 500, 6, F32, seed=8)
    low = z.clone()
    low.scatter_add_(1, idx.long(), torch.full((4, 6), -95.0, device=device))
    high = z.clone()
    high.scatter_add_(1, idx.long(), torch.full((4, 6), 95.0, device=device))
    for t in (low, high):
        args = (t, top, idx, lse, 1.0, w)
        _check(_both(*args), *_definition(*args))


def test_unweighted_rows_are_zeros(device):
    """Weight 0 gives zeros whatever the row holds, and NaN stays in its row."""
    z, top, idx, lse, w = _inputs(device, 9, 700, 12, BF16, seed=9)
    want = ops.top_logits_kl(z, top, idx, clean_lse=lse, row_weight=w, want_grad=True)
    for bad in (math.nan, math.inf):
        zb, wb = z.clone(), w.clone()
        zb[2, 5], zb[4, int(idx[4, 0])] = bad, bad
        wb[2] = 0
        kl, grad = ops.top_logits_kl(zb, top, idx, clean_lse=lse, row_weight=wb, want_grad=True)
        assert (grad[2] == 0).all() and torch.isnan(kl[2]) and torch.isnan(kl[4]) and torch.isnan(grad[4]).any()
        keep = [0, 1, 3, 5, 6, 7, 8]
        assert torch.equal(kl[keep], want[0][keep]) and torch.equal(grad[keep], want[1][keep])


def test_shapes_views_and_types(device):
    z, top, idx, lse, w = _inputs(device, 12, 333, 9, BF16, seed=10, top_dtype=F32)
    args = (z, top, idx, lse, 1.0, w)
    want = _both(*args)
    _check(want, *_definition(*args))
    kl, grad = ops.top_logits_kl(z.view(3, 4, 333), top.view(3, 4, 9), idx.view(3, 4, 9).long(),
                                 clean_lse=lse.view(3, 4), row_weight=w.view(3, 4), want_grad=True)
    assert kl.shape == (3, 4) and torch.equal(kl.flatten(), want[0]) and torch.equal(grad.view(12, 333), want[1])
    # rows that start at any 2-byte boundary, and a gradient aligned otherwise
    for lead in (1, 3, 8):
        shifted = torch.cat([z.flatten()[:lead], z.flatten()])[lead:].view(12, 333)
        # (threads hold other elements of a row there: its sums are in another order)
        _check(ops.top_logits_kl(shifted, top, idx, clean_lse=lse, row_weight=w, want_grad=True), *_definition(*args))
    wide = torch.cat([z, z], 1)
    leaf = wide.detach().requires_grad_()
    kl = losses.top_logits_position_kl(leaf[:, 333:], top, idx, clean_lse=lse)
    (g,) = torch.autograd.grad(kl, leaf, w)
    assert (g[:, :333] == 0).all() and torch.equal(g[:, 333:], want[1])
    assert ops.top_logits_kl(z, top, idx, want_kl=False) == (None, None)
    # no row weights: ones
    ones = ops.top_logits_kl(z, top, idx, row_weight=torch.ones_like(w), want_grad=True)
    for x, y in zip(ops.top_logits_kl(z, top, idx, want_grad=True), ones):
        assert torch.equal(x, y)


def test_no_rows(device):
    z, top, idx, lse, w = _inputs(device, 2, 50, 4, F32)
    kl, grad = ops.top_logits_kl(z[:0], top[:0], idx[:0], row_weight=w[:0], want_grad=True)
    assert kl.shape == (0,) and grad.shape == (0, 50)


def test_mean_and_its_gradient_by_differences(device):
    z, top, idx, lse, _ = _inputs(device, 7, 120, 10, F32, tau=1.3, seed=11)
    for l in (None, lse):
        leaf = z.clone().requires_grad_()
        loss = losses.top_logits_kl(leaf, top, idx, clean_lse=l, temperature=1.3)
        loss.backward()
        gen = torch.Generator(device=device).manual_seed(2)
        r = torch.randn(z.shape, dtype=F64, device=device, generator=gen)
        w = torch.ones(7, device=device)
        at = lambda t: _definition(z.double() + t * r, top, idx, l, 1.3, w)[0][0].mean()  # noqa: E731
        want = float(at(1e-5) - at(-1e-5)) / 2e-5
        have = float((leaf.grad.double() * r).sum())
        assert abs(want - have) <= 1e-4 * float((leaf.grad.double().abs() * r.abs()).sum())
        assert abs(float(loss) - float(at(0.0))) <= 700 * E * (1 + float(loss))


def test_stream_and_graph(device):
    static = list(_inputs(device, 30, 5000, 20, BF16, seed=0))

    def calls(z, top, idx, lse, w):
        return ops.top_logits_kl(z, top, idx, clean_lse=lse, row_weight=w, want_grad=True)

    want = calls(*static)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(device=device)
    with torch.cuda.stream(side):
        got = calls(*static)
    side.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls(*static)
    for i in range(3):
        for dst, src in zip(static, _inputs(device, 30, 5000, 20, BF16, seed=i + 1)):
            dst.copy_(src)
        for t in got:
            t.fill_(float("nan"))
        graph.replay()
        want = calls(*static)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_mixed_devices_are_refused(device):
    z, top, idx, lse, w = _inputs(device, 2, 50, 4, F32)
    with pytest.raises(L.PDError, match="top_indices is on cpu"):
        ops.top_logits_kl(z, top, idx.cpu())


def test_temperature_keeps_its_64_bits(device):
    """0.7 in 32 bits is 2^-25.8 off: of a logit of 30000 that would be 7e-4 in an exponent."""
    z, top, idx, _, w = _inputs(device, 40, 700, 8, F32, 0.7, seed=31)
    z, top = z + 30000, top + 30000
    clean = torch.logsumexp(top.double() / 0.7, -1) + 0.4
    args = (z, top, idx, clean.float(), 0.7, w)
    _check(_both(*args), *_definition(*args))
