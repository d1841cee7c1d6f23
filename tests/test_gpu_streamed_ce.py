"""The streamed cross entropy against the formula in 64 bits.

Tolerances: a logit is a sum of n = d products in fp32, off by at most (n + 1) 2^-24 sum |act head| =: e. An fp32
product is the sum of six of bf16 parts, what is left out below 2^-24 of it: n counts them, and 1 more each. The
loss is a difference of two of them and of a logarithm: 2 e and 16 2^-24 of what is added (it, the largest
logit's distance, 1). G's entries are off by (2 e + 16 2^-24) p g and, in bf16, by half a step (2^-8 of
them; the one-call form rounds to 2^-12 of them before, in fp16 relative to the largest of 64 neighbours:
2^15 p / p_max has steps of 2^-24 at least, which is 2^-39 of p_max <= 1, so 2^-40 g more); what is summed from them likewise times the other
operand, with n 2^-24 of the sum of magnitudes for n terms, and half a step of the result. The matrix cores take and give
no denormal numbers: each part of an entry, product and sum may be off by 2^-126 besides (the entries of G go down
to 10^-36 where logits are large, and their third parts to 10^-41)."""

import pytest
import torch

from param_decomp_amd import _lib as L
from param_decomp_amd import losses, ops

pytestmark = pytest.mark.gpu

F64, BF16, F32 = torch.float64, torch.bfloat16, torch.float32
U = 2.0**-24
TINY = 2.0**-126
HALF = {BF16: 2.0**-8, F32: U}


def _inputs(device, N, d, V, dtype, seed=0, skip=0.0, scale=1.0, bits=64):
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    act, head = rnd(N, d).to(dtype), (rnd(V, d) * (2 * scale / d**0.5)).to(dtype)
    t = torch.randint(V, (N,), device=device, generator=g)
    off = torch.rand(N, device=device, generator=g) < skip
    t = torch.where(off, torch.tensor([-100, -1, V, V + 7], device=device)[torch.arange(N, device=device) % 4], t)
    w = torch.randn(N, device=device, generator=g)
    return act, head, t.to(torch.int32 if bits == 32 else torch.int64), w


def _expected(act, head, t, w):
    """(loss, d_act, d_head) and their bounds, in 64 bits."""
    dt, (N, d), V = act.dtype, act.shape, head.shape[0]
    a, h, w = act.double(), head.double(), w.double()
    on = (t >= 0) & (t < V)
    a = torch.where(on[:, None], a, torch.zeros_like(a))
    w = torch.where(on, w, torch.zeros_like(w))
    many = 1 if dt == BF16 else 7  # products and roundings for each
    z, e = a @ h.T, (many * d + 1) * U * (a.abs() @ h.abs().T)
    at = t.long().clamp(0, V - 1)[:, None]
    lp = torch.log_softmax(z, -1)
    loss = torch.where(on, -lp.gather(1, at)[:, 0], torch.zeros(N, dtype=F64, device=z.device))
    spread = z.amax(-1) - z.gather(1, at)[:, 0]
    bl = 2 * e.amax(-1) + 16 * U * (1 + loss.abs() + spread.abs())
    p = lp.exp()
    G = (p.scatter_add(1, at, -torch.ones_like(p[:, :1]))) * w[:, None]
    bG = (2 * e.amax(-1, keepdim=True) + 16 * U) * p * w.abs()[:, None] + 16 * U * G.abs()
    bG = bG + (HALF[dt] + (2.0**-12 if dt == BF16 else 0)) * (G.abs() + bG)
    if dt == BF16:
        bG = bG + 2.0**-40 * w.abs()[:, None]
    bG = bG + 3 * TINY
    da, dh = G @ h, G.T @ a
    ba = bG @ h.abs() + (many * V + 64) * U * (G.abs() @ h.abs())
    bh = bG.T @ a.abs() + (many * N + 64) * U * (G.abs().T @ a.abs())
    return (loss, da, dh), (bl, ba + HALF[dt] * (da.abs() + ba) + 2 * many * V * TINY, bh + HALF[dt] * (dh.abs() + bh) + 2 * many * N * TINY)


def _check(got, want, bounds):
    for n, a, b, c in zip(("loss", "d_act", "d_head"), got, want, bounds):
        err = (a.double() - b).abs()
        assert (err <= c).all(), (n, float((err - c).max()), float((err / c.clamp(min=1e-300)).max()))


def _both_forms(act, head, t, w, ignore=-100):
    one = ops.streamed_cross_entropy(act, head, t, ignore_index=ignore, row_weight=w, want_dact=True, want_dhead=True)
    loss, stats = ops.streamed_cross_entropy_fwd(act, head, t, ignore_index=ignore, want_stats=True)
    forms = [one, (loss, *ops.streamed_cross_entropy_bwd(act, head, t, stats, w, ignore_index=ignore))]
    loss, kept = ops.streamed_cross_entropy_kept_fwd(act, head, t, ignore_index=ignore)
    if kept is not None:
        ops.streamed_cross_entropy_kept_bwd(act, head, t, kept, 3 * w, ignore_index=ignore)  # leaves it as it is
        forms.append((loss, *ops.streamed_cross_entropy_kept_bwd(act, head, t, kept, w, ignore_index=ignore)))
    large = max(act.element_size() * act.shape[0] * head.shape[0], 2 * head.numel() * (act.dtype == BF16)) > 2**31 - 2**23
    assert (kept is None) == large
    return forms


SHAPES = [(1, 8, 1), (1, 64, 7), (2, 16, 129), (33, 72, 1000), (127, 64, 64), (128, 128, 65), (129, 200, 257), (300, 136, 3001),
          (513, 64, 777), (1000, 520, 4099)]


@pytest.mark.parametrize("N, d, V", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("skip", [0.0, 0.4])
def test_loss_and_gradients(device, N, d, V, dtype, skip):
    act, head, t, w = _inputs(device, N, d, V, dtype, N + V, skip, bits=32 if V % 2 else 64)
    want, bounds = _expected(act, head, t, w)
    for got in _both_forms(act, head, t, w):
        assert got[1].dtype == got[2].dtype == dtype and got[0].dtype == F32
        _check(got, want, bounds)


@pytest.mark.parametrize("d", [1, 33, 100, 1000])
def test_odd_widths_through_autograd(device, d):
    for dtype in (BF16, F32):
        act, head, t, w = _inputs(device, 70, d, 333, dtype, d, 0.2)
        act, head = act.requires_grad_(), head.requires_grad_()
        loss = losses.streamed_position_cross_entropy(act.view(7, 10, d), head, t.view(7, 10))
        assert loss.shape == (7, 10)
        got = (loss.view(-1), *torch.autograd.grad(loss, (act, head), w.view(7, 10), retain_graph=True))
        want = _expected(act.detach(), head.detach(), t, w)
        _check(got, *want)
        for a, b in zip(got[1:], torch.autograd.grad(loss, (act, head), w.view(7, 10))):
            assert torch.equal(a, b)
        loss = losses.streamed_position_cross_entropy(act, head, t, keep=False)
        _check((loss, *torch.autograd.grad(loss, (act, head), w)), *want)


def test_mean_and_one_gradient_alone(device):
    act, head, t, _ = _inputs(device, 200, 64, 500, F32, 3, 0.3)
    on = (t >= 0) & (t < 500)
    want, bounds = _expected(act, head, t, on.float() / on.sum())
    a = act.clone().requires_grad_()
    loss = losses.streamed_cross_entropy(a, head, t)
    assert abs(float(loss) - float(want[0].sum() / on.sum())) <= float(bounds[0].mean()) * 200 / int(on.sum()) + 200 * U * float(loss)
    (da,) = torch.autograd.grad(loss, a)
    # the weight 1 / count is rounded
    assert ((da.double() - want[1]).abs() <= bounds[1] + 4 * U * want[1].abs()).all()
    h = head.clone().requires_grad_()
    (dh,) = torch.autograd.grad(losses.streamed_cross_entropy(act, h, t), h)
    assert ((dh.double() - want[2]).abs() <= bounds[2] + 4 * U * want[2].abs()).all()
    assert float(losses.streamed_cross_entropy(act, head, torch.full_like(t, -100))) == 0.0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_positions_that_do_not_count_reach_nothing(device, dtype):
    act, head, t, w = _inputs(device, 300, 64, 400, dtype, 4, 0.3)
    w[5::9] = 0  # counts in the loss, has no gradient
    skip = (t < 0) | (t >= 400)
    clean = _both_forms(act, head, t, w)
    act[skip] = float("nan")
    got = _both_forms(act, head, t, w)
    for a, b in zip(clean, got):
        assert (b[0][skip] == 0).all() and (b[1][skip] == 0).all()
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    zero = (w == 0) & ~skip
    act[zero] = float("inf")
    for a, b in zip(clean, _both_forms(act, head, t, w)):
        assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2]) and (b[1][zero] == 0).all()
        assert not torch.isfinite(b[0][zero]).any() and torch.equal(a[0][~zero], b[0][~zero])


def test_a_nan_that_counts_shows(device):
    for dtype in (BF16, F32):
        act, head, t, w = _inputs(device, 140, 64, 300, dtype, 5)
        w = w.abs() + 0.1
        clean = _both_forms(act, head, t, w)
        act[17, 3] = float("nan")
        for a, b in zip(clean, _both_forms(act, head, t, w)):
            bad = torch.zeros(140, dtype=torch.bool, device=device)
            bad[17] = True
            assert torch.equal(torch.isnan(b[0]), bad) and torch.isnan(b[1][17]).all()
            assert torch.equal(a[0][~bad], b[0][~bad]) and torch.equal(a[1][~bad], b[1][~bad])
            assert torch.isnan(b[2]).all()


def test_none_counts(device):
    for dtype, N in ((BF16, 3), (BF16, 500), (F32, 5)):
        act, head, t, w = _inputs(device, N, 32, 100, dtype, 6)
        for loss, da, dh in _both_forms(act, head, torch.full_like(t, 7), w, ignore=7):
            assert not loss.any() and not da.any() and not dh.any()
        loss, da, dh = ops.streamed_cross_entropy(act[:0], head, t[:0], want_dact=True, want_dhead=True)
        assert loss.numel() == 0 and da.shape == (0, 32) and not dh.any()
        a = act[:0].clone().requires_grad_()
        h = head.clone().requires_grad_()
        da, dh = torch.autograd.grad(losses.streamed_position_cross_entropy(a, h, t[:0]).sum(), (a, h))
        assert da.shape == (0, 32) and not dh.any()


@pytest.mark.parametrize("scale", [1e-3, 10.0, 60.0])
def test_small_and_large_logits(device, scale):
    """From logits that are all but equal to rows of one probability: what is 1 less a probability keeps its digits."""
    for dtype in (BF16, F32):
        act, head, t, w = _inputs(device, 260, 64, 600, dtype, 7, 0.0, scale)
        t[::2] = (act[::2].double() @ head.double().T).argmax(-1)
        want, bounds = _expected(act, head, t, w)
        for got in _both_forms(act, head, t, w):
            _check(got, want, bounds)


def test_pieces_of_the_vocabulary_and_chunks_of_positions(device):
    """More than 1 GiB of G in the backward, and more than 2 GiB of softmax in the one-call form."""
    act, head, t, w = _inputs(device, 8200, 16, 140000, BF16, 8, 0.02)
    one, two = _both_forms(act, head, t, w)
    want, bounds = None, None
    dh, bh = torch.zeros(140000, 16, dtype=F64, device=device), torch.zeros(140000, 16, dtype=F64, device=device)
    for r in range(0, 8200, 820):
        s = slice(r, r + 820)
        want, bounds = _expected(act[s], head, t[s], w[s])
        for got in (one, two):
            _check((got[0][s], got[1][s]), want[:2], bounds[:2])
        # the rest of the sum's roundings is that of 8200 terms in place of 820
        dh += want[2]
        bh += bounds[2] * 11
    for got in (one, two):
        _check((got[0][:0], got[1][:0], got[2]), (dh[:0, 0], dh[:0], dh), (bh[:0, 0], bh[:0], bh))


def test_a_head_of_more_than_2_gib(device):
    act, head, t, w = _inputs(device, 5, 4096, 263000, BF16, 13)
    t[3] = 262999
    got = _both_forms(act, head, t, w)
    z = torch.cat([act.double() @ head[c:c + 65536].double().T for c in range(0, 263000, 65536)], -1)
    e = 4097 * U * torch.cat([act.double().abs() @ head[c:c + 65536].double().abs().T for c in range(0, 263000, 65536)], -1).amax(-1)
    loss = torch.logsumexp(z, -1) - z.gather(1, t[:, None])[:, 0]
    G = torch.softmax(z, -1).scatter_add(1, t[:, None], -torch.ones(5, 1, dtype=F64, device=device)) * w.double()[:, None]
    bG = (2 * e[:, None] + 16 * U + 2.0**-8 + 2.0**-12) * 2 * G.abs() + 2.0**-40 * w.abs()[:, None]
    da, ba = torch.zeros(5, 4096, dtype=F64, device=device), torch.zeros(5, 4096, dtype=F64, device=device)
    for c in range(0, 263000, 65536):
        h = head[c:c + 65536].double()
        da += G[:, c:c + 65536] @ h
        ba += (bG + 264000 * U * G.abs())[:, c:c + 65536] @ h.abs()
        dh, bh = G[:, c:c + 65536].T @ act.double(), (bG + 70 * U * G.abs())[:, c:c + 65536].T @ act.double().abs()
        for g in got:
            assert ((g[2][c:c + 65536].double() - dh).abs() <= bh + 2.0**-8 * (dh.abs() + bh) + 1e-36).all()
    for g in got:
        assert ((g[0].double() - loss).abs() <= 2 * e + 16 * U * (1 + loss.abs() + 20)).all()
        assert ((g[1].double() - da).abs() <= ba + 2.0**-8 * (da.abs() + ba)).all()


def test_unaligned_views(device):
    act, head, t, w = _inputs(device, 20, 64, 300, BF16, 14)
    flat = torch.empty(20 * 64 + 3, dtype=BF16, device=device)
    flat[3:] = act.view(-1)
    a = losses.streamed_position_cross_entropy(act, head, t)
    assert torch.equal(a, losses.streamed_position_cross_entropy(flat[3:].view(20, 64), head, t))
    with pytest.raises(L.PDError, match="aligned"):
        ops.streamed_cross_entropy_fwd(flat[3:].view(20, 64), head, t)


def test_pieces_of_fp32(device):
    """More than 1 GiB of G in the backward."""
    act, head, t, w = _inputs(device, 4000, 24, 80000, F32, 12, 0.1)
    want, bounds = _expected(act, head, t, w)
    for got in _both_forms(act, head, t, w):
        _check(got, want, bounds)


def test_twice_the_same_and_on_other_streams(device):
    act, head, t, w = _inputs(device, 400, 128, 1500, BF16, 9, 0.1)
    first = _both_forms(act, head, t, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _both_forms(act, head, t, w)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_gradients_are_the_losses_differences(device):
    """Directional differences of the loss in fp32, where the loss is off by about 1e-6."""
    act, head, t, w = _inputs(device, 50, 24, 90, F32, 10, 0.2)
    w = w.abs()
    _, da, dh = ops.streamed_cross_entropy(act, head, t, row_weight=w, want_dact=True, want_dhead=True)
    g = torch.Generator(device=device).manual_seed(1)
    for x, d in ((act, da), (head, dh)):
        v = torch.randn(x.shape, device=device, generator=g)
        h = 1e-3
        f = lambda s: float((ops.streamed_cross_entropy(*((x + s * v, head) if x is act else (act, x + s * v)), t)[0].double()  # noqa: E731
                             * w.double()).sum())
        diff, want = (f(h) - f(-h)) / (2 * h), float((d.double() * v.double()).sum())
        dz = v.double() @ head.double().T if x is act else act.double() @ v.double().T
        # h^2 / 6 times a third derivative (a third central moment of dz), and the losses' own bounds and the
        # moved operand's rounding over h
        third = h * h / 6 * float((w.double() * (2 * dz.abs().amax(-1))**3).sum())
        noise = float((w.double() * (_expected(act, head, t, w)[1][0] + 2 * U * (act.double().abs() @ head.double().abs().T).amax(-1))).sum())
        assert abs(diff - want) <= third + noise / h + 1e-4 * abs(want)


def test_refusals(device):
    act, head, t, w = _inputs(device, 4, 16, 9, BF16)
    for bad in ((act.cpu(), head, t), (act, head.cpu(), t), (act, head, t.cpu()), (act.t(), head, t)):
        with pytest.raises(L.PDError):
            ops.streamed_cross_entropy_fwd(*bad)
    with pytest.raises(L.PDError, match="row_weight"):
        ops.streamed_cross_entropy(act, head, t, row_weight=w.double(), want_dact=True)
    kept = ops.streamed_cross_entropy_kept_fwd(act, head, t)[1]
    for bad in (kept[1:], kept.float(), kept.cpu()):
        with pytest.raises(L.PDError, match="kept"):
            ops.streamed_cross_entropy_kept_bwd(act, head, t, bad, w)
    with pytest.raises(L.PDError, match="g is"):
        ops.streamed_cross_entropy_kept_bwd(act, head, t, kept, w[:3])
    with pytest.raises(L.PDError, match="stats"):
        ops.streamed_cross_entropy_bwd(act, head, t, w, w)


def _sure(device, V, dtype, N=64):
    """Logits that bf16 holds: position i's are row i of head^T. 1 - p of the target from 0.5 to 10^-13, the target at
    any place, entries of its tile and of others in the rest, two of them as large as the target in the last rows."""
    g = torch.Generator(device=device).manual_seed(V)
    z = (torch.randint(-16, 9, (N, V), device=device, generator=g) / 8.0)
    t = torch.randperm(V, device=device, generator=g)[:N]
    z[torch.arange(N, device=device), t] = torch.arange(N, device=device) / 2.0
    # all of the rest in a single entry of the target's 64
    few, col, other = torch.arange(N, device=device) % 4 == 3, torch.arange(V, device=device), torch.where((t ^ 1) < V, t ^ 1, t - 1)
    z = torch.where(few[:, None] & (col != other[:, None]) & (col != t[:, None]), torch.full_like(z, -60.0), z)
    z[-3, (t[-3] + 7) % V] = z[-3, t[-3]]
    z[-2, (t[-2] + V // 2) % V] = z[-2, t[-2]]
    return torch.eye(N, device=device).to(dtype), z.t().contiguous().to(dtype), t, z.double()


@pytest.mark.parametrize("V", [65, 129, 640, 5000, 20000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_is_one_less_a_probability(device, V, dtype):
    """The loss and the target's gradient relative to 1 - p. Logits are exact, e^x is off by |x| 2^-24 and a few roundings
    of itself, sums by 2^-24 for each of their additions (a wave's 64 columns, then tiles); bf16 gradients by two
    roundings more, d_head has one term."""
    act, head, t, z = _sure(device, V, dtype)
    N = 64
    at = torch.arange(N, device=device)
    w = torch.linspace(-2, 2, N, device=device)
    w = torch.where(w == 0, torch.ones_like(w), w)
    rest = torch.where(torch.arange(V, device=device) == t[:, None], torch.zeros_like(z),
                       (z - z[at, t][:, None]).exp()).sum(-1)  # (1 - p) / p
    loss, miss = torch.log1p(rest), rest / (1 + rest)
    rel = (2 * (z.amax(-1) - z.amin(-1).clamp(min=-3)) + 128 + V / 64) * U
    for got in _both_forms(act, head, t, w):
        _check_sure(got[0], got[2], t, at, w, loss, miss, rel, dtype)


def _check_sure(got, dh, t, at, w, loss, miss, rel, dtype):
    assert ((got.double() - loss).abs() <= rel * loss + 2**-126).all(), float(((got.double() - loss).abs() / loss).max())
    d = dh.double()[t, at]  # positions are columns of the identity: G at the target
    bound = (rel + (2 * HALF[dtype] if dtype == BF16 else 0)) * miss * w.double().abs()
    assert ((d + miss * w.double()).abs() <= bound + 2**-126).all(), float(((d / -w.double() - miss).abs() / miss).max())


@pytest.mark.parametrize("dtype, N, V", [(BF16, 8200, 140000), (BF16, 2100, 300000), (F32, 4000, 80000)])
def test_what_is_one_less_a_probability_in_pieces(device, dtype, N, V):
    """The same where the backward forms the logits in pieces of the vocabulary, which may take other tiles: the positions of
    the identity among others that have no gradient."""
    few, head, t, z = _sure(device, V, dtype)
    g = torch.Generator(device=device).manual_seed(N)
    at, rows = torch.arange(64, device=device), torch.randperm(N, device=device, generator=g)[:64]
    act = torch.randn(N, 64, device=device, generator=g).to(dtype)
    targets = torch.randint(V, (N,), device=device, generator=g)
    w = torch.zeros(N, device=device)
    act[rows], targets[rows], w[rows] = few, t, torch.linspace(1, 2, 64, device=device)
    rest = torch.where(torch.arange(V, device=device) == t[:, None], torch.zeros_like(z), (z - z[at, t][:, None]).exp()).sum(-1)
    rel = (2 * (z.amax(-1) - z.amin(-1).clamp(min=-3)) + 128 + V / 64) * U
    for got in _both_forms(act, head, targets, w):
        _check_sure(got[0][rows], got[2], t, at, w[rows], torch.log1p(rest), rest / (1 + rest), rel, dtype)


@pytest.mark.parametrize("N, V", [(3, 200), (200, 3000)])
def test_logits_that_leave_fp32_downwards_are_no_part_of_the_sum(device, N, V):
    """Whole tiles of entries whose logits are -1e40: their probability is 0, in the loss and in both gradients."""
    act, head, t, w = _inputs(device, N, 64, V, BF16, V)
    act[:, 0], head[:, 0] = 1e20, 0
    head[60:195, 0] = -1e20
    t[:] = torch.where((t >= 60) & (t < 195), torch.full_like(t, 7), t)
    # as without those entries
    rest = torch.cat([head[:60], head[195:]])
    want, bounds = _expected(act, rest, torch.where(t >= 195, t - 135, t), w)
    for loss, da, dh in _both_forms(act, head, t, w):
        assert not dh[60:195].any()
        _check((loss, da, torch.cat([dh[:60], dh[195:]])), want, bounds)


def test_a_row_of_nothing_but_such_logits_is_nan(device):
    act, head, t, w = _inputs(device, 9, 64, 300, BF16, 3)
    act[4], head[:, 0] = 0, -1e20
    act[:, 0] = 0
    act[4, 0] = 1e20
    for got in _both_forms(act, head, t, w):
        bad = torch.arange(9, device=device) == 4
        assert torch.equal(torch.isnan(got[0]), bad) and torch.isnan(got[1][4]).all() and torch.isfinite(got[1][~bad]).all()


@pytest.mark.parametrize("N, d, V", [(1024, 256, 20000), (1500, 1032, 20011), (3000, 264, 40000), (900, 2048, 12000)])
def test_wide_activations_in_slices(device, N, d, V):
    """Sums of d_act's slices of the vocabulary, in tiles of either size, whole and with an edge on every side."""
    act, head, t, w = _inputs(device, N, d, V, BF16, N, 0.2)
    want, bounds = _expected(act, head, t, w)
    for got in _both_forms(act, head, t, w):
        _check(got, want, bounds)


def test_chunks_of_fp32_positions(device):
    """More than 2 GiB of logits in the one-call form: the second chunk's d_head is added to the first's."""
    act, head, t, w = _inputs(device, 7000, 24, 80000, F32, 15, 0.05)
    want, bounds = _expected(act, head, t, w)
    for got in _both_forms(act, head, t, w):
        _check(got, want, bounds)
