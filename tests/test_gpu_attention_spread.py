"""Packed attention in limits that a missing or turned gradient fails at every size and scale.

The elementwise bounds of `test_gpu_attention` add up worst cases: for key gradients over
thousands of queries and several heads they pass the gradient itself, and they hold for
positive scales alone. Here a result's distance from the definition, in the root of its summed
squares, is at most twice the root of the summed squares of what the single roundings do to it;
they are independent of each other. With u half a step of the type and P, dP, D, dS of the
definition:
  out: u^2 (P^2 V^2 + out^2);  D of the unrounded out: do^2 (u^2 P^2 V^2);  ds: u^2 ds^2 + P^2 that
  dq: scale^2 (ds's) k^2 + u^2 dq^2;  dk: scale^2 (ds's)^T q^2 + u^2 dk^2
  dv: u^2 ((P^2)^T do^2 + dv^2)
For fp32 tensors u is that of its products' and sums' rounding, (D + n) 2^-24."""

import math

import pytest
import torch
from test_gpu_attention import _grads, _inputs, _offsets

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
NAMES = ("out", "dq", "dk", "dv")


def _definition(q, k, v, g, lengths, scale):
    """(values, limits of the distances' norms) of out, dq, dk, dv in 64 bits."""
    H, D, r = q.shape[1], q.shape[2], q.shape[1] // k.shape[1]
    val = [torch.zeros(t.shape, dtype=F64, device=q.device) for t in (q, q, k, v)]
    squares = [torch.zeros((), dtype=F64, device=q.device) for _ in val]
    heads = lambda t: t.double().transpose(0, 1).contiguous()  # noqa: E731
    T = lambda t: t.transpose(1, 2).contiguous()  # noqa: E731
    a = 0
    for n in lengths:
        u = 2.0**-8 if q.dtype == BF16 else (D + n) * 2.0**-24
        at, a = slice(a, a + n), a + n
        Q, K, V, G = (heads(t[at]) for t in (q, k, v, g))
        K, V = K.repeat_interleave(r, 0), V.repeat_interleave(r, 0)
        S = (Q @ T(K)) * scale
        S.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1), -math.inf)
        P = torch.softmax(S, -1)
        O, dP = P @ V, G @ T(V)
        dS = P * (dP - (G * O).sum(-1, keepdim=True))
        dQ, dK, dV = dS @ K * scale, T(dS) @ Q * scale, T(P) @ G
        o2 = u**2 * (P**2 @ V**2)
        s2 = u**2 * dS**2 + P**2 * (G**2 * o2).sum(-1, keepdim=True)
        rows = lambda t, m: t.view(m, -1, n, D).sum(1).transpose(0, 1)  # noqa: E731
        for i, (x, e, m) in enumerate(((O, o2, H), (dQ, scale**2 * (s2 @ K**2), H),
                                       (dK, scale**2 * (T(s2) @ Q**2), H // r), (dV, u**2 * (T(P**2) @ G**2), H // r))):
            val[i][at] = rows(x, m)
            squares[i] += e.sum() + u**2 * val[i][at].square().sum()
    return val, [2 * s.sqrt() for s in squares]


def _outside(got, val, limit):
    return [n for n, x, y, e in zip(NAMES, got, val, limit) if not (x.double() - y).norm() <= e]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.3, -0.3])
@pytest.mark.parametrize("N, H, KV, D, lengths", [(100, 2, 1, 64, [60, 40]), (700, 8, 1, 128, [1, 699])])
def test_limits_tell_results_apart(dtype, scale, N, H, KV, D, lengths):
    """On the CPU: the definition is within its limits, with the other scale's sign nothing
    is, and neither are gradients of zero, turned, or of one key head's query heads but one."""
    q, k, v, g = _inputs("cpu", N, H, KV, D, dtype, seed=3)
    val, limit = _definition(q, k, v, g, lengths, scale)
    for y, e in zip(val, limit):
        assert 0 < e <= 0.05 * y.norm()
    assert not _outside(val, val, limit)
    assert _outside(_definition(q, k, v, g, lengths, -scale)[0], val, limit) == list(NAMES)
    assert _outside([val[0], *(0 * t for t in val[1:])], val, limit) == ["dq", "dk", "dv"]
    assert _outside([val[0], *(-t for t in val[1:])], val, limit) == ["dq", "dk", "dv"]
    g[:, 0] = 0
    less, _ = _definition(q, k, v, g, lengths, scale)
    assert _outside([val[0], *less[1:]], val, limit) == ["dq", "dk", "dv"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.3, -0.05, -0.3])
@pytest.mark.parametrize("N, H, KV, D, lengths", [
    (100, 2, 1, 64, [60, 40]), (130, 2, 2, 128, [127, 3]), (90, 4, 2, 40, [50, 40]), (2100, 32, 32, 64, [1, 700, 1399]),
    (2100, 32, 4, 128, [64, 2036]), (2100, 36, 4, 96, [5, 1, 900, 1194]), (2600, 4, 2, 64, [1999, 1, 600]),
    (2100, 64, 1, 64, [3, 2097])])
def test_spread(device, dtype, scale, N, H, KV, D, lengths):
    q, k, v, g = _inputs(device, N, H, KV, D, dtype, seed=3)
    got = _grads(q, k, v, g, _offsets(device, lengths), scale=scale)
    val, limit = _definition(q, k, v, g, lengths, scale)
    for y, e in zip(val, limit):
        assert 0 < e <= 0.05 * y.norm()
    assert not _outside(got, val, limit)
    # -q under -scale: the same scores to the bit. (dk sums products with q, and those of -q;
    # the matrix instructions do not round both alike.)
    same = _grads(-q, k, v, g, _offsets(device, lengths), scale=-scale)
    assert torch.equal(got[0], same[0]) and torch.equal(got[3], same[3]) and torch.equal(got[1], -same[1])
