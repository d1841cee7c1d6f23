"""Gradients of packed attention where a row's scores are far from zero, and its forward where
they lie around a large offset.

The scores are sums of products that 32 bits hold exactly, as in the tests of the forward, so
what is left are the weights' rounding and 32-bit sums. Bounds, u half a step of the type, e =
2^-24, n a sequence's rows, r query heads a key head: a weight is off by g = (n + 128) e (its
exponent and log of the sum at most 64 where it counts, and the row's sum) and by u as an
operand, and with P, dP, D, dS of the definition
  D:  |do| . (error of out) + (D + 2) e |do| . |out|
  ds: (u + 2 g) |ds| + P ((D + 2) e |do| |v|^T + error of D) + n r e |ds| for the sums
  dq: scale (that) |k| + u |dq|;  dk: scale (that)^T |q| + u |dk|
  dv: (u + 2 g + (n r + 32) e) P^T |do| + u |dv|"""

import math

import pytest
import torch

from param_decomp_amd.attention import packed_attention

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E = 2.0**-24


def _definition(q, k, v, g, lengths, scale):
    """Values and bounds of out, dq, dk, dv in 64 bits."""
    N, H, D = q.shape
    KV = k.shape[1]
    r = H // KV
    u = torch.finfo(q.dtype).eps / 2
    val = [torch.zeros(t.shape, dtype=F64, device=q.device) for t in (q, q, k, v)]
    tol = [torch.zeros_like(t) for t in val]
    heads = lambda t: t.double().transpose(0, 1).contiguous()  # noqa: E731
    T = lambda t: t.transpose(1, 2).contiguous()  # noqa: E731
    a = 0
    for n in lengths:
        at, a = slice(a, a + n), a + n
        Q, K, V, G = (heads(t[at]) for t in (q, k, v, g))
        K, V = K.repeat_interleave(r, 0), V.repeat_interleave(r, 0)
        S = (Q @ T(K)) * scale
        S.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1), -math.inf)
        P = torch.softmax(S, -1)
        O = P @ V
        w = u + 2 * (n + 128) * E
        eo = 1.05 * (w * (P @ V.abs()) + u * O.abs())
        dP = G @ T(V)
        Di = (G * O).sum(-1, keepdim=True)
        dS = P * (dP - Di)
        eD = (G.abs() * eo).sum(-1, keepdim=True) + (D + 2) * E * (G.abs() * O.abs()).sum(-1, keepdim=True)
        eS = (w + (n * r + 32) * E) * dS.abs() + P * ((D + 2) * E * (G.abs() @ T(V.abs())) + eD)
        eV = (w + (n * r + 32) * E) * (T(P) @ G.abs())
        dQ, dK, dV = dS @ K * scale, T(dS) @ Q * scale, T(P) @ G
        rows = lambda t, m: t.view(m, -1, n, D).sum(1).transpose(0, 1)  # noqa: E731
        s = abs(scale)
        for i, (x, e, m) in enumerate(((O, eo, H), (dQ, 1.05 * (eS @ K.abs() * s + u * dQ.abs()), H),
                                       (dK, 1.05 * (T(eS) @ Q.abs() * s + u * dK.abs()), KV),
                                       (dV, 1.05 * (eV + u * dV.abs()), KV))):
            val[i][at], tol[i][at] = rows(x, m), rows(e, m)
    return val, [t + 1e-30 for t in tol]


def _check(q, k, v, g, lengths, scale):
    off = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=q.device)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, off, scale=scale)
    got = (out.detach(), *torch.autograd.grad(out, leaves, g))
    val, tol = _definition(q, k, v, g, lengths, q.shape[2]**-0.5 if scale is None else scale)
    for x, y, t, name in zip(got, val, tol, ("out", "dq", "dk", "dv")):
        assert torch.isfinite(x.float()).all(), name
        assert (t >= 1e-30).all(), name  # a bound that nothing fails is none
        worst = ((x.double() - y).abs() / t).max().item()
        assert worst <= 1.0, f"{name}: {worst:.3g} of the bound"
    return got, val, tol


GRIDS = [(70, 2, 1, 64, [1, 33, 1, 35]), (140, 3, 1, 128, [139, 1]), (2100, 32, 4, 64, [1, 130, 2, 700, 1267]),
         (2100, 36, 4, 96, [5, 1, 900, 1194]), (2100, 32, 8, 128, [1, 64, 2035])]


def _rows(device, N, H, KV, D, dtype, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda h: torch.randn(N, h, D, device=device, generator=g).to(dtype)  # noqa: E731
    zero = lambda h: torch.zeros(N, h, D, device=device, dtype=dtype)  # noqa: E731
    return zero(H), zero(KV), rnd(KV), rnd(H), g


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("size", [20, 40, 99, 110])
@pytest.mark.parametrize("N, H, KV, D, lengths", GRIDS)
def test_keys_far_apart_and_equal(device, dtype, sign, size, N, H, KV, D, lengths):
    """Scores sign 2^size (1 + t / 8): a row's weight is shared by its equal keys."""
    for steps in (0, 7):
        for scale in (None, -0.25, 1.0):
            q, k, v, g, gen = _rows(device, N, H, KV, D, dtype, seed=size + steps)
            half = size // 2
            q[:, :, D - 3] = 2.0**half
            t = torch.randint(0, steps + 1, (N, KV), device=device, generator=gen).float()
            k[:, :, D - 3] = (sign * 2.0**(size - half) * (1 + t / 8)).to(dtype)
            _check(q, k, v, g, lengths, scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("size", [12, 18, 22])
@pytest.mark.parametrize("N, H, KV, D, lengths", GRIDS)
def test_scores_around_an_offset(device, dtype, sign, size, N, H, KV, D, lengths):
    """Scores sign 2^size + t, t whole and up to 64: the offset changes nothing."""
    q, k, v, g, gen = _rows(device, N, H, KV, D, dtype, seed=size)
    half = size // 2
    q[:, :, 0], q[:, :, 1] = 2.0**half, 1.0
    k[:, :, 0] = sign * 2.0**(size - half)
    k[:, :, 1] = torch.randint(-64, 65, (N, KV), device=device, generator=gen).to(dtype)
    for scale in (0.125, -0.125):
        got, val, tol = _check(q, k, v, g, lengths, scale)
        k0 = k.clone()
        k0[:, :, 0] = 0.0
        near = _check(q, k0, v, g, lengths, scale)
        for i in (0, 3):  # (dq and dk hold the offset's channel)
            assert ((got[i].double() - near[0][i].double()).abs() <= tol[i] + near[2][i]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H, KV, N", [(2, 2, 60), (32, 32, 2100)])
@pytest.mark.parametrize("scale", [0.125, -0.2])
def test_one_key_rows_give_their_cotangent(device, dtype, H, KV, N, scale):
    """Sequences of one row with ordinary channels and scores of any size: out = v, dv = do and
    no other gradient (the products round, but there is nothing to compare a score with)."""
    gen = torch.Generator(device=device).manual_seed(5)
    q, k, v, g = (torch.randn(N, H, 64, device=device, generator=gen).to(dtype) for _ in range(4))
    sizes = torch.logspace(0, 18, N, device=device)[:, None, None]
    q, k = (q * sizes).to(dtype), (k * sizes).to(dtype)
    off = torch.arange(N + 1, dtype=torch.int32, device=device)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, off, scale=scale)
    dq, dk, dv = torch.autograd.grad(out, leaves, g)
    u = torch.finfo(dtype).eps / 2
    # weight, operand and result: two roundings of the type and the weight's own in 32 bits
    near = lambda x, y: ((x.double() - y.double()).abs() <= (2.1 * u + 64 * E) * y.double().abs()).all()  # noqa: E731
    assert near(out, v) and near(dv, g)
    # ds = p (do . v - do . out), each with the error of out, of a product sum and of p
    size = (g.double().abs() * v.double().abs()).sum(-1, keepdim=True) * (2.1 * u + 200 * E) * abs(scale)
    assert (dq.double().abs() <= 1.05 * size * k.double().abs() + 1e-30).all()
    assert (dk.double().abs() <= 1.05 * size * q.double().abs() + 1e-30).all()
