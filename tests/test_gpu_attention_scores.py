"""Packed attention where a row's scores are far from zero: one key, equal keys and keys far
apart, with scores up to the end of fp32's range on both sides.

Every score here is a sum of products that 32 bits hold exactly, so the definition in 64 bits
and the kernels see the same ones, and what is left is the weights' rounding. Bounds, u half
a step of the type, e = 2^-24 and n the row's keys: an exponential, its exponent (at most 64
where its weight counts: 2^-64 of a row is nothing) and a row's sum are off by g = (n + 128)
e, so with weights P
  out: (u + 2 g) P |v| + u |out|: the weights as operands, the sums, and the result."""

import math

import pytest
import torch

from param_decomp_amd import ops
from param_decomp_amd.attention import packed_attention

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E = 2.0**-24


def _weights(q, k, scale):
    """[H, n, n] weights of one sequence in 64 bits (q [n, H, D], k [n, KV, D])."""
    n, H = q.shape[:2]
    Q, K = q.double().transpose(0, 1), k.double().transpose(0, 1).repeat_interleave(H // k.shape[1], 0)
    s = (Q @ K.transpose(1, 2).contiguous()) * scale
    s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1), -math.inf)
    return torch.softmax(s, -1)


def _check_out(out, q, k, v, lengths, scale):
    u, a = torch.finfo(q.dtype).eps / 2, 0
    H, rep = q.shape[1], q.shape[1] // k.shape[1]
    assert torch.isfinite(out.float()).all()
    for n in lengths:
        at, a = slice(a, a + n), a + n
        P = _weights(q[at], k[at], scale)
        V = v[at].double().transpose(0, 1).repeat_interleave(rep, 0)
        want = P @ V
        bound = 1.05 * ((u + 2 * (n + 128) * E) * (P @ V.abs()) + u * want.abs()) + 1e-30
        off = (out[at].double().transpose(0, 1) - want).abs() / bound
        assert off.max() <= 1.0, (n, float(off.max()))


def _far(device, N, H, KV, D, dtype, size, sign, steps, seed):
    """q, k, v whose scores are sign 2^size times 1, 1 + 1/8, .. 1 + steps / 8, a key's at
    random: keys far apart, many of them equal."""
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g).to(dtype)  # noqa: E731
    q, k = torch.zeros(N, H, D, device=device, dtype=dtype), torch.zeros(N, KV, D, device=device, dtype=dtype)
    half = size // 2
    q[:, :, D - 3] = 2.0**half
    t = torch.randint(0, steps + 1, (N, KV), device=device, generator=g).float()
    k[:, :, D - 3] = (sign * 2.0**(size - half) * (1 + t / 8)).to(dtype)
    assert torch.equal(k[:, :, D - 3].float(), sign * 2.0**(size - half) * (1 + t / 8))
    return q, k, rnd(N, KV, D)


# (rows, heads, key heads, width, lengths): 32-row and 128-row tiles
GRIDS = [(70, 2, 1, 64, [1, 33, 1, 35]), (140, 3, 1, 128, [139, 1]), (2100, 32, 4, 64, [1, 130, 2, 700, 1267]),
         (2100, 36, 4, 96, [5, 1, 900, 1194])]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("size", [40, 99, 100, 126])  # 2^100 = 1.27e30, 2^126 (1 + 7/8) = 1.6e38
@pytest.mark.parametrize("N, H, KV, D, lengths", GRIDS)
def test_scores_of_any_size(device, dtype, sign, size, N, H, KV, D, lengths):
    off = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=device)
    for steps in (0, 7):  # all keys equal, and far apart
        for scale in (None, -0.25, 1.0):
            q, k, v = _far(device, N, H, KV, D, dtype, size, sign, steps, seed=size + steps)
            out = packed_attention(q, k, v, off, scale=scale)
            _check_out(out, q, k, v, lengths, D**-0.5 if scale is None else scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H, KV", [(2, 2), (32, 32)])
@pytest.mark.parametrize("size", [2.0**63, 2.0**63 * 219 / 128, 2.0**30 * 219 / 128])
def test_low_scores_before_ordinary_ones(device, dtype, H, KV, size):
    """The first rows see keys of scores of large negative size alone; later ones ordinary keys too, in
    the same tile and in later ones; -inf among them has no weight."""
    N, D = 2100, 64
    g = torch.Generator(device=device).manual_seed(3)
    q, k, v = (torch.randn(N, h, D, device=device, generator=g).to(dtype) for h in (H, KV, KV))
    q[:, :, 0] = min(size, 2.0**63)
    q[:, :, 1:] = q[:, :, 1:].round()  # scores that 32 bits hold exactly
    k[:, :, 1:] = k[:, :, 1:].round()
    k[:, :, 0] = 0.0
    starts = [0, 40, 700]
    low = {0: 31, 40: 100, 700: 200}  # as many keys of low scores first
    for a in starts:
        n = low[a]
        k[a:a + n, :, 0] = -size
        k[a:a + n, :, 1:] = 0.0
        k[a + 3, :, 0] = -math.inf
    off = torch.tensor(starts + [N], dtype=torch.int32, device=device)
    out = packed_attention(q, k, v, off)
    kk = k.clone()
    kk[[a + 3 for a in starts], :, 0] = -2.0 * size  # a score of no weight beside the others
    _check_out(out, q, kk, v, [40, 660, 1400], D**-0.5)
    out = packed_attention(q, k, v, off, scale=0.3)
    _check_out(out, q, kk, v, [40, 660, 1400], 0.3)


def test_no_finite_score_is_no_number(device):
    """A row whose only scores are -inf has no softmax; the rows that see another do."""
    q, k, v = (torch.randn(40, 2, 64, device=device).to(F32) for _ in range(3))
    q[:, :, 0] = 1.0
    k[:3, :, 0] = -math.inf
    out = packed_attention(q, k, v, torch.tensor([0, 40], dtype=torch.int32, device=device))
    assert torch.isnan(out[:3]).all() and torch.isfinite(out[3:]).all()
    stats = ops.packed_attention_fwd(q, k, v, torch.tensor([0, 40], dtype=torch.int32, device=device),
                                     want_saved=True)[1][0]
    assert not torch.isfinite(stats[..., :3]).all() and torch.isfinite(stats[..., 3:]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N, H, KV, D, lengths", GRIDS)
def test_values_at_the_end_of_fp32(device, dtype, N, H, KV, D, lengths):
    """A mean of values stays among them, where their sum or a product with a weight past 1
    would be infinite."""
    g = torch.Generator(device=device).manual_seed(9)
    q, k, v = (torch.randn(N, h, D, device=device, generator=g).round().to(dtype) for h in (H, KV, KV))
    v = (v.float().clamp(-1, 1) * 2.0**127).to(dtype)
    off = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=device)
    _check_out(packed_attention(q, k, v, off, scale=0.125), q, k, v, lengths, 0.125)
