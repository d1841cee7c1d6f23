"""Packed attention on inputs that hold NaN or infinities: a result is not finite where its
definition is not, and nowhere else, whether the tile's result was kept or formed again.

With b(x) the entries of x that are not finite, per sequence (j keys, i queries that see them):
  row i has no weights, w_i: b(q_i) or b(k_j) for a j <= i (NaN here)
  out_ic: w_i or b(v_jc) for a j <= i;  D_i: b(out_i) or b(do_i);  dq_i: w_i or D_i
  dk_j: w_i or D_i for an i >= j, over the heads that share the key head;  dv_jc: w_i or b(do_ic)
Everywhere else the values are those of the definition with zeros in place of what is not
finite, in the bounds of the gradients' tests."""

import math

import pytest
import torch
from test_gpu_attention_score_gradients import _definition

from param_decomp_amd.attention import packed_attention

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _expected(q, k, v, g, lengths):
    r = q.shape[1] // k.shape[1]
    b = lambda t: ~torch.isfinite(t.float())  # noqa: E731
    bq, bk, bv, bg = (b(t) for t in (q, k, v, g))
    bk, bv = bk.repeat_interleave(r, 1), bv.repeat_interleave(r, 1)
    out, dq, dk, dv = (torch.zeros_like(bq) for _ in range(4))
    a = 0
    since = lambda t: t.cumsum(0) > 0  # noqa: E731
    until = lambda t: t.flip(0).cumsum(0).flip(0) > 0  # noqa: E731
    for n in lengths:
        at, a = slice(a, a + n), a + n
        w = (bq[at].any(-1) | since(bk[at].any(-1)))[..., None]
        out[at] = w | since(bv[at])
        d = (out[at] | bg[at]).any(-1, keepdim=True)
        dq[at] = w | d
        dk[at] = until(w | d)
        dv[at] = until(w | bg[at])
    heads = lambda t: t.view(t.shape[0], -1, r, t.shape[2]).any(2)  # noqa: E731
    return out, dq, heads(dk), heads(dv)


GRIDS = [(71, 4, 2, 64, [1, 33, 2, 35]), (140, 3, 1, 128, [139, 1]), (2100, 32, 32, 64, [517, 790, 3, 790]),
         (2100, 32, 8, 128, [1, 64, 2035]), (2100, 36, 4, 96, [5, 1, 900, 1194])]


def _poisons(N, H, KV, D, lengths):
    """name -> what it puts where, in the sequence that holds the middle of the rows."""
    a = 0
    for n in lengths:
        if a + n > N // 2:
            break
        a += n
    early, late = a + min(2, n - 1), a + n // 2

    def all_of(q, k, v, g, x):
        for t in (q, k, v, g):
            t.fill_(x)

    def keys(q, k, v, g, x):
        k[early, 0, D // 2] = math.nan

    def channel(q, k, v, g, x):
        v[early, :, 3] = x
        v[late, 0, D - 1] = x

    def values(q, k, v, g, x):
        v[a:a + n] = x

    def queries(q, k, v, g, x):
        q[late, H - 1, 0] = math.nan
        q[a + n - 1, 0] = math.nan

    def cotangents(q, k, v, g, x):
        g[late, 0, 5], g[early, H - 1, D - 1] = x, x

    def one_channel_of_all(q, k, v, g, x):
        g[:, :, 1] = x

    def mixed(q, k, v, g, x):
        v[early, 0, 0], g[late, 1, 2] = x, x
        q[max(a - 1, 0)] = math.nan
        k[min(a + n, N - 1)], v[min(a + n, N - 1)] = math.nan, x

    return [all_of, keys, channel, values, queries, cotangents, one_channel_of_all, mixed]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("x", [math.nan, math.inf])
@pytest.mark.parametrize("which", range(8))
@pytest.mark.parametrize("N, H, KV, D, lengths", GRIDS)
def test_not_finite_where_the_definition_is_not(device, dtype, x, which, N, H, KV, D, lengths):
    gen = torch.Generator(device=device).manual_seed(N + which)
    t = [torch.randn(N, h, D, device=device, generator=gen).to(dtype) for h in (H, KV, KV, H)]
    poison = _poisons(N, H, KV, D, lengths)[which]
    if poison.__name__ == "all_of" and x == math.inf:
        x = -math.inf
    poison(*t, x)
    off = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=device)
    leaves = [s.detach().clone().requires_grad_() for s in t[:3]]
    out = packed_attention(*leaves, off)
    got = (out.detach(), *torch.autograd.grad(out, leaves, t[3]))
    val, tol = _definition(*(torch.where(torch.isfinite(s.float()), s, torch.zeros_like(s)) for s in t), lengths, D**-0.5)
    for y, b, z, e, name in zip(got, _expected(*t, lengths), val, tol, ("out", "dq", "dk", "dv")):
        assert not torch.isfinite(y.float())[b].any(), name
        assert ((y.double() - z).abs() <= e)[~b].all(), name
    again = torch.autograd.grad(packed_attention(*leaves, off), leaves, t[3])
    for y, z in zip(got[1:], again):
        assert torch.equal(y.nan_to_num(1.25), z.nan_to_num(1.25))


def test_a_batch_without_numbers_takes_about_the_usual_time(device):
    """Where every row is NaN by its own inputs none is formed again: with each of them again
    the call took 40 times as long (2048 tokens, 12 heads); six times is the limit here."""
    N, H, D = 2048, 12, 64
    off = torch.tensor([0, N], dtype=torch.int32, device=device)

    def least(t):
        leaves, times = [s.requires_grad_() for s in t[:3]], []
        for _ in range(6):
            ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            ev[0].record()
            torch.autograd.grad(packed_attention(*leaves, off), leaves, t[3])
            ev[1].record()
            torch.cuda.synchronize()
            times.append(ev[0].elapsed_time(ev[1]))
        return min(times)

    usual = least([torch.randn(N, H, D, device=device).to(BF16) for _ in range(4)])
    for which in ((0, 1, 2, 3), (1,), (2,), (3,)):
        t = [torch.randn(N, H, D, device=device).to(BF16) for _ in range(4)]
        for i in which:
            t[i].fill_(math.nan)
        assert least(t) <= 6 * usual, which
