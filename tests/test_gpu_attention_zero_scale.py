"""Packed attention under a scale of 0: the mean of the values a row sees, whatever the scores'
size, and no gradient but that of the values. (Sizes and types of the other tests' forms.)"""

import pytest
import torch

from param_decomp_amd.attention import packed_attention

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.0])
@pytest.mark.parametrize("size", [1.0, 2.0**40, 2.0**60])
@pytest.mark.parametrize("N, H, KV, D, lengths", [(70, 2, 1, 64, [1, 33, 36]), (2100, 32, 8, 128, [5, 95, 2000])])
def test_zero_scale(device, dtype, scale, size, N, H, KV, D, lengths):
    gen = torch.Generator(device=device).manual_seed(1)
    q, k, v, g = (torch.randn(N, h, D, device=device, generator=gen).to(dtype) for h in (H, KV, KV, H))
    leaves = [t.requires_grad_() for t in ((q * size).to(dtype), (k * size).to(dtype), v)]
    off = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=device)
    out = packed_attention(*leaves, off, scale=scale)
    dq, dk, dv = torch.autograd.grad(out, leaves, g)
    assert (dq == 0).all() and (dk == 0).all()
    u, a, r = torch.finfo(dtype).eps / 2, 0, H // KV
    for n in lengths:
        at, a = slice(a, a + n), a + n
        count = torch.arange(1, n + 1, device=device, dtype=torch.float64)[:, None, None]
        mean = lambda t: t.double().cumsum(0) / count  # noqa: E731
        later = lambda t: (t / count).flip(0).cumsum(0).flip(0)  # noqa: E731
        for got, want, size_ in ((out[at], mean(v[at]).repeat_interleave(r, 1), mean(v[at].abs()).repeat_interleave(r, 1)),
                                 (dv[at], later(g[at].double()).view(n, KV, r, D).sum(2),
                                  later(g[at].double().abs()).view(n, KV, r, D).sum(2))):
            # weights as operands and their sums in 32 bits, the result's rounding; exponents of
            # 2^-20 at most from the scores' sizes
            bound = 1.05 * (u + 2 * (n * r + 128) * 2.0**-24 + 2.0**-19) * size_ + u * want.abs()
            assert ((got.double() - want).abs() <= bound).all()
