"""Packed causal attention against its definition in 64 bits, one sequence and head at a time.

Tolerances are elementwise bounds from the roundings made: u is half a step of the type
(2^-8 bf16, 2^-24 fp32), g_i a row's relative error of p from 32-bit scores and sums. With
the weights P and P |V| etc. of the definition:
  out: the operand P and the result are rounded to the type: (u + 2 g) sum p |v| + u |o|
  D_i = do . o from the stored out: |do| . (that error) + 32-bit sum
  ds:  u |ds| + 2 g p (|dp| + |D|) + p dD;  dq: scale ds_err |k| + u |dq|
  dv:  (u + 2 g) p^T |do| + u |dv|;  dk: scale ds_err^T |q| + u |dk|
A rounding takes at most half a step, so u is used as it is, with 5% for second orders."""

import math

import pytest
import torch

from param_decomp_amd import _lib as L
from param_decomp_amd import ops
from param_decomp_amd.attention import packed_attention

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _inputs(device, N, H, KV, D, dtype, seed=0, scale=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    return [(torch.randn(N, h, D, device=device, generator=g) * scale).to(dtype) for h in (H, KV, KV, H)]


def _offsets(device, lengths, first=0):
    o = [first]
    for n in lengths:
        o.append(o[-1] + n)
    return torch.tensor(o, dtype=torch.int32, device=device)


def _definition(q, k, v, g, lengths, first=0, scale=None):
    """(values, bounds) of out, dq, dk, dv in 64 bits."""
    N, H, D = q.shape
    rep = H // k.shape[1]
    scale = D**-0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    val = [torch.zeros(t.shape, dtype=F64, device=q.device) for t in (q, q, k, v)]
    tol = [torch.zeros_like(t) for t in val]
    a = first
    for n in lengths:
        at, a = slice(a, a + n), a + n
        if n == 0:
            continue
        above = torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1)
        for h in range(H):
            hk = h // rep
            Q, K, V, G = (t[at, i].double() for t, i in ((q, h), (k, hk), (v, hk), (g, h)))
            S = (Q @ K.T * scale).masked_fill_(above, -math.inf)
            P = torch.softmax(S, -1)
            O = P @ V
            mag = (Q.abs() @ K.abs().T * scale).masked_fill_(above, 0).amax(-1, keepdim=True)
            g1 = 2.0**-24 * ((D + 8) * mag + n + 32)  # 32-bit products, exponent and row sum
            eo = 1.05 * ((u + 2 * g1) * (P @ V.abs()) + u * O.abs())
            dP = G @ V.T
            Di = (G * O).sum(-1, keepdim=True)
            dS = P * (dP - Di)
            pair = 2.0**-24 * (D + 2) * (G.abs() @ V.abs().T)
            eD = (G.abs() * eo).sum(-1, keepdim=True) + 2.0**-24 * (D + 2) * (G.abs() * O.abs()).sum(-1, keepdim=True)
            eS = (u + 2 * g1) * dS.abs() + P * (pair + eD)
            sums = 2.0**-24 * (n * rep + 32)  # the 32-bit sums over positions (and heads)
            dQ, dK, dV = dS @ K * scale, dS.T @ Q * scale, P.T @ G
            eQ = (eS + sums * dS.abs()) @ K.abs() * scale + u * dQ.abs()
            eK = (eS + sums * dS.abs()).T @ Q.abs() * scale + u * dK.abs()
            eV = ((u + 2 * g1 + sums) * P).T @ G.abs() + u * dV.abs()
            for i, (x, e) in enumerate(((O, eo), (dQ, 1.05 * eQ), (dK, 1.05 * eK), (dV, 1.05 * eV))):
                at_head = h if i < 2 else hk
                val[i][at, at_head] += x
                tol[i][at, at_head] += e
    # the result's own rounding is of the sum over heads, at most that of its terms
    return val, [t + 1e-30 for t in tol]


def _check(got, val, tol, names=("out", "dq", "dk", "dv")):
    for x, y, e, name in zip(got, val, tol, names):
        assert x.shape == y.shape
        d = (x.double() - y).abs()
        assert torch.isfinite(x.float()).all(), name
        worst = (d / e).max().item()
        assert worst <= 1.0, f"{name}: {worst:.3g} of the bound, off by {d.max().item():.3g}"


def _grads(q, k, v, g, off, **kw):
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, off, **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


CASES = [
    # N, H, KV, D, lengths, first row
    (1, 1, 1, 64, [1], 0),
    (2, 2, 1, 64, [1, 1], 0),
    (33, 3, 3, 64, [33], 0),
    (64, 4, 2, 128, [31, 33], 0),
    (130, 2, 2, 128, [127, 3], 0),
    (200, 8, 2, 64, [1, 2, 0, 3, 64, 0, 65, 32, 33], 0),  # ends exactly at the last row
    (300, 4, 1, 128, [100, 129], 7),  # rows of no sequence before and behind
    (257, 6, 2, 80, [256, 1], 0),
    (515, 2, 1, 96, [511, 4], 0),
    (150, 3, 1, 8, [70, 80], 0),
    (140, 2, 2, 40, [139], 1),
    (129, 2, 1, 104, [128, 1], 0),
    (900, 2, 2, 64, [5] * 180, 0),
    (1030, 1, 1, 128, [1030], 0),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N, H, KV, D, lengths, first", CASES)
def test_forward_and_backward(device, dtype, N, H, KV, D, lengths, first):
    q, k, v, g = _inputs(device, N, H, KV, D, dtype, seed=N)
    val, tol = _definition(q, k, v, g, lengths, first)
    got = _grads(q, k, v, g, _offsets(device, lengths, first))
    _check(got, val, tol)
    # rows of no sequence: zeros
    rest = torch.ones(N, dtype=torch.bool, device=device)
    rest[first:first + sum(lengths)] = False
    for t in got:
        assert (t[rest] == 0).all()
    # the same bits without a gradient and a second time
    assert torch.equal(packed_attention(q, k, v, _offsets(device, lengths, first)), got[0])
    for x, y in zip(_grads(q, k, v, g, _offsets(device, lengths, first)), got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_sequence_of_many_tiles(device, dtype):
    N, H, KV, D, lengths = 2600, 4, 2, 64, [1999, 1, 600]
    q, k, v, g = _inputs(device, N, H, KV, D, dtype, seed=5, scale=1.5)
    _check(_grads(q, k, v, g, _offsets(device, lengths)), *_definition(q, k, v, g, lengths))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H, KV, D", [(32, 32, 64), (36, 36, 80), (32, 8, 128), (32, 4, 96), (64, 1, 64)])
def test_grids_that_fill_the_gpu(device, dtype, H, KV, D):
    """Enough rows and heads for 128-row tiles, shared key heads over one and several shares
    of their query heads, a tile that ends a sequence inside, rows behind the last."""
    N, lengths, first = 2100, [1, 700, 31, 1200, 100], 3
    q, k, v, g = _inputs(device, N, H, KV, D, dtype, seed=D)
    got = _grads(q, k, v, g, _offsets(device, lengths, first))
    _check(got, *_definition(q, k, v, g, lengths, first))
    rest = torch.ones(N, dtype=torch.bool, device=device)
    rest[first:first + sum(lengths)] = False
    for t in got:
        assert (t[rest] == 0).all()
    for x, y in zip(_grads(q, k, v, g, _offsets(device, lengths, first)), got):
        assert torch.equal(x, y)
    # NaN behind the last sequence and in one of them
    for t in (q, k, v, g):
        t[first + sum(lengths):] = math.nan
    for x, y in zip(_grads(q, k, v, g, _offsets(device, lengths, first)), got):
        assert torch.equal(x, y)
    k[first + 720] = v[first + 720] = math.inf  # inside the third sequence
    q[first + 715, H // 2], g[first + 716, 0] = math.nan, -math.inf
    val, tol = _definition(q.nan_to_num(0), k.nan_to_num(0), v.nan_to_num(0), g.nan_to_num(0), lengths, first)
    keep = ~rest
    keep[first + 701:first + 732] = False
    for x, y, e in zip(_grads(q, k, v, g, _offsets(device, lengths, first)), val, tol):
        assert ((x.double() - y).abs() <= e)[keep].all()


@pytest.mark.parametrize("H, KV", [(2, 1), (32, 32)])
def test_more_sequences_than_a_block_holds_offsets_of(device, H, KV):
    lengths = ([1, 2, 0, 3, 1] * 500)[:2300]
    N = sum(lengths) + 7
    q, k, v, g = _inputs(device, N, H, KV, 64, BF16, seed=12)
    got = _grads(q, k, v, g, _offsets(device, lengths, 4))
    _check(got, *_definition(q, k, v, g, lengths, 4))


@pytest.mark.parametrize("scale", [0.5, 0.0, -0.3])
def test_scale(device, scale):
    q, k, v, g = _inputs(device, 100, 2, 1, 64, BF16, seed=3)
    _check(_grads(q, k, v, g, _offsets(device, [60, 40]), scale=scale),
           *_definition(q, k, v, g, [60, 40], scale=scale))


def test_scores_that_grow_along_the_sequence(device):
    """The running maximum rises at every tile, and falls from the first key on in the
    other head: large scores of both signs."""
    N, D = 700, 64
    q, k, v, g = _inputs(device, N, 2, 2, D, F32, seed=4, scale=0.2)
    ramp = torch.linspace(-20, 20, N, device=device)
    q[:, :, 0] = 8.0
    k[:, 0, 0], k[:, 1, 0] = ramp, -ramp
    _check(_grads(q, k, v, g, _offsets(device, [N])), *_definition(q, k, v, g, [N]))


def test_no_sequences_and_no_rows(device):
    q, k, v, g = _inputs(device, 70, 2, 1, 64, BF16)
    for off in (torch.zeros(1, dtype=torch.int32, device=device), _offsets(device, [0, 0], first=70),
                _offsets(device, [0], first=5)):
        for t in _grads(q, k, v, g, off):
            assert (t == 0).all()
    e = [t[:0] for t in (q, k, v, g)]
    for t, like in zip(_grads(*e, _offsets(device, [0])), (e[0], e[0], e[1], e[2])):
        assert t.shape == like.shape


def test_head_width_not_a_multiple_of_8(device):
    q, k, v, g = _inputs(device, 90, 4, 2, 20, BF16, seed=8)
    _check(_grads(q, k, v, g, _offsets(device, [50, 40])), *_definition(q, k, v, g, [50, 40]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views_of_one_projection(device, dtype):
    """q, k and v as views of one buffer (the same results as dense copies), and views
    whose rows are not aligned (copied by the caller-facing function)."""
    N, H, KV, D = 210, 4, 2, 64
    gen = torch.Generator(device=device).manual_seed(1)
    qkv = torch.randn(N, (H + 2 * KV) * D + 24, device=device, generator=gen).to(dtype)
    off = _offsets(device, [100, 110])
    for lead in (0, 8, 1, 3):
        parts, at = [], lead
        for heads in (H, KV, KV):
            parts.append(qkv[:, at:at + heads * D].view(N, heads, D))
            at += heads * D
        g = torch.randn(N, H, D, device=device, generator=gen).to(dtype)
        for x, y in zip(_grads2(parts, g, off), _grads2([t.contiguous() for t in parts], g, off)):
            assert torch.equal(x, y)
    # head-major storage, and a key head shared by a broadcast
    hm = qkv[:, :H * D].reshape(N, H, D).transpose(0, 1).contiguous().transpose(0, 1)
    one = qkv[:, :D].reshape(N, 1, D).expand(N, KV, D)
    g = torch.randn(N, H, D, device=device, generator=gen).to(dtype)
    for x, y in zip(_grads2([hm, one, one], g, off), _grads2([hm.contiguous(), one.contiguous(), one.contiguous()], g, off)):
        assert torch.equal(x, y)


def _grads2(qkv, g, off):
    leaves = [t.detach().requires_grad_() for t in qkv]  # the views themselves
    out = packed_attention(*leaves, off)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


def test_broadcast_leaf_sums_its_gradient(device):
    """One key head expanded to all: the gradient of the shared leaf is the heads' sum."""
    q, k, v, g = _inputs(device, 120, 4, 1, 64, F32, seed=2)
    off = _offsets(device, [120])
    k1, v1 = k.clone().requires_grad_(), v.clone().requires_grad_()
    out = packed_attention(q, k1.expand(-1, 4, -1), v1.expand(-1, 4, -1), off)
    dk, dv = torch.autograd.grad(out, (k1, v1), g)
    val, tol = _definition(q, k, v, g, [120])
    _check((dk, dv), val[2:], tol[2:], ("dk", "dv"))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 128])
def test_hidden_rows_reach_nobody(device, dtype, poison, D):
    """NaN or infinities in rows of no sequence, in another sequence and in later rows of
    the same one change no bit of the other sequences, and no finite value of rows before."""
    N, H, KV, lengths, first = 230, 2, 1, [50, 60, 100], 5
    q, k, v, g = _inputs(device, N, H, KV, D, dtype, seed=11)
    off = _offsets(device, lengths, first)
    clean = _grads(q, k, v, g, off)
    val, tol = _definition(q, k, v, g, lengths, first)
    bad = [t.clone() for t in (q, k, v, g)]
    late = first + 50 + 40  # a row in the middle of the second sequence
    for t in bad:
        t[:first] = poison
        t[first + sum(lengths):] = poison
    edge = _grads(*bad, off)
    for x, y in zip(edge, clean):
        assert torch.equal(x, y)
    for t in bad[1:3]:
        t[late] = poison
    got = _grads(*bad, off)
    seen = slice(first + 50, first + 110)
    for x, y, e, name in zip(got, val, tol, ("out", "dq", "dk", "dv")):
        others = torch.ones(N, dtype=torch.bool, device=device)
        others[seen] = False
        inside = torch.zeros_like(others)
        inside[first:first + sum(lengths)] = True
        assert ((x.double() - y).abs() <= e)[others & inside].all(), name
    before = slice(first + 50, late)  # outputs and dq of earlier rows do not see it
    for i in (0, 1):
        assert ((got[i].double() - val[i]).abs() <= tol[i])[before].all()
    assert not torch.isfinite(got[0][late].float()).all()
    # poison in queries and cotangents: dk and dv of later rows do not see it
    bad = [t.clone() for t in (q, k, v, g)]
    bad[0][late] = poison
    bad[3][late] = poison
    got = _grads(*bad, off)
    for x, y, e in zip(got, val, tol):
        ok = (x.double() - y).abs() <= e
        assert ok[first:first + 50].all() and ok[first + 110:first + 210].all()
    after = slice(late + 1, first + 110)
    for i in range(4):
        assert ((got[i].double() - val[i]).abs() <= tol[i])[after].all()


def test_scores_of_the_lowest_value(device):
    """Scores at -inf from infinite keys leave the others' weights alone; a lowest finite
    value does too."""
    q, k, v, g = _inputs(device, 40, 1, 1, 64, F32, seed=6)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    for low in (-math.inf, -3e38):
        kk = k.clone()
        kk[10, 0, 0] = low
        out = packed_attention(q, kk, v, _offsets(device, [40]))
        keep = torch.ones(40, dtype=torch.bool, device=device)
        keep[10] = False
        want = torch.zeros(40, 64, dtype=F64, device=device)
        for i in range(40):
            js = [j for j in range(i + 1) if j != 10]
            s = (q[i, 0].double() @ k[js, 0].double().T) / 8
            want[i] = torch.softmax(s, -1) @ v[js, 0].double()
        if low == -math.inf:
            assert (out[keep, 0].double() - want[keep]).abs().max() < 1e-5
        else:  # q k = -3e38 |q|: a finite score of no weight
            assert (out[11:, 0].double() - want[11:]).abs().max() < 1e-5


def test_out_keeps_rows_of_no_sequence(device):
    q, k, v, _ = _inputs(device, 300, 2, 2, 64, BF16)
    off = _offsets(device, [10, 200], first=20)
    out = torch.full_like(q, 7.0)
    same, saved = ops.packed_attention_fwd(q, k, v, off, out=out)
    assert same is out and saved is None
    assert (out[:20] == 7).all() and (out[230:] == 7).all()
    assert torch.equal(out[20:230], packed_attention(q, k, v, off)[20:230])


def test_offsets_that_are_out_of_order_stay_inside(device):
    """Wrong offsets give wrong rows, not accesses outside: rows behind the tensors and
    around them keep their values."""
    N = 200
    big = torch.full((N + 256, 2, 64), 3.0, dtype=BF16, device=device)
    q, k, v, g = _inputs(device, N, 2, 2, 64, BF16)
    for o in ([50, 20, 199], [0, 5000, 7], [-9, 4, 90], [150, 150, 100], [300, 400]):
        out = big[128:128 + N]
        ops.packed_attention_fwd(q, k, v, torch.tensor(o, dtype=torch.int32, device=device), out=out)
        _grads(q, k, v, g, torch.tensor(o, dtype=torch.int32, device=device))
        torch.cuda.synchronize()
        assert (big[:128] == 3).all() and (big[128 + N:] == 3).all()


def test_rows_past_32_bit_offsets(device):
    """Row strides that put the last rows beyond 2^31 elements and 2^32 bytes; rows further
    apart than the kernels reach are copied."""
    for N, stride in ((140, 1 << 24), (600, 1 << 22)):
        _far_rows(device, N, stride)


def _far_rows(device, N, stride):
    D = 64
    q, k, v, g = _inputs(device, N, 1, 1, D, BF16, seed=9)
    off = _offsets(device, [N - 1], first=1)
    far = torch.empty(N * stride, dtype=BF16, device=device).view(N, stride)
    far[:, :D], far[:, D:2 * D], far[:, 2 * D:3 * D] = q[:, 0], k[:, 0], v[:, 0]
    views = [far[:, i * D:(i + 1) * D].view(N, 1, D) for i in range(3)]
    for x, y in zip(_grads2(views, g, off), _grads(q, k, v, g, off)):
        assert torch.equal(x, y)


def test_partial_gradients_and_no_second_derivative(device):
    q, k, v, g = _inputs(device, 80, 2, 1, 64, F32, seed=3)
    off = _offsets(device, [80])
    full = _grads(q, k, v, g, off)
    k1 = k.clone().requires_grad_()
    out = packed_attention(q, k1, v, off)
    assert torch.equal(torch.autograd.grad(out, k1, g)[0], full[2])
    out = packed_attention(q, k1, v, off)
    gg = g.clone().requires_grad_()
    (dk,) = torch.autograd.grad(out, k1, gg, create_graph=True)
    with pytest.raises(RuntimeError):
        dk.sum().backward()


def test_gradient_is_the_difference_of_the_definition(device):
    """Along a random direction, the definition's central difference in 64 bits."""
    lengths, N = [37, 53], 90
    q, k, v, g = _inputs(device, N, 4, 2, 64, F32, seed=7)
    got = _grads(q, k, v, g, _offsets(device, lengths))[1:]
    gen = torch.Generator(device=device).manual_seed(3)
    dirs = [torch.randn(t.shape, device=device, generator=gen, dtype=F64) for t in (q, k, v)]

    def loss(t):
        moved = [x.double() + t * d for x, d in zip((q, k, v), dirs)]
        total = 0.0
        a = 0
        for n in lengths:
            at, a = slice(a, a + n), a + n
            for h in range(4):
                Q, K, V = moved[0][at, h], moved[1][at, h // 2], moved[2][at, h // 2]
                S = (Q @ K.T / 8).masked_fill(torch.ones(n, n, dtype=torch.bool, device=device).triu(1), -math.inf)
                total = total + ((torch.softmax(S, -1) @ V) * g[at, h].double()).sum()
        return float(total)

    h = 1e-5
    want = (loss(h) - loss(-h)) / (2 * h)
    have = sum(float((x.double() * d).sum()) for x, d in zip(got, dirs))
    # the difference is off by h^2 times a third derivative and 2^-52 |loss| / h; the
    # gradients by their 32-bit bound
    size = sum(float((x.double().abs() * d.abs()).sum()) for x, d in zip(got, dirs))
    assert abs(want - have) <= 2e-5 * size


def test_another_stream(device):
    q, k, v, g = _inputs(device, 500, 4, 2, 128, BF16, seed=2)
    off = _offsets(device, [123, 377])
    want = _grads(q, k, v, g, off)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(device=device)
    with torch.cuda.stream(side):
        got = _grads(q, k, v, g, off)
    side.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_graph_replays(device):
    """Captured forward and backward calls replay on new inputs, offsets included, with
    eager calls between the replays."""
    N, H, KV, D = 400, 4, 2, 64
    static = _inputs(device, N, H, KV, D, BF16, seed=0)
    off = _offsets(device, [100, 300])

    def calls(q, k, v, g, off):
        out, saved = ops.packed_attention_fwd(q, k, v, off, want_saved=True)
        return (out, *ops.packed_attention_bwd(q, k, v, off, out, saved, g))

    calls(*static, off)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs over the same inputs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = calls(*static, off)
        graphs.append((graph, got))
    for i, lengths in enumerate(([400, 0], [1, 399], [250, 100], [7, 13])):
        for dst, src in zip(static, _inputs(device, N, H, KV, D, BF16, seed=i + 1)):
            dst.copy_(src)
        off.copy_(_offsets(device, lengths))
        for graph, got in graphs:
            for t in got:
                t.fill_(float("nan"))
            graph.replay()
        want = calls(*static, off)
        torch.cuda.synchronize()
        for _, got in graphs:
            for x, y in zip(got, want):
                assert torch.equal(x, y)


def test_mixed_devices_are_refused(device):
    q, k, v, _ = _inputs(device, 10, 2, 1, 64, BF16)
    with pytest.raises(L.PDError, match="offsets is on cpu"):
        packed_attention(q, k, v, torch.tensor([0, 10], dtype=torch.int32))
    with pytest.raises(L.PDError, match="k is on cpu"):
        packed_attention(q, k.cpu(), v, _offsets(device, [10]))


@pytest.mark.parametrize("dtype, H, KV, D", [(BF16, 32, 8, 64), (BF16, 32, 32, 128), (F32, 36, 36, 64)])
@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_hidden_rows_reach_nobody_in_large_grids(device, dtype, H, KV, D, poison):
    """Waves of 128-row tiles that hold one sequence's end and the next one's start see
    whole blocks in some lanes only: poison in the one sequence stays there."""
    N, lengths, first = 2100, [517, 790, 3, 700], 2
    q, k, v, g = _inputs(device, N, H, KV, D, dtype, seed=23)
    off = _offsets(device, lengths, first)
    clean = _grads(q, k, v, g, off)
    val, tol = _definition(q, k, v, g, lengths, first)
    _check(clean, val, tol)
    seen = slice(first + 517, first + 517 + 790)
    bad = [t.clone() for t in (q, k, v, g)]
    for t in bad:
        t[seen.start + 400] = poison
        t[:first] = poison
        t[first + sum(lengths):] = poison
    others = torch.zeros(N, dtype=torch.bool, device=device)
    others[first:first + sum(lengths)] = True
    others[seen] = False
    for x, y, e in zip(_grads(*bad, off), val, tol):
        assert ((x.double() - y).abs() <= e)[others].all()


@pytest.mark.parametrize("N, H, lengths, first", [(8300, 3, [1, 64, 700, 31] * 10, 5), (4100, 9, [129] * 31, 0)])
def test_every_tile_is_taken_once(device, N, H, lengths, first):
    """More tiles than the blocks put in order, and as many as they do, in 32-row forms."""
    q, k, v, g = _inputs(device, N, H, 1, 64, BF16, seed=29)
    got = _grads(q, k, v, g, _offsets(device, lengths, first))
    _check(got, *_definition(q, k, v, g, lengths, first))


def test_offsets_that_are_out_of_order_stay_inside_in_large_grids(device):
    N = 2100
    big = torch.full((N + 256, 32, 64), 3.0, dtype=BF16, device=device)
    q, k, v, g = _inputs(device, N, 32, 32, 64, BF16)
    for o in ([50, 20, 1999], [0, 5000, 7], [-9, 4, 2090], [2**31 - 1, -(2**31), 100], [1500, 100, 900, 0, 2100]):
        out = big[128:128 + N]
        ops.packed_attention_fwd(q, k, v, torch.tensor(o, dtype=torch.int32, device=device), out=out)
        _grads(q, k, v, g, torch.tensor(o, dtype=torch.int32, device=device))
        torch.cuda.synchronize()
        assert (big[:128] == 3).all() and (big[128 + N:] == 3).all()
