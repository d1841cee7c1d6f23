"""The packed attention, the layer norm and the top-logits KL as a language-model target's
masked run uses them: norm, decomposed q/k/v/o projections around the attention, residual,
norm, head, and the KL to the clean run's stored top logits, with every gradient.

Tolerances: the same run in 64 bits with one of its intermediates moved by e times the
tensor's largest entry, up or down at random per entry, in the forward pass and in the
gradient that comes back through it, is off by as much as a run that rounds there. e is the
roundings' bound: half a step of the type where a tensor is stored in it, and n 2^-24 for a
sum of n terms in 32 bits (the tensor's largest entry stands for the sums' magnitudes). A
result may be off by the sum over the intermediates (the worst of three draws each)."""

import threading

import pytest
import torch

from param_decomp_amd import losses, ops
from param_decomp_amd.attention import packed_attention
from param_decomp_amd.decomposed_linear import SiteWeights, site_forward
from param_decomp_amd.norms import layer_norm

pytestmark = pytest.mark.gpu

F64 = torch.float64
D_MODEL, H, KV, D, C, VOCAB, TOP = 128, 4, 2, 32, 96, 1003, 16
LENGTHS, TAIL = (33, 1, 70, 19), 5  # sequences, and rows behind the last
SITES = {"q": (H * D, D_MODEL), "kv": (2 * KV * D, D_MODEL), "o": (D_MODEL, H * D)}


class _Move(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, e, gen):
        ctx.e, ctx.gen = e, gen
        return _moved(x, e, gen)

    @staticmethod
    def backward(ctx, g):
        return _moved(g, ctx.e, ctx.gen), None, None


def _moved(x, e, gen):
    sign = torch.randint(0, 2, x.shape, device=x.device, generator=gen).double() * 2 - 1
    return x + e * x.abs().max() * sign


def _make(device, dtype):
    g = torch.Generator(device=device).manual_seed(11)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    rows = sum(LENGTHS) + TAIL
    t = {"x": rnd(rows, D_MODEL), "head": rnd(VOCAB, D_MODEL) * D_MODEL**-0.5 * 2}
    for n, (out, inp) in SITES.items():
        t["V." + n], t["U." + n] = rnd(inp, C) * inp**-0.5, rnd(C, out) * C**-0.5
        t["W." + n] = (t["V." + n] @ t["U." + n]).T + 0.3 * rnd(out, inp) * inp**-0.5
        t["m." + n] = torch.rand(rows, C, device=device, generator=g)
        t["d." + n] = torch.rand(rows, device=device, generator=g)
    t = {n: v.to(dtype).contiguous() for n, v in t.items()}
    for n in ("1", "2"):
        t["w" + n], t["b" + n] = 1 + 0.2 * rnd(D_MODEL), 0.2 * rnd(D_MODEL)
    o = [0]
    for n in LENGTHS:
        o.append(o[-1] + n)
    return t, torch.tensor(o, dtype=torch.int32, device=device)


LEAVES = ("x", "w1", "b1", "w2", "b2", "head", "m.q", "m.kv", "m.o", "d.q", "d.kv", "d.o", "V.q", "U.kv", "V.o")


def _logits(t, offsets, site, masked=True):
    rows = t["x"].shape[0]
    h = layer_norm(t["x"], t["w1"], t["b1"])
    q = site(t, "q", h, masked).view(rows, H, D)
    kv = site(t, "kv", h, masked).view(rows, 2, KV, D)
    a = packed_attention(q, kv[:, 0], kv[:, 1], offsets)
    y = t["x"] + site(t, "o", a.reshape(rows, H * D), masked)
    return layer_norm(y, t["w2"], t["b2"]) @ t["head"].T


def _site(t, n, x, masked):
    w = SiteWeights(t["W." + n], t["V." + n], t["U." + n])
    if not masked:
        return x @ t["W." + n].T
    return site_forward(x, w, t["m." + n], t["d." + n], None).output


def _definition(t, offsets, top, idx, lse, at=None, e=None, gen=None):
    """Loss and gradients in 64 bits, with the intermediate `at` moved; e of each of them."""
    t = {n: v.detach().double().requires_grad_(n in LEAVES) for n, v in t.items()}
    names = []

    def mv(name, x, n):  # n: terms summed in 32 bits
        names.append((name, n))
        return _Move.apply(x, e[name], gen) if name == at else x

    def norm(x, n):
        z = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        return mv("norm" + n, z * t["w" + n] + t["b" + n], D_MODEL)

    def site(n, x):
        W, V, U = (t[k + n] for k in ("W.", "V.", "U."))
        xv = mv("xv." + n, x @ V, x.shape[1])
        delta = mv("delta." + n, x @ mv("W - VU." + n, W - (V @ U).T, C).T, x.shape[1])
        return mv("out." + n, mv("mask." + n, xv * t["m." + n], 1) @ U + t["d." + n][:, None] * delta, C)

    rows, rep = t["x"].shape[0], H // KV
    h = norm(t["x"], "1")
    q = site("q", h).view(rows, H, D)
    kv = site("kv", h).view(rows, 2, KV, D)
    pos = torch.arange(rows, device=q.device)
    seq = torch.bucketize(pos, offsets.long(), right=True)
    sees = (seq[:, None] == seq[None]) & (pos[:, None] >= pos[None]) & (pos < offsets[-1])[:, None]
    k, v = (kv[:, i].repeat_interleave(rep, 1).transpose(0, 1) for i in (0, 1))
    s = mv("scores", q.transpose(0, 1) @ k.transpose(1, 2) * D**-0.5, D)
    p = mv("p", torch.where(sees, torch.where(sees, s, -1e300).softmax(-1), 0.0), max(LENGTHS))
    a = mv("attention", (p @ v).transpose(0, 1).reshape(rows, H * D), max(LENGTHS))
    y = mv("residual", t["x"] + site("o", a), 1)
    z = mv("logits", norm(y, "2") @ t["head"].T, D_MODEL)
    lq = mv("log q", torch.log_softmax(z, -1), VOCAB)
    lp = top.double() - lse.double()[:, None]
    rest_p = (1 - lp.exp().sum(-1)).clamp_min(0)
    at_top = lq.gather(1, idx)
    rest_q = 1 - at_top.exp().sum(-1)
    kl = (lp.exp() * (lp - at_top)).sum(-1) + rest_p * (rest_p.clamp_min(1e-300).log() - rest_q.log())
    loss = kl.mean()
    grads = torch.autograd.grad(loss, [t[n] for n in LEAVES])
    return [loss.detach()] + [g.detach() for g in grads], names


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_and_its_gradients(device, dtype):
    t, offsets = _make(device, dtype)
    with torch.no_grad():
        clean = _logits(t, offsets, _site, masked=False)
        top, idx = clean.topk(TOP, -1)
        lse = torch.logsumexp(clean.float(), -1)
    for n in LEAVES:
        t[n].requires_grad_()
    loss = losses.top_logits_kl(_logits(t, offsets, _site), top, idx, clean_lse=lse)
    got = [loss.detach()] + [g.detach() for g in torch.autograd.grad(loss, [t[n] for n in LEAVES])]

    want, names = _definition(t, offsets, top, idx, lse)
    u = torch.finfo(dtype).eps / 2
    e = {n: u + k * 2.0**-24 for n, k in names}
    tol = [u * w.abs().max() for w in want]  # the results' own rounding
    for name in e:
        moves = []
        for seed in range(3):
            gen = torch.Generator(device=device).manual_seed(seed)
            moves.append(_definition(t, offsets, top, idx, lse, name, e, gen)[0])
        tol = [a + max((m[i] - w).abs().max() for m in moves) for i, (a, w) in enumerate(zip(tol, want))]
    for n, a, b, c in zip(("loss",) + LEAVES, got, want, tol):
        assert torch.isfinite(a).all(), n
        err = (a.double() - b).abs().max()
        assert err <= c, (n, float(err), float(c), float(b.abs().max()))


def _served(t, offsets, top, idx, lse, out):
    """Norm, attention and loss of one call without gradients."""
    rows = t["x"].shape[0]
    h = layer_norm(t["x"], t["w1"], t["b1"])
    q = (h @ t["W.q"].T).view(rows, H, D)
    kv = (h @ t["W.kv"].T).view(rows, 2, KV, D)
    a = packed_attention(q, kv[:, 0], kv[:, 1], offsets)
    z = layer_norm(a.reshape(rows, H * D), t["w2"], t["b2"]) @ t["head"].T
    kl, grad = ops.top_logits_kl(z, top, idx, clean_lse=lse, want_grad=True)
    for o, r in zip(out, (a, kl, grad)):
        o.copy_(r)


def _served_case(device, seed):
    t, offsets = _make(device, torch.bfloat16)
    g = torch.Generator(device=device).manual_seed(seed)
    rows = t["x"].shape[0]
    t["x"] = torch.randn(rows, D_MODEL, device=device, generator=g).bfloat16()
    clean = torch.randn(rows, VOCAB, device=device, generator=g).bfloat16()
    top, idx = clean.topk(TOP, -1)
    out = [torch.empty(rows, H, D, device=device, dtype=torch.bfloat16), torch.empty(rows, device=device),
           torch.empty(rows, VOCAB, device=device, dtype=torch.bfloat16)]
    return t, offsets, top, idx, torch.logsumexp(clean.float(), -1), out


def test_captured_run_replays_on_new_inputs(device):
    case = _served_case(device, 1)
    t, out = case[0], case[-1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _served(*case)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _served(*case)
    for seed in range(2, 6):
        t["x"].copy_(_served_case(device, seed)[0]["x"])
        graph.replay()
        got = [o.clone() for o in out]
        _served(*case)
        torch.cuda.synchronize()
        for a, b in zip(got, out):
            assert torch.equal(a, b), seed


def test_two_threads_on_two_streams(device):
    cases = [_served_case(device, s) for s in (7, 8)]
    want = []
    for c in cases:
        _served(*c)
        want.append([o.clone() for o in c[-1]])
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(2)

    def run(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                gate.wait(30)
                for _ in range(20):
                    for o in cases[i][-1]:
                        o.zero_()
                    _served(*cases[i])
                    s.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(cases[i][-1], want[i])):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001  (a thread's failure is the test's)
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    assert not wrong, wrong
