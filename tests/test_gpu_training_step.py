"""A training step of a mixture-of-experts language-model target as its operators are used together: norm,
router, experts' products, residual norm with a gate, cross entropy over the vocabulary, all gradients, and the
optimizer's step, against the same formulas in 64 bits and against differences of the loss.

Tolerances: the same step in 64 bits with one of its intermediates moved by e times the tensor's largest
entry, up or down at random per entry, forward and in the gradient that comes back through it, is off by as much
as a step that rounds there. e is half a step of bf16 where a tensor is stored in it, and n 2^-24 for a sum of n
terms in 32 bits. A result may be off by the sum over the intermediates (the worst of three draws each). The
choice of experts is that of the 64-bit scores of the stored logits on both sides."""

import threading

import pytest
import torch

from param_decomp_amd import losses
from param_decomp_amd.norms import residual_norm, rms_norm
from param_decomp_amd.optim import AdamW
from param_decomp_amd.routed import experts

pytestmark = pytest.mark.gpu

F64, BF16 = torch.float64, torch.bfloat16
B, T, D, HID, E, K, V = 3, 40, 64, 64, 16, 4, 515
HALF, U = 2.0**-8, 2.0**-24
LEAVES = ("x", "wpre", "wpost", "wout", "gate", "router", "up", "down", "head")


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


def _make(device, seed=1):
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    t = dict(x=rnd(B, T, D), router=rnd(D, E) * D**-0.5 * 2, up=rnd(E, D, HID) * D**-0.5, down=rnd(E, HID, D) * HID**-0.5,
             head=rnd(V, D) * D**-0.5 * 2)
    t = {n: v.bfloat16() for n, v in t.items()}
    t.update(wpre=1 + 0.2 * rnd(D), wpost=1 + 0.2 * rnd(D), wout=1 + 0.2 * rnd(D), gate=0.5 + 0.3 * rnd(B, D))
    bias = 0.1 * rnd(E)
    targets = torch.randint(V, (B, T), device=device, generator=g)
    targets[:, :7] = -100  # a prompt
    return t, bias, targets


def _step(t, bias, targets):
    """(loss, chosen experts) by the framework."""
    h = rms_norm(t["x"], t["wpre"])
    flat = h.view(B * T, D)
    w, idx = experts.route_scores(flat @ t["router"], K, scoring="sigmoid", bias=bias, n_groups=4, top_groups=2, scale=1.5)
    jobs = experts.routed_jobs(idx, E)
    a = experts.grouped_matmul(experts.gather_tokens(flat, jobs), t["up"], jobs)
    b = experts.combine_jobs(experts.grouped_matmul(a * torch.sigmoid(a), t["down"], jobs), jobs, w)
    _, y = residual_norm(t["x"], b.view(B, T, D), post_weight=t["wpost"], gate=t["gate"], pre_weight=t["wout"], scale=0.8)
    return losses.streamed_cross_entropy(y, t["head"], targets), idx


def _exact(t, targets, idx, move=None, draw=0):
    """The loss in 64 bits for the experts idx, with intermediate `move` moved."""
    gen = torch.Generator(device=targets.device).manual_seed(100 * draw + 7)
    at = [0]

    def r(x, e):  # one of the step's intermediates
        at[0] += 1
        return _Move.apply(x, e, gen) if at[0] == move else x

    x = t["x"].view(B * T, D)
    norm = lambda u: u / (u.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    h = r(norm(x) * t["wpre"], HALF + 64 * U)
    z = r(h @ t["router"], HALF + D * U)
    s = torch.sigmoid(z).gather(1, idx.long())
    w = r(1.5 * s / s.sum(-1, keepdim=True), 64 * U)
    a = r(torch.einsum("td,tkdh->tkh", h, t["up"][idx.long()]), HALF + D * U)
    g = r(r(torch.sigmoid(a), HALF) * a, HALF)
    o = r(torch.einsum("tkh,tkhd->tkd", g, t["down"][idx.long()]), HALF + HID * U)
    b = r((o * w[..., None]).sum(1), 2 * HALF + K * U)  # weights may enter in bf16
    n = norm(b) * t["wpost"]
    st = r(x + 0.8 * t["gate"].repeat_interleave(T, 0) * n, HALF + 64 * U)
    y = r(norm(st) * t["wout"], HALF + 64 * U)
    q = r(y @ t["head"].T, D * U)
    on = targets.view(-1) >= 0
    lp = r(torch.log_softmax(q, -1), HALF)  # G enters its products in bf16
    return -lp[on, targets.view(-1)[on]].mean(), at[0]


def _grads(t, targets, idx, move=None, draw=0):
    leaves = {n: t[n].detach().double().requires_grad_() for n in LEAVES}
    loss, n = _exact(leaves, targets, idx, move, draw)
    return [loss.detach(), *torch.autograd.grad(loss, [leaves[n] for n in LEAVES])], n


def test_the_step_and_its_gradients(device):
    t, bias, targets = _make(device)
    leaves = {n: t[n].requires_grad_() for n in LEAVES}
    loss, idx = _step(leaves, bias, targets)
    got = [loss.detach(), *torch.autograd.grad(loss, [leaves[n] for n in LEAVES])]
    want, n = _grads(t, targets, idx)
    tol = [torch.zeros((), device=device, dtype=F64) for _ in want]
    for i in range(1, n + 1):
        worst = [torch.zeros((), device=device, dtype=F64) for _ in want]
        for draw in range(3):
            for k, (a, b) in enumerate(zip(_grads(t, targets, idx, i, draw)[0], want)):
                worst[k] = torch.maximum(worst[k], (a - b).abs().max())
        tol = [a + b for a, b in zip(tol, worst)]
    for name, a, b, c in zip(("loss",) + LEAVES, got, want, tol):
        half = HALF if a.dtype == BF16 else U
        err = (a.double() - b).abs().max()
        assert torch.isfinite(a).all() and err <= c + half * b.abs().max(), (name, float(err), float(c), float(b.abs().max()))


def test_gradients_are_the_losses_differences(device):
    """The 64-bit step's gradients, which the test above holds the kernels to, against its own differences."""
    t, bias, targets = _make(device, 2)
    with torch.no_grad():
        _, idx = _step(t, bias, targets)
    want, _ = _grads(t, targets, idx)
    g = torch.Generator(device=device).manual_seed(3)
    for n, d in zip(LEAVES, want[1:]):
        v = torch.randn(t[n].shape, device=device, generator=g, dtype=F64)
        h = 1e-5
        f = lambda s: float(_exact({m: t[m].double() + (s * v if m == n else 0) for m in LEAVES}, targets, idx)[0])  # noqa: E731
        diff = (f(h) - f(-h)) / (2 * h)
        assert abs(diff - float((d * v).sum())) <= 1e-6 * float((d * v).abs().sum()) + 1e-9, n


def _train(device, seed, steps, capture=False, bits=8):
    """Master weights after some steps; captured: the step and the optimizer in one graph."""
    t, bias, targets = _make(device, seed)
    names = ("router", "up", "down", "head", "wpre", "wpost", "wout", "gate")
    leaves = {n: t[n].detach().clone().requires_grad_() for n in LEAVES}
    master = [leaves[n].detach().float().clone() if leaves[n].dtype == BF16 else leaves[n].detach() for n in names]
    copies = [leaves[n].detach() if leaves[n].dtype == BF16 else None for n in names]
    opt = AdamW(master, lr=1e-2, weight_decay=0.01, state_bits=bits, key=(seed, 5), copies=copies)

    def step():
        loss, _ = _step(leaves, bias, targets)
        opt.step(torch.autograd.grad(loss, [leaves[n] for n in names]))
        return loss.detach()

    if not capture:
        for _ in range(steps):
            loss = step()
        return master + [loss]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    for _ in range(steps - 1):
        graph.replay()
        torch.cuda.synchronize()
    return master + [loss]


def test_captured_training_is_the_same(device):
    for a, b in zip(_train(device, 4, 5), _train(device, 4, 5, capture=True)):
        assert torch.equal(a, b)


def test_two_threads_on_two_streams(device):
    want = [_train(device, s, 4) for s in (5, 6)]
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(2)

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait(30)
                for _ in range(3):
                    got = _train(device, 5 + i, 4)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001  (a thread's failure is the test's)
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    assert not wrong, wrong
