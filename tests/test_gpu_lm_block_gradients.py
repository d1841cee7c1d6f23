"""Gradients of the masked run of `test_gpu_lm_block` in bounds that a missing gradient fails.

Every intermediate is stored with a rounding of at most half a step of its own value (u |x|)
and, where it is a sum of n terms in 32 bits, n 2^-24 of the tensor's largest; so is the
gradient that comes back through it. The roundings of different entries are independent of
each other, so a result is off, in the root of its summed squares, by the root of the summed
squares of what each intermediate does to it: here of the definition in 64 bits with one
intermediate moved by its full bound, up or down at random per entry (a rounding is off by
less: 1 / sqrt(3) of it on average). Twice that is the limit. It has to be small beside the
gradient itself, or it would say nothing."""

import threading

import pytest
import test_gpu_lm_block as block
import torch

from param_decomp_amd import losses

F64 = torch.float64
LEAVES = block.LEAVES
SMALL = 0.1  # of a result: what its limit may be at most


def _moved(x, e, gen):
    sign = torch.randint(0, 2, x.shape, device=x.device, generator=gen).double() * 2 - 1
    return x + (e[0] * x.abs() + e[1] * x.abs().max()) * sign


def _limits(monkeypatch, t, offsets, top, idx, lse, dtype):
    monkeypatch.setattr(block, "_moved", _moved)
    u = torch.finfo(dtype).eps / 2
    want, names = block._definition(t, offsets, top, idx, lse)
    # the log of q stays in 32 bits whatever the logits' type
    e = {n: (2.0**-24 if n == "log q" else u, k * 2.0**-24) for n, k in names}
    squares = [(u * w.norm())**2 for w in want]
    draws = 3
    for name in e:
        for seed in range(draws):
            gen = torch.Generator(device=t["x"].device).manual_seed(seed)
            got = block._definition(t, offsets, top, idx, lse, name, e, gen)[0]
            squares = [s + (g - w).norm()**2 / draws for s, g, w in zip(squares, got, want)]
    return want, [2 * s.sqrt() for s in squares]


def _case(device, dtype, clean):
    t, offsets = block._make(device, dtype)
    z = clean(t, offsets)
    top, idx = z.topk(block.TOP, -1)
    return t, offsets, top, idx, torch.logsumexp(z.float(), -1)


def test_limits_are_small_beside_the_gradients(monkeypatch):
    """On the CPU, with any clean logits: what the comparison on the GPU rests on."""
    t, offsets, top, idx, lse = _case("cpu", torch.bfloat16, lambda t, _: (
        torch.randn(t["x"].shape[0], block.VOCAB, generator=torch.Generator().manual_seed(2)) * 2).bfloat16())
    want, tol = _limits(monkeypatch, t, offsets, top, idx, lse, torch.bfloat16)
    for n, w, c in zip(("loss",) + LEAVES, want, tol):
        assert c <= SMALL * w.norm(), (n, float(c / w.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_gradients(monkeypatch, device, dtype):
    with torch.no_grad():
        t, offsets, top, idx, lse = _case(device, dtype, lambda t, o: block._logits(t, o, block._site, masked=False))
    for n in LEAVES:
        t[n].requires_grad_()
    loss = losses.top_logits_kl(block._logits(t, offsets, block._site), top, idx, clean_lse=lse)
    got = [loss.detach()] + [g.detach() for g in torch.autograd.grad(loss, [t[n] for n in LEAVES])]
    want, tol = _limits(monkeypatch, t, offsets, top, idx, lse, dtype)
    for n, a, b, c in zip(("loss",) + LEAVES, got, want, tol):
        assert c <= SMALL * b.norm(), (n, float(c / b.norm()))
        err = (a.double() - b).norm()
        assert err <= c, (n, float(err / b.norm()), float(c / b.norm()))


@pytest.mark.gpu
def test_two_threads_with_gradients(device):
    """Two training runs at once, each on its own stream, give the bits of a run alone."""
    cases = []
    for seed in (3, 4):
        with torch.no_grad():
            t, offsets, top, idx, lse = _case(device, torch.bfloat16, lambda t, o: block._logits(t, o, block._site, masked=False))
            t["x"] = torch.randn(t["x"].shape, device=device, generator=torch.Generator(device=device).manual_seed(seed)).bfloat16()
        for n in LEAVES:
            t[n].requires_grad_()
        cases.append((t, offsets, top, idx, lse))

    def run(case):
        t, offsets, top, idx, lse = case
        loss = losses.top_logits_kl(block._logits(t, offsets, block._site), top, idx, clean_lse=lse)
        return [loss.detach()] + list(torch.autograd.grad(loss, [t[n] for n in LEAVES]))

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    wrong, gate, done = [], threading.Barrier(2), []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                gate.wait(30)
                for _ in range(10):
                    got = run(cases[i])
                    s.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
            done.append(i)
        except Exception as e:  # noqa: BLE001  (a thread's failure is the test's)
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,), daemon=True) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    assert not any(th.is_alive() for th in threads)
    assert not wrong and sorted(done) == [0, 1], wrong
