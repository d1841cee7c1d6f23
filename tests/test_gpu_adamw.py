"""AdamW over many tensors against the formula in 64 bits.

Tolerances count roundings of the kernel's fp32 arithmetic (2^-24 each, relative to the magnitudes of
what is added): m and v take three, the step about 16 (bias corrections, square root, reciprocal and
products), and p one more for its own size. An 8-bit code is one of the two e4m3 neighbours of what it
rounds, the one that the 16 random bits choose; a value within 2^-12 of a code's step of the threshold may go
either way (m and v are a few 2^-24 off, a step is at least 2^-4 of the value)."""

import math

import numpy as np
import pytest
import torch

from oracle import threefry as tf
from param_decomp_amd import _lib as L
from param_decomp_amd.optim import AdamW

pytestmark = pytest.mark.gpu

F64 = torch.float64
U = 2.0**-24
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.99, 1e-8, 0.02
SIZES = [1, 2, 255, 256, 257, 1023, 1024, 1025, 5000, 0, 70000]


def _tensors(device, sizes, seed=0, grad=torch.float32, offset=0):
    g = torch.Generator(device=device).manual_seed(seed)
    p, gr = [], []
    for n in sizes:
        flat = torch.randn(n + offset, device=device, generator=g)
        p.append(flat[offset:])
        gr.append((torch.randn(n, device=device, generator=g) * 10.0**float(torch.randint(-6, 2, (1,), generator=g, device=device)))
                  .to(grad))
    return p, gr


def _expected(p, g, m, v, t, lr=LR):
    """(p, m, v, bound of p, m, v) in 64 bits."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m2, v2 = m + (1 - B1) * (g - m), v + (1 - B2) * (g * g - v)
    step = lr * (m2 / (1 - B1**t)) / ((v2 / (1 - B2**t)).sqrt() + EPS)
    bm, bv = 4 * U * (m.abs() + g.abs()), 4 * U * (v + g * g)
    # m's own error against the denominator, and the step's roundings
    bp = 4 * U * p.abs() + 32 * U * step.abs() + lr / (1 - B1**t) * bm / ((v2 / (1 - B2**t)).sqrt() + EPS)
    return p - lr * WD * p - step, m2, v2, bp, bm, bv


def _within(a, want, bound):
    err = (a.double() - want).abs()
    assert (err <= bound).all(), float((err - bound).max())


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_fp32_states(device, grad, offset):
    p, g = _tensors(device, SIZES, 1, grad, offset)
    copies = [torch.empty(n + 1, dtype=torch.bfloat16, device=device)[1:] if i % 2 else None for i, n in enumerate(SIZES)]
    opt = AdamW(p, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, copies=copies)
    for t in range(1, 4):
        before = [[x.clone() for x in ts] for ts in (p, opt.state["m"], opt.state["v"])]
        opt.step([x * t for x in g])
        for i in range(len(SIZES)):
            want = _expected(before[0][i], g[i] * t, before[1][i], before[2][i], t)
            for a, w, b in zip((p[i], opt.state["m"][i], opt.state["v"][i]), want[:3], want[3:]):
                _within(a, w, b)
            if copies[i] is not None:
                assert torch.equal(copies[i], p[i].bfloat16())
    assert int(opt.state["step"]) == 3


def _bits(key, step, n, base):
    """The random words of n values from index `base` on."""
    kt = tf.fold_in(key, step)
    pair = (np.arange(n) + base) // 2
    x0, x1 = tf.threefry2x32(kt, (pair >> 32).astype(np.uint32), (pair & 0xFFFFFFFF).astype(np.uint32))
    return np.where((np.arange(n) + base) % 2, x1, x0).astype(np.uint64)


def _check_codes(codes, scale, x, bits, floor):
    """codes (e4m3) of x / scale: the neighbour that the bits choose."""
    n = x.numel()
    per = scale.double().repeat_interleave(256)[:n]
    x, q = x.double().cpu(), codes.double().cpu()
    a = torch.where(per.cpu() > 0, x.abs() / per.cpu().clamp(min=1e-300), torch.zeros_like(x)).clamp(max=448.0)
    step = torch.where(a >= 2.0**-6, 2.0**(torch.floor(torch.log2(a.clamp(min=2.0**-6))) - 3), torch.full_like(a, 2.0**-9))
    low = torch.floor(a / step) * step
    frac = (a - low) / step
    up = frac + torch.from_numpy((bits & 0xFFFF).astype(np.float64)) / 65536
    want = low + step * (up >= 1)
    sure = ((up - 1).abs() > 2.0**-12) & (frac > 2.0**-12) & (frac < 1 - 2.0**-12)
    if floor:
        want = torch.where((a > 0) & (want == 0), torch.full_like(want, 2.0**-9), want)
    got = q.abs()
    assert torch.equal(got[sure], want[sure])
    assert ((got - a).abs() <= step * 1.01).all()
    assert (q * x >= 0).all()
    assert sure.double().mean() > 0.9 or n < 64


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
def test_8_bit_states(device, grad):
    sizes, key = [1, 255, 256, 257, 3000, 40000], (123, 0xFFFFFFF0)
    p, g = _tensors(device, sizes, 2, grad)
    opt = AdamW(p, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8, key=key)
    st = opt.state
    for t in range(1, 4):
        wide = lambda n, i: st[n][i].double() * st[n + "_scale"][i].double().repeat_interleave(256)[:sizes[i]]  # noqa: E731
        before = [(p[i].clone(), wide("m", i).float(), wide("v", i).float()) for i in range(len(sizes))]
        opt.step([x * t for x in g])
        base = 0
        for i, n in enumerate(sizes):
            p0, m0, r0 = before[i]
            want = _expected(p0, g[i] * t, m0, r0.double()**2, t)
            _within(p[i], want[0], want[3])
            bits = _bits(key, t, n, base)
            for name, x, b, floor in (("m", want[1], bits, False), ("v", want[2].sqrt(), bits >> 16, True)):
                top = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256).amax(-1) / 448
                assert ((st[name + "_scale"][i].double() - top).abs() <= 16 * U * top + 1e-40).all()
                _check_codes(st[name][i], st[name + "_scale"][i], x, b, floor)
            base += -(-n // 256) * 256


def test_8_bit_rounding_has_no_bias(device):
    """A constant gradient moves sqrt(v) by far less than a code a step: its mean over many values follows all the
    same, which rounding to the nearest would not."""
    n, steps = 1 << 16, 40
    p = torch.zeros(n, device=device)
    st = dict(step=torch.full((1,), 1000, dtype=torch.int32, device=device), m=[torch.zeros(n, device=device).to(torch.float8_e4m3fn)],
              m_scale=[torch.zeros(n // 256, device=device)], v=[torch.full((n,), 200.0, device=device).to(torch.float8_e4m3fn)],
              v_scale=[torch.full((n // 256,), 1 / 192.0, device=device)])
    st["v"][0].view(torch.uint8)[::256] = torch.full((1,), 448.0, device=device).to(torch.float8_e4m3fn).view(torch.uint8)
    opt = AdamW([p], lr=0.0, betas=(0.0, 0.999), eps=1e-8, weight_decay=0.0, state_bits=8, state=st, key=(1, 2))
    g = torch.zeros(n, device=device)
    g[::256] = 448 / 192.0  # the largest of each 256 stays, and with it the scale
    first = float(st["v"][0].float().view(-1, 256)[:, 1:].mean() * (1 / 192.0))
    for _ in range(steps):
        opt.step([g])
    r = (st["v"][0].float() * st["v_scale"][0].repeat_interleave(256)).view(-1, 256)[:, 1:]
    want = first * 0.999**(steps / 2)
    # 65280 independent values, each of which takes a code's step (1 / 8 of it at most) with a probability
    # below 0.01 a step: five standard deviations of their mean
    assert abs(float(r.mean()) / want - 1) < 5 * 0.125 * math.sqrt(steps * 0.01) / math.sqrt(65280)


def test_mixed_tensors_missing_gradients_and_many(device):
    sizes = [10, 5000, 300] * 40  # more tensors than one launch holds
    p, g = _tensors(device, sizes, 3)
    opt = AdamW(p, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8, min_8bit_size=1000)
    assert opt.state["m"][0].dtype == torch.float32 and opt.state["m"][1].dtype == torch.float8_e4m3fn
    before = [x.clone() for x in p]
    g[3] = g[-1] = None
    g[5] = g[5].bfloat16()
    opt.step(g)
    for i in range(len(sizes)):
        if g[i] is None:
            assert torch.equal(p[i], before[i])
        else:
            z = torch.zeros_like(before[i])
            want = _expected(before[i], g[i], z, z, 1)
            _within(p[i], want[0], want[3])
    assert int(opt.state["step"]) == 1
    opt.step([None] * len(sizes))
    assert int(opt.state["step"]) == 2


def test_not_finite_gradients_stay_where_they_are(device):
    p, g = _tensors(device, [1000], 4)
    g[0] = g[0].abs().clamp(min=1e-3)
    want = _expected(p[0], g[0], torch.zeros_like(p[0]), torch.zeros_like(p[0]), 1)
    g[0][7], g[0][600] = float("nan"), float("inf")
    opt = AdamW(p, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8)
    opt.step(g)
    bad = torch.zeros(1000, dtype=torch.bool, device=device)
    bad[[7, 600]] = True
    for x in (p[0], opt.state["m"][0].float(), opt.state["v"][0].float()):
        assert torch.equal(~torch.isfinite(x), bad)
    _within(p[0][~bad], want[0][~bad], want[3][~bad])


def test_learning_rate_and_scale_on_the_device(device):
    a, g = _tensors(device, [700, 3], 5)
    b = [x.clone() for x in a]
    lr, scale = torch.tensor([LR / 2], device=device), torch.tensor([0.25], device=device)
    one, two = (AdamW(x, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD) for x in (a, b))
    one.step(g, lr=lr, grad_scale=scale)
    two.step([x * 0.25 for x in g], lr=float(lr))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_captured_steps_go_on_counting(device):
    a, g = _tensors(device, [3000, 17], 6)
    b = [x.clone() for x in a]
    kw = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8, key=(5, 6))
    one, two = AdamW(a, **kw), AdamW(b, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one.step(g)
        two.step(g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.step(g)
    for i in range(4):
        for x in g:
            x.mul_(-1.1)
        graph.replay()
        two.step(g)
        torch.cuda.synchronize()
        assert int(one.state["step"]) == i + 2 and int(one._ticket) == 0
        for x, y in zip(a + one.state["m"] + one.state["v"] + one.state["m_scale"], b + two.state["m"] + two.state["v"] + two.state["m_scale"]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_states_travel_and_memory_may_be_exchanged(device):
    a, g = _tensors(device, [500, 1300], 7)
    b = [x.clone() for x in a]
    kw = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8)
    one, two = AdamW(a, **kw), AdamW(b, **kw)
    one.step(g)
    for x, y in zip(b, a):
        x.copy_(y)
    two.load_state_dict({k: v.clone() if isinstance(v, torch.Tensor) else [x.clone() for x in v] for k, v in one.state_dict().items()})
    two.params[0].data = two.params[0].data.clone()  # other memory, the same values
    one.step(g)
    two.step(g)
    for x, y in zip(a, two.params):
        assert torch.equal(x, y)
    with pytest.raises(L.PDError, match="sizes or bits"):
        two.load_state_dict(AdamW([x.clone() for x in a], **{**kw, "state_bits": 32}).state_dict())


def test_refusals(device):
    p, g = _tensors(device, [64, 8], 8)
    for bad in (p + [p[0]], p + [p[0][3:9]], [p[0].bfloat16()], [p[0][::2]], [p[0], p[1].cpu()]):
        with pytest.raises(L.PDError):
            AdamW(bad)
    with pytest.raises(L.PDError, match="copies"):
        AdamW(p, copies=[None])
    with pytest.raises(L.PDError, match="copy 0"):
        AdamW(p, copies=[p[0].clone(), None])
    opt = AdamW(p)
    with pytest.raises(L.PDError, match="state"):
        AdamW(p, state={**opt.state, "m": opt.state["m"][:1]})
    with pytest.raises(L.PDError):
        AdamW(p, state_bits=8, state=opt.state)
    half = torch.zeros(64, dtype=torch.bfloat16, device=device)
    for kw in (dict(copies=[half, half[:8]]), dict(state={**opt.state, "v": opt.state["m"]}),
               dict(state={**opt.state, "m": [p[0], opt.state["m"][1]]})):
        with pytest.raises(L.PDError, match="share memory"):
            AdamW(p, **kw)
    for bad in (g[:1], [g[0][:5], g[1]], [g[0].double(), g[1]], [g[0].cpu(), g[1]]):
        with pytest.raises(L.PDError):
            opt.step(bad)
    with pytest.raises(L.PDError, match="lr"):
        opt.step(g, lr=torch.tensor([1.0]))
    assert int(opt.state["step"]) == 0


def test_saved_tensors_notice_the_step(device):
    p = torch.randn(8, device=device, requires_grad=True)
    loss = (p * p).sum()
    AdamW([p]).step([torch.ones_like(p)])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


@pytest.mark.parametrize("lr, wd", [(1e-3, 1e-2), (1e-6, 1e-2), (1e-7, 1e-1)])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_small_decay_is_not_lost(device, lr, wd, bits):
    """lr * decay below the spacing of fp32 at 1, against the step in 64 bits rounded once. The update is off by 32 2^-24
    of itself, which moves the mean of the rounded values by as much, and a value that lies so close to a border
    becomes its neighbour, a step of 2^-23 (p in [1, 2)) up or down: five standard deviations of the mean if all did. (A mean of
    uniform roundings is not what to compare with: at lr 1e-7 updates are below a step, and p' follows them in steps.)"""
    n = 1 << 20
    g = torch.Generator(device=device).manual_seed(1)
    p = 1 + torch.rand(n, device=device, generator=g)
    grad = torch.randn(n, device=device, generator=g) * (0.5 + torch.rand(n, device=device, generator=g))
    before = p.double()
    opt = AdamW([p], lr=lr, betas=(B1, B2), eps=0.5, weight_decay=wd, state_bits=bits)
    opt.step([grad])
    update = lr * grad.double() / (grad.double().abs() + 0.5)
    off = (p.double() - (before - lr * wd * before - update).float().double()).mean()
    tol = 32 * U * update.abs().mean() + 5 * 2.0**-23 / math.sqrt(n)
    assert tol < 0.2 * lr * wd * before.mean()  # what is lost would show
    assert abs(off) <= tol, (float(off), float(tol))


@pytest.mark.parametrize("size", [1e-19, 1e-20, 1e-21])
def test_roots_of_subnormal_squares(device, size):
    """v below fp32's normal numbers and an eps below its root: the step goes by the root of the v that is stored."""
    n = 3000
    p = torch.zeros(n, device=device)
    g = torch.Generator(device=device).manual_seed(2)
    grad = (1 + torch.rand(n, device=device, generator=g)) * size
    opt = AdamW([p], lr=LR, betas=(B1, B2), eps=2.0**-126, weight_decay=0.0)
    opt.step([grad])
    m, v = opt.state["m"][0].double(), opt.state["v"][0].double()
    assert (v > 0).all() and (v < 2.0**-100).all()
    want = -LR * (m / (1 - B1)) / ((v / (1 - B2)).sqrt() + 2.0**-126)
    _within(p, want, 32 * U * want.abs())


def test_tensors_that_are_exchanged_are_those_that_the_steps_use(device):
    sizes, kw = [300, 5000], dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8, min_8bit_size=1000, key=(3, 4))
    a, g = _tensors(device, sizes, 9)
    b = [x.clone() for x in a]
    half = lambda: [torch.empty(n, dtype=torch.bfloat16, device=device) for n in sizes]  # noqa: E731
    one, two = AdamW(a, copies=half(), **kw), AdamW(b, copies=half(), **kw)
    for opt in (one, two):
        opt.step(g)
    own = lambda t: None if t is None else t.clone()  # noqa: E731
    old = [x.clone() for x in two.params]
    kept = [(x, own(x)) for k in ("m", "v", "m_scale", "v_scale") for x in two.state[k]] + [(x, own(x)) for x in two.copies]
    first = two.params[0]
    two.params[0] = first.clone()
    for k in ("m", "v", "m_scale", "v_scale"):
        two.state[k] = [own(x) for x in two.state[k]]  # another list
    two.state["m"][0] = two.state["m"][0].clone()       # another tensor of it
    two.state["v"][1].data = two.state["v"][1].data.clone()
    two.state["step"] = two.state["step"].clone()
    two.copies[1] = two.copies[1].clone()
    for opt in (one, two):
        opt.step(g)
    assert torch.equal(first, old[0])
    for x, y in kept[:-2] + kept[-1:]:
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    for x, y in zip(one.params + one.copies, two.params + two.copies):
        assert torch.equal(x, y)
    for k in ("m", "v", "m_scale", "v_scale"):
        for x, y in zip(one.state[k], two.state_dict()[k]):
            assert (x is None) == (y is None) and (x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8)))
    assert int(two.state["step"]) == 2


def test_exchanged_tensors_are_checked(device):
    sizes, kw = [2000, 600], dict(state_bits=8, min_8bit_size=1000)
    p, g = _tensors(device, sizes, 10)
    other = torch.zeros(40, dtype=torch.int32, device=device)

    def make():
        return AdamW([x.clone() for x in p], copies=[torch.zeros(n, dtype=torch.bfloat16, device=device) for n in sizes], **kw)

    def shrink(t):
        t.data = t.data[:t.numel() // 2]

    for change in (lambda o: shrink(o.params[0]), lambda o: shrink(o.state["m"][0]), lambda o: shrink(o.state["v"][1]),
                   lambda o: shrink(o.state["m_scale"][0]), lambda o: shrink(o.copies[1]),
                   lambda o: o.state["m"].__setitem__(0, o.state["m"][0][:1000]), lambda o: o.state["v"].__setitem__(0, torch.zeros(2000, device=device)),
                   lambda o: o.state["v_scale"].__setitem__(0, None), lambda o: o.state["m"].pop(), lambda o: o.copies.pop(),
                   lambda o: o.copies.__setitem__(0, o.copies[0].float()), lambda o: o.params.pop(), lambda o: o.params.__setitem__(1, p[0]),
                   lambda o: o.params.__setitem__(0, None), lambda o: o.state["v"].__setitem__(0, None), lambda o: o.copies.clear(),
                   lambda o: o.state.update(step=other[:2]), lambda o: o.state.update(step=torch.zeros(1, device=device)),
                   lambda o: o.state["m"].__setitem__(1, o.state["v"][1]), lambda o: o.state.update(v=o.state["m"]),
                   lambda o: o.params[0].__setattr__("data", o.params[0].data.cpu()), lambda o: o.copies.__setitem__(0, o.copies[0].cpu())):
        opt = make()
        opt.step(g)
        before = [x.clone() for x in opt.params]
        change(opt)
        with pytest.raises(L.PDError):
            opt.step(g)
        for x, y in zip(before[1:], opt.params[1:]):
            assert x.shape != y.shape or torch.equal(x, y)


def test_states_without_scales_travel(device):
    """States of 32 bits may come without lists of scales and in any shape, and go to optimizers that have them flat."""
    a, g = _tensors(device, [30, 40, 50], 11)
    b = [x.clone() for x in a]
    plain = dict(step=torch.zeros(1, dtype=torch.int32, device=device), m=[torch.zeros_like(x).view(5, -1) for x in a],
                 v=[torch.zeros_like(x) for x in a])
    one, two = AdamW(a, state=plain), AdamW(b)
    one.step(g)
    for x, y in zip(b, a):
        x.copy_(y)
    two.load_state_dict(one.state_dict())
    one.step(g)
    two.step(g)
    one.load_state_dict(two.state_dict())
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    eight = AdamW([x.clone() for x in a], state_bits=8)
    for opt, state in ((one, eight.state), (eight, one.state)):
        with pytest.raises(L.PDError, match="sizes or bits"):
            opt.load_state_dict(state)


def test_parameters_and_copies_may_become_tuples(device):
    a, g = _tensors(device, [30, 40], 12)
    opt = AdamW(a, copies=[None, torch.empty(40, dtype=torch.bfloat16, device=device)])
    opt.params, opt.copies, opt.state = tuple(x.clone() for x in a), tuple(opt.copies), dict(opt.state, m=tuple(opt.state["m"]))
    before = [x.clone() for x in a]
    opt.step(g)
    assert all(torch.equal(x, y) for x, y in zip(a, before)) and not any(torch.equal(x, y) for x, y in zip(a, opt.params))
    assert torch.equal(opt.copies[1], opt.params[1].bfloat16())
