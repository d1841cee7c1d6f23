"""Argument checks of the streamed cross entropy, AdamW, routing by scores and the residual norms:
every call here is refused before anything is launched (CPU tensors or host pointers throughout)."""

import ctypes
import os

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fw

from param_decomp_amd import _lib as L
from param_decomp_amd import losses, ops
from param_decomp_amd.norms import residual_norm, rms_norm
from param_decomp_amd.optim import AdamW
from param_decomp_amd.routed import experts

BF16, F32 = torch.bfloat16, torch.float32
needs_library = pytest.mark.skipif(not os.path.exists(L.LIB_PATH), reason="HIP library not built")


def _ce(N=4, d=16, V=9, dt=BF16):
    return torch.zeros(N, d, dtype=dt), torch.zeros(V, d, dtype=dt), torch.zeros(N, dtype=torch.int64)


@pytest.mark.parametrize("change, message", [
    (lambda a, h, t: (a[0], h, t), "act \\[N, d\\]"),
    (lambda a, h, t: (a, h[:, :8], t), "act \\[N, d\\]"),
    (lambda a, h, t: (a, h, t[:3]), "targets"),
    (lambda a, h, t: (a, h.float(), t), "share one dtype"),
    (lambda a, h, t: (a.half(), h.half(), t), "share one dtype"),
    (lambda a, h, t: (a, h, t.float()), "int32 or int64"),
    (lambda a, h, t: (a[:, :12].contiguous(), h[:, :12].contiguous(), t), "multiple of 8"),
    (lambda a, h, t: (a, h[:0], t), "V >= 1"),
    (lambda a, h, t: (a, h, t), "GPU tensors"),
])
def test_cross_entropy_refuses(change, message):
    args = change(*_ce())
    for call in (ops.streamed_cross_entropy_fwd, lambda *a: ops.streamed_cross_entropy(*a, want_dact=True),
                 lambda *a: ops.streamed_cross_entropy_bwd(*a, torch.zeros(4, 2), torch.zeros(4))):
        with pytest.raises(L.PDError, match=message):
            call(*args)


def test_cross_entropy_refuses_weights_and_statistics():
    a, h, t = _ce()
    with pytest.raises(L.PDError, match="row_weight"):
        ops.streamed_cross_entropy(a, h, t, row_weight=torch.zeros(3), want_dact=True)
    with pytest.raises(L.PDError, match="row_weight"):
        ops.streamed_cross_entropy(a, h, t, row_weight=torch.zeros(4, dtype=torch.float64))
    with pytest.raises(L.PDError, match="GPU tensors"):
        ops.streamed_cross_entropy_bwd(a, h, t, torch.zeros(4, 3), torch.zeros(4))
    with pytest.raises(L.PDError, match="targets are"):
        losses.streamed_position_cross_entropy(a[None], h, t)


@needs_library
def test_cross_entropy_entry_points_refuse():
    b = np.zeros(64, np.float32).ctypes.data
    lib = L.load()
    ok = dict(dtype=L.BF16, N=4, d=16, V=9, bits=64)

    def fwd(ws=2**62, **kw):
        c = {**ok, **kw}
        return lib.pd_streamed_ce_fwd(c["dtype"], c["N"], c["d"], c["V"], b, b, b, c["bits"], -100, b, None, b, ws, None)

    for kw, rc in ((dict(dtype=5), 3), (dict(d=12), 3), (dict(V=0), 1), (dict(N=-1), 1), (dict(bits=16), 1),
                   (dict(N=(1 << 21) + 1), 3), (dict(V=1 << 24), 3), (dict(N=1 << 20, d=1024), 3),
                   (dict(ws=16), 4)):
        assert fwd(**kw) == rc, kw
    assert fwd(N=0) == 0
    size = lib.pd_streamed_ce_train_workspace_size
    assert size(L.BF16, 4, 16, 9, 1, 1) > 0 and size(L.BF16, 0, 16, 9, 1, 1) == 0
    kept = lib.pd_streamed_ce_kept_size
    assert kept(L.BF16, 4, 16, 9) > 0 and kept(L.BF16, 0, 16, 9) == 0 and kept(L.F32, 8192, 16, 131072) == 0
    assert 8192 * 50277 * 2 <= kept(L.BF16, 8192, 768, 50277) < 1 << 30 and kept(L.BF16, 1 << 18, 16, 131072) == 0
    a = (b, b, b, 64, -100)
    assert lib.pd_streamed_ce_kept_fwd(L.F32, 8192, 16, 131072, *a, b, b, 2**62, b, 2**62, None) == 3  # nothing is kept
    assert lib.pd_streamed_ce_kept_fwd(L.BF16, 4, 16, 9, *a, b, b, 16, b, 2**62, None) == 4
    assert lib.pd_streamed_ce_kept_fwd(L.BF16, 4, 16, 9, *a, b, b, 2**62, b, 16, None) == 4
    assert lib.pd_streamed_ce_kept_fwd(L.BF16, 0, 16, 9, *a, b, b, 2**62, b, 2**62, None) == 1
    assert lib.pd_streamed_ce_kept_bwd(L.BF16, 4, 16, 9, *a, b, 16, b, b, b, b, 2**62, None) == 4
    assert lib.pd_streamed_ce_kept_bwd(L.BF16, 4, 16, 9, *a, b, 2**62, None, b, b, b, 2**62, None) == 1
    # the softmax of a chunk, not of all positions: below 2 GiB and what goes with it
    assert size(L.BF16, 1 << 18, 16, 131072, 1, 1) < (3 << 30)


def _route(T=4, E=8):
    return torch.zeros(T, E)


@pytest.mark.parametrize("kw, message", [
    (dict(k=0), "chosen"), (dict(k=9), "chosen"), (dict(k=2, n_groups=3), "groups"),
    (dict(k=2, n_groups=4, top_groups=5), "groups"), (dict(k=2, n_groups=4, top_groups=0), "groups"),
    (dict(k=5, n_groups=4, top_groups=2), "groups"), (dict(k=2, scoring="tanh"), "scoring"),
    (dict(k=2, scale=float("inf")), "scale"), (dict(k=2, bias=torch.zeros(7)), "bias"),
    (dict(k=2, bias=torch.zeros(8, dtype=BF16)), "bias"), (dict(k=2), "GPU tensors"),
])
def test_route_scores_refuses(kw, message):
    with pytest.raises(L.PDError, match=message):
        experts.route_scores(_route(), **kw)


def test_route_scores_refuses_logits():
    for x in (_route().half(), _route()[0], _route(E=1025), torch.zeros(4, 0), _route()[None]):
        with pytest.raises(L.PDError):
            experts.route_scores(x, 1)
    with pytest.raises(L.PDError, match="top_idx"):
        ops.route_scores_bwd(_route(), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2))
    with pytest.raises(L.PDError, match="top_idx"):
        ops.route_scores_bwd(_route(), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 3))


@needs_library
def test_route_scores_entry_points_refuse():
    b = np.zeros(64, np.float32).ctypes.data
    f = L.load().pd_route_scores_fwd
    args = lambda **k: [b, k.get("dt", 0), k.get("T", 4), k.get("E", 8), k.get("k", 2), 0, None, k.get("g", 1),  # noqa: E731
                        k.get("top", 1), 1, k.get("scale", 1.0), k.get("w", b), b, None]
    for kw, rc in ((dict(dt=2), 3), (dict(T=-1), 1), (dict(T=1 << 26), 3), (dict(k=9), 1), (dict(E=2000), 3), (dict(E=100, k=65), 3),
                   (dict(g=3), 1), (dict(g=8, top=1), 1), (dict(scale=float("nan")), 1), (dict(w=None), 1)):
        assert f(*args(**kw)) == rc, kw
    assert f(*args(T=0)) == 0


@needs_library
def test_route_scores_entry_points_refuse_grids_that_a_launch_does_not_take():
    b = np.zeros(64, np.float32).ctypes.data
    lib, T = L.load(), (1 << 26) - 3
    for E in (8, 300, 1024):
        assert lib.pd_route_scores_fwd(b, 0, T, E, 2, 0, None, 1, 1, 1, 1.0, b, b, None) == 3
        assert lib.pd_route_scores_bwd(b, 0, T, E, 2, 0, 1, 1.0, b, b, b, None) == 3


X = torch.zeros(6, 8)


@pytest.mark.parametrize("args, kw, message", [
    ((X, X[:5]), {}, "branch is"), ((X.half(), X.half()), {}, "stream and branch"), ((X.bfloat16(), X), {}, "stream and branch"),
    ((X, X), dict(pre_weight=torch.ones(7)), "pre_weight"), ((X, X), dict(post_weight=torch.ones(8, dtype=BF16)), "post_weight"),
    ((X, X), dict(post_norm=False, post_weight=torch.ones(8)), "without the branch's norm"),
    ((X, X), dict(gate=torch.ones(4, 8)), "gate"), ((X, X), dict(gate=torch.ones(7)), "gate"),
    ((X, X), dict(gate=torch.ones(6, 8).half()), "gate"), ((X, X), dict(scale=float("nan")), "scale"),
    ((X.view(2, 3, 8), X.view(2, 3, 8)), dict(gate=torch.ones(3, 8)), "leading axes"),  # of the second axis
    ((X.view(2, 3, 8), X.view(2, 3, 8)), dict(gate=torch.ones(1, 3, 8)), "leading axes"),
    ((torch.zeros(2, 16385), torch.zeros(2, 16385)), {}, "16384"), ((X, X), {}, "GPU tensors"),
])
def test_residual_norm_refuses(args, kw, message):
    with pytest.raises(L.PDError, match=message):
        residual_norm(*args, **kw)


def test_rms_norm_refuses():
    for call in (lambda: rms_norm(X.half()), lambda: rms_norm(X, torch.ones(7)), lambda: rms_norm(X.bfloat16(), dtype=F32),
                 lambda: rms_norm(X)):
        with pytest.raises(L.PDError):
            call()


@needs_library
def test_residual_norm_entry_points_refuse():
    b = np.zeros(64, np.float32).ctypes.data
    f = L.load().pd_residual_norm_fwd
    args = lambda **k: [k.get("x", b), k.get("xd", 0), b, k.get("bd", 0), k.get("rows", 6), k.get("d", 8),  # noqa: E731
                        k.get("post", 1), k.get("w"), k.get("gate"), k.get("gd", 0), k.get("gr", 0), 1.0, None, 0.0,
                        k.get("eps", 1e-6), b, b, None, None]
    for kw, rc in ((dict(xd=1), 3), (dict(bd=2), 3), (dict(rows=-1), 1), (dict(d=0), 1), (dict(d=16392), 3),
                   (dict(gate=b, gr=4), 1), (dict(gate=b, gr=0), 1), (dict(gate=b, gr=6, gd=2), 3), (dict(eps=-1.0), 1),
                   (dict(eps=float("inf")), 1), (dict(x=None), 1), (dict(post=0, w=b), 1)):
        assert f(*args(**kw)) == rc, kw
    assert f(*args(rows=0, x=None)) == 0


@needs_library
def test_adamw_entry_point_refuses():
    one = (ctypes.c_void_p * 1)(np.zeros(64, np.float32).ctypes.data)
    sizes, types = (ctypes.c_int64 * 1)(64), (ctypes.c_int32 * 1)(0)
    b = one[0]

    def step(n=1, sizes=sizes, p=one, g=one, types=types, m=one, v=one, ms=None, vs=None, count=b, ticket=b, lr=1e-3,
             betas=(0.9, 0.99), eps=1e-8, wd=0.0):
        return L.load().pd_adamw_step(n, sizes, p, g, types, m, v, ms, vs, None, count, ticket, lr, None, None, *betas, eps, wd,
                                      0, 0, None)

    null = (ctypes.c_void_p * 1)(None)
    for kw in (dict(n=-1), dict(p=None), dict(count=None), dict(ticket=None), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
               dict(eps=0.0), dict(eps=1e-60), dict(eps=1e-40), dict(eps=1e39), dict(lr=float("nan")), dict(wd=float("inf")), dict(p=null), dict(m=null),
               dict(ms=one), dict(sizes=(ctypes.c_int64 * 1)(-1))):
        assert step(**kw) == 1, kw
    assert step(types=(ctypes.c_int32 * 1)(2)) == 3


def test_adamw_refuses():
    p = torch.zeros(4, 4)
    for call in (lambda: AdamW([]), lambda: AdamW([p], state_bits=16), lambda: AdamW([p])):
        with pytest.raises(L.PDError):
            call()


def _calls(device):
    """(call, its differentiable inputs) of each operator."""
    x, w = torch.randn(4, 16, device=device), torch.ones(16, device=device)
    t = torch.zeros(4, dtype=torch.int64, device=device)
    return [
        (lambda a, h: losses.streamed_position_cross_entropy(a, h, t), [x, x[:3].clone()]),
        (lambda a, h: losses.streamed_cross_entropy(a, h, t), [x, x[:3].clone()]),
        (lambda z: experts.route_scores(z, 2)[0], [x]),
        (lambda x, b, p, g, q: residual_norm(x, b, post_weight=p, gate=g, pre_weight=q)[1], [x, x.clone(), w, w.clone(), w.clone()]),
        (lambda x, q: rms_norm(x, q), [x, w]),
    ]


def _refuse_tangents(device):
    for call, inputs in _calls(device):
        for i, t in enumerate(inputs):
            for grad in (True, False):
                with fw.dual_level(), torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="jvp"):
                    call(*inputs[:i], fw.make_dual(t, torch.ones_like(t)), *inputs[i + 1:])
        with fw.dual_level():  # no tangent, no refusal
            assert call(*inputs).grad_fn is None
        leaf = inputs[0].detach().clone().requires_grad_()
        assert call(leaf, *inputs[1:]).grad_fn is not None
        with torch.no_grad():
            assert call(leaf, *inputs[1:]).grad_fn is None


def test_tangents_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "streamed_cross_entropy_kept_fwd", lambda *a, **k: (None, None))
    monkeypatch.setattr(ops, "streamed_cross_entropy_fwd", lambda a, h, t, ignore_index=0, want_stats=False:
                        (a.new_zeros(4), a.new_zeros(4, 2)))
    monkeypatch.setattr(ops, "route_scores_fwd", lambda z, k, **kw: (z.new_zeros(4, k), torch.zeros(4, k, dtype=torch.int32)))
    monkeypatch.setattr(ops, "residual_norm_fwd", lambda x, b=None, **kw: (torch.zeros_like(x), torch.zeros_like(x), x.new_zeros(1)))
    _refuse_tangents("cpu")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_gpu(device):
    _refuse_tangents(device)
