"""Argument checks of packed attention, layer norm and the top-logits KL: every call here is
refused before anything is launched (CPU tensors or host pointers throughout)."""

import ctypes
import os

import numpy as np
import pytest
import torch

from param_decomp_amd import _lib as L
from param_decomp_amd import losses, ops
from param_decomp_amd.attention import packed_attention
from param_decomp_amd.norms import layer_norm

BF16, F32 = torch.bfloat16, torch.float32


def _qkv(N=6, H=4, KV=2, D=16, dt=BF16):
    return torch.zeros(N, H, D, dtype=dt), torch.zeros(N, KV, D, dtype=dt), torch.zeros(N, KV, D, dtype=dt)


OFF = torch.tensor([0, 2, 6], dtype=torch.int32)


@pytest.mark.parametrize("change, message", [
    (lambda q, k, v: (q, k, v[:, :1], OFF), "kv heads"),
    (lambda q, k, v: (q, k[:5], v[:5], OFF), "kv heads"),
    (lambda q, k, v: (q[0], k, v, OFF), "kv heads"),
    (lambda q, k, v: (q, k.float(), v, OFF), "share one dtype"),
    (lambda q, k, v: (q.half(), k.half(), v.half(), OFF), "share one dtype"),
    (lambda q, k, v: (q[:, :3], k, v, OFF), "no multiple"),
    (lambda q, k, v: (q[:, :0], k, v, OFF), "no multiple"),
    (lambda q, k, v: (q, k, v, OFF.long()), "int32 vector"),
    (lambda q, k, v: (q, k, v, OFF[:0]), "int32 vector"),
    (lambda q, k, v: (q, k, v, OFF[::2]), "int32 vector"),
    (lambda q, k, v: (q, k, v, OFF[None]), "int32 vector"),
])
def test_attention_refuses(change, message):
    args = change(*_qkv())
    with pytest.raises(L.PDError, match=message):
        ops.packed_attention_fwd(*args)
    with pytest.raises(L.PDError, match=message):
        packed_attention(*args)


def test_attention_refuses_head_widths():
    for D in (12, 136, 256):
        with pytest.raises(L.PDError, match="head_dim"):
            ops.packed_attention_fwd(*_qkv(D=D), OFF)
    with pytest.raises(L.PDError, match="head_dim"):
        packed_attention(*_qkv(D=136), OFF)


def test_attention_refuses_strides():
    wide = torch.zeros(6, 4, 32, dtype=BF16)
    _, k, v = _qkv()
    for q in (wide[..., ::2], torch.zeros(6, 4, 20, dtype=BF16)[..., :16], wide.flatten()[1:1 + 6 * 64].view(6, 4, 16)):
        with pytest.raises(L.PDError, match="dense last axis"):
            ops._strides("packed_attention_fwd", "q", q)
    assert ops._strides("packed_attention_fwd", "q", wide[..., 16:]) == (128, 32)
    # one row or one head: its stride is never used
    assert ops._strides("packed_attention_fwd", "q", torch.zeros(3, 1, 16, dtype=BF16)[1:2]) == (16, 16)


def test_attention_backward_refuses():
    q, k, v = _qkv()
    stats = torch.zeros(4, 6)
    with pytest.raises(L.PDError, match="d_out"):
        ops.packed_attention_bwd(q, k, v, OFF, q, (stats, q), q.float())
    with pytest.raises(L.PDError, match="stats"):
        ops.packed_attention_bwd(q, k, v, OFF, q, (stats[:, :5], q), q)
    with pytest.raises(L.PDError, match="out_rest"):
        ops.packed_attention_bwd(q, k, v, OFF, q, (stats, None), q)
    with pytest.raises(L.PDError, match="out is"):
        ops.packed_attention_bwd(q, k, v, OFF, q[:, :2], (stats, q), q)


def test_layer_norm_refuses():
    x, w = torch.zeros(3, 8, dtype=BF16), torch.ones(8)
    for args, message in (((x.half(),), "float32 or bfloat16"), ((x, w.to(BF16)), "weight is float32"),
                          ((x, w[:7]), "weight is float32"), ((x, w, w[None]), "bias is float32"),
                          ((x[:, :0],), "no last axis"), ((x[0, 0],), "no last axis")):
        with pytest.raises(L.PDError, match=message):
            ops.layer_norm_fwd(*args)
        with pytest.raises(L.PDError, match=message):
            layer_norm(*args)
    with pytest.raises(L.PDError, match="d_y"):
        ops.layer_norm_bwd(x, x.float(), w, torch.zeros(3, 3))
    with pytest.raises(L.PDError, match="stats"):
        ops.layer_norm_bwd(x, x, w, torch.zeros(3, 2))


def test_top_logits_kl_refuses():
    z, t, i = torch.zeros(3, 10, dtype=BF16), torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int32)
    lse = torch.zeros(3)
    for kw, message in ((dict(z=z.half()), "float32 or bfloat16"), (dict(t=t.half()), "float32 or bfloat16"),
                        (dict(i=i.to(torch.int16)), "int32 or int64"), (dict(i=i[:, :3]), "top logits and indices"),
                        (dict(t=t[:2], i=i[:2]), "top logits and indices"),
                        (dict(t=t[:, :0], i=i[:, :0]), "top logits and indices"),
                        (dict(t=torch.zeros(3, 1025), i=torch.zeros(3, 1025, dtype=torch.int32)), "k <= 1024"),
                        (dict(z=z[:, :0]), "2\\^19"), (dict(z=torch.zeros(3, (1 << 19) + 1, dtype=BF16)), "2\\^19"),
                        (dict(clean_lse=lse[:2]), "clean_lse"), (dict(clean_lse=lse.double()), "clean_lse"),
                        (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
                        (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature")):
        kw = dict(kw)
        a = [kw.pop(n, d) for n, d in (("z", z), ("t", t), ("i", i))]
        with pytest.raises(L.PDError, match=message):
            ops.top_logits_kl(*a, **kw)
        with pytest.raises(L.PDError, match=message):
            losses.top_logits_kl(*a, **kw)
    with pytest.raises(L.PDError, match="row_weight"):
        ops.top_logits_kl(z, t, i, row_weight=lse[:, None])


def test_cpu_tensors_are_refused():
    with pytest.raises(L.PDError, match="GPU tensors"):
        packed_attention(*_qkv(), OFF)
    with pytest.raises(L.PDError, match="GPU tensors"):
        layer_norm(torch.zeros(3, 8))
    with pytest.raises(L.PDError, match="GPU tensors"):
        losses.top_logits_position_kl(torch.zeros(3, 8), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64))


built = pytest.mark.skipif(not os.path.exists(L.LIB_PATH), reason="HIP library not built")


def _buffer():
    raw = np.zeros(4096, np.uint8)
    return raw, (raw.ctypes.data + 63) // 64 * 64


@built
@pytest.mark.parametrize("kw, message", [
    (dict(dtype=2), "dtype"), (dict(H=3), "multiple of n_kv_head"), (dict(KV=0), "multiple of n_kv_head"),
    (dict(D=12), "head_dim"), (dict(D=0), "head_dim"), (dict(D=136), "head_dim"), (dict(rows=-1), ">= 0"),
    (dict(n_seq=-1), ">= 0"), (dict(rows=1 << 31), "too many"), (dict(n_seq=1 << 31), "too many"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q_row=1), "strides"),
    (dict(v_head=4), "strides"), (dict(q_row=1 << 23), "row strides"), (dict(q_row=-64), "row strides"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(off=None), "offsets"),
    (dict(shift=8), "aligned"),
])
def test_attention_entry_points_refuse(kw, message):
    keep, p = _buffer()
    d = dict(dtype=1, rows=4, H=4, KV=2, D=16, n_seq=1, scale=1.0, q=p, out=p, off=p, q_row=64, v_head=16, shift=0)
    d.update(kw)
    q = None if d["q"] is None else d["q"] + d["shift"]
    head = [q, d["q_row"], 16, p, 32, 16, p, 32, d["v_head"], d["dtype"], d["rows"], d["H"], d["KV"], d["D"], d["off"],
            d["n_seq"], d["scale"], 1]
    with pytest.raises(L.PDError, match=message):
        L.call("pd_packed_attention_fwd", *head, d["out"], None, p, None)
    with pytest.raises(L.PDError, match=message):
        L.call("pd_packed_attention_bwd", *head, d["out"], p, p, p, p, p, p, p, 1 << 30, None)


@built
def test_entry_points_refuse_workspaces_and_stats():
    keep, p = _buffer()
    head = [p, 64, 16, p, 32, 16, p, 32, 16, 1, 4, 4, 2, 16, p, 1, 1.0, 1]
    need = L.load().pd_packed_attention_bwd_workspace_size(4, 4, 2, 16)
    assert need == 4 * 4 * 4 + 2 * 2 * 4 * 2 * 16 * 4  # D of every row; dk and dv of two shares of the heads
    assert L.load().pd_packed_attention_bwd_workspace_size(65536, 4, 4, 16) == 65536 * 4 * 4
    with pytest.raises(L.PDError, match="workspace"):
        L.call("pd_packed_attention_bwd", *head, p, p, p, p, p, p, p, p, need - 1, None)
    with pytest.raises(L.PDError, match="workspace"):
        L.call("pd_packed_attention_bwd", *head, p, p, p, p, p, p, p, None, need, None)
    with pytest.raises(L.PDError, match="stats"):
        L.call("pd_packed_attention_bwd", *head, p, p, None, p, p, p, p, p, need, None)
    with pytest.raises(L.PDError, match="out_rest"):
        L.call("pd_packed_attention_bwd", *head, p, None, p, p, p, p, p, p, need, None)
    head[9] = 0
    with pytest.raises(L.PDError, match="out_rest"):
        L.call("pd_packed_attention_fwd", *head, p, p, p, None)
    need = L.load().pd_layer_norm_bwd_workspace_size(4, 8)
    with pytest.raises(L.PDError, match="workspace"):
        L.call("pd_layer_norm_bwd", p, p, 1, 4, 8, None, p, p, p, None, p, need - 1, None)
    assert L.load().pd_layer_norm_bwd_workspace_size(0, 8) == 0


@built
def test_norm_and_kl_entry_points_refuse():
    keep, p = _buffer()
    for args, message in (((p, 2, 4, 8), "dtype"), ((p, 1, -1, 8), "rows"), ((p, 1, 4, 0), "rows"),
                          ((None, 1, 4, 8), "null"), ((p, 1, 1 << 31, 8), "too large")):
        with pytest.raises(L.PDError, match=message):
            L.call("pd_layer_norm_fwd", *args, None, None, 1e-5, p, None, None)
        with pytest.raises(L.PDError, match=message):
            L.call("pd_layer_norm_bwd", args[0], p, *args[1:], None, p, p, None, None, None, 0, None)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(L.PDError, match="eps"):
            L.call("pd_layer_norm_fwd", p, 1, 4, 8, None, None, eps, p, None, None)

    def kl(z=p, dtype=1, rows=2, V=10, top_dtype=0, bits=32, k=3, tau=1.0, out=p, ws=p):
        L.call("pd_top_kl", z, dtype, rows, V, p, top_dtype, p, bits, k, None, tau, None, out, None, ws, 64, None)

    for kw, message in ((dict(dtype=2), "fp32 or bf16"), (dict(top_dtype=2), "fp32 or bf16"), (dict(bits=16), "indices"),
                        (dict(rows=-1), "rows"), (dict(V=0), "vocab"), (dict(k=0), "k >= 1"), (dict(k=1025), "1024"),
                        (dict(V=(1 << 19) + 1), "2\\^19"), (dict(tau=0.0), "temperature"),
                        (dict(tau=float("nan")), "temperature"), (dict(z=None), "null"), (dict(out=None), "null"),
                        (dict(ws=None), "workspace"), (dict(ws=p + 8), "workspace"), (dict(rows=3), "workspace"),
                        (dict(rows=1 << 31), "rows")):
        with pytest.raises(L.PDError, match=message):
            kl(**kw)


@built
def test_no_rows_is_no_launch():
    """Without rows nothing is read, written or launched (no GPU is needed)."""
    L.call("pd_packed_attention_fwd", *[None, 64, 16] * 3, 1, 0, 4, 2, 16, None, 0, 1.0, 1, None, None, None, None)
    L.call("pd_packed_attention_bwd", *[None, 64, 16] * 3, 1, 0, 4, 2, 16, None, 0, 1.0, 1, *[None] * 8, 0, None)
    L.call("pd_layer_norm_fwd", None, 1, 0, 8, None, None, 1e-5, None, None, None)
    L.call("pd_top_kl", None, 1, 0, 10, None, 0, None, 32, 3, None, 1.0, None, None, None, None, 0, None)
    assert ctypes.sizeof(ctypes.c_size_t) == 8
