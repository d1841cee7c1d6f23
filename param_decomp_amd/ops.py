"""Tensor-level wrappers over the C ABI: shape checks, output allocation, streams.

Each function maps one-to-one onto an `include/pd_mi355x.h` entry point. Higher-level
modules (`masking`, `decomposed_linear`, `losses`, `routed.experts`) add autograd.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

from param_decomp_amd import _lib as L
from param_decomp_amd.prng import Key


def _flat_rows(t: torch.Tensor) -> tuple[int, int]:
    return int(math.prod(t.shape[:-1])), int(t.shape[-1])


def uniform(key: Key, shape, draw_dtype: torch.dtype, device, *, out_dtype: torch.dtype | None = None,
            layout: int = L.LAYOUT_PARTITIONABLE) -> torch.Tensor:
    out = torch.empty(tuple(shape), dtype=out_dtype or draw_dtype, device=device)
    L.call("pd_uniform", key[0], key[1], out.numel(), L.dtype_code(draw_dtype), layout, L.ptr(out),
           L.dtype_code(out.dtype), L.stream())
    return out


def squash_fwd(pre: torch.Tensor, lower: bool = True, upper: bool = True):
    lo = torch.empty_like(pre) if lower else None
    up = torch.empty_like(pre) if upper else None
    L.call("pd_squash_fwd", L.ptr(pre), L.dtype_code(pre.dtype), pre.numel(), L.ptr(lo), L.ptr(up), L.stream())
    return lo, up


def squash_bwd(pre, g_lower, g_upper):
    d = torch.empty_like(pre)
    L.call("pd_squash_bwd", L.ptr(pre), L.ptr(g_lower), L.ptr(g_upper), L.dtype_code(pre.dtype), pre.numel(),
           L.ptr(d), L.stream())
    return d


def _device_key(key) -> bool:
    """A key given as a device tensor of two 32-bit words (read when the kernel runs: the
    form a captured graph replays with fresh keys) rather than a host pair."""
    if isinstance(key, torch.Tensor):
        if key.dtype not in (torch.int32, torch.uint32) or key.numel() != 2 or not key.is_cuda:
            raise L.PDError("a device key is a CUDA tensor of two 32-bit words")
        return True
    return False


def component_mask_fwd(ci, key, draw_dtype: torch.dtype, layout=L.LAYOUT_PARTITIONABLE):
    m = torch.empty_like(ci)
    if _device_key(key):
        L.call("pd_component_mask_fwd_dkey", L.ptr(ci), L.dtype_code(ci.dtype), ci.numel(), L.ptr(key),
               L.dtype_code(draw_dtype), layout, L.ptr(m), L.stream())
    else:
        L.call("pd_component_mask_fwd", L.ptr(ci), L.dtype_code(ci.dtype), ci.numel(), key[0], key[1],
               L.dtype_code(draw_dtype), layout, L.ptr(m), L.stream())
    return m


def component_mask_bwd(g_mask, key, draw_dtype: torch.dtype, layout=L.LAYOUT_PARTITIONABLE):
    d = torch.empty_like(g_mask)
    if _device_key(key):
        L.call("pd_component_mask_bwd_dkey", L.ptr(g_mask), L.dtype_code(g_mask.dtype), g_mask.numel(), L.ptr(key),
               L.dtype_code(draw_dtype), layout, L.ptr(d), L.stream())
    else:
        L.call("pd_component_mask_bwd", L.ptr(g_mask), L.dtype_code(g_mask.dtype), g_mask.numel(), key[0], key[1],
               L.dtype_code(draw_dtype), layout, L.ptr(d), L.stream())
    return d


def gate_fwd(h, w_in, b_in, w_out, b_out, precise: bool):
    rows, C = _flat_rows(h)
    g = torch.empty(h.shape, dtype=torch.float32, device=h.device)
    L.call("pd_gate_fwd", L.ptr(h), L.dtype_code(h.dtype), rows, C, w_in.shape[1], L.ptr(w_in), L.ptr(b_in),
           L.ptr(w_out), L.ptr(b_out), int(precise), L.ptr(g), L.stream())
    return g


def gate_bwd(h, w_in, b_in, w_out, b_out, dg_raw, precise: bool):
    rows, C = _flat_rows(h)
    H = w_in.shape[1]
    dh = torch.empty_like(h)
    dwi, dbi, dwo = torch.empty_like(w_in), torch.empty_like(b_in), torch.empty_like(w_out)
    dbo = torch.empty_like(b_out)
    lib = L.load()
    ws = L.workspace(lib.pd_gate_bwd_workspace_size(rows, C, H), h.device)
    L.call("pd_gate_bwd", L.ptr(h), L.dtype_code(h.dtype), rows, C, H, L.ptr(w_in), L.ptr(b_in), L.ptr(w_out),
           L.ptr(b_out), L.ptr(dg_raw.contiguous()), int(precise), L.ptr(dh), L.ptr(dwi), L.ptr(dbi), L.ptr(dwo),
           L.ptr(dbo), L.ptr(ws), ws.numel(), L.stream())
    return dh, dwi, dbi, dwo, dbo


def impmin(ci_upper, *, kind: int, p=1.0, eps=0.0, beta=0.0, world_size=1.0, gamma=1.0, normalize_at_one=False,
           ref_count=0.0, coeff_act=1.0, coeff_freq=0.0, want_grad=False, ema=None, ema_out=None, ema_count=0.0,
           ema_halflife=0.0):
    """out[0] = activity, out[1] = frequency penalty, out[2] = the batch penalty when
    `ema` (the fp32 [C] estimate before this batch) is given; `ema_out` receives the new
    estimate (may be `ema` itself)."""
    rows, C = _flat_rows(ci_upper)
    out = torch.zeros(3, dtype=torch.float32, device=ci_upper.device)
    grad = torch.empty_like(ci_upper) if want_grad else None
    ws = L.workspace(L.load().pd_impmin_workspace_size(rows, C), ci_upper.device)
    L.call("pd_impmin", L.ptr(ci_upper), L.dtype_code(ci_upper.dtype), rows, C, kind, p, eps, beta, world_size, gamma,
           int(normalize_at_one), ref_count, L.ptr(ema), L.ptr(ema_out), float(ema_count), float(ema_halflife),
           coeff_act, coeff_freq, L.ptr(out), L.ptr(grad), L.ptr(ws), ws.numel(), L.stream())
    return out, grad


def mse(a, b, coeff=1.0, want_grad=False):
    out = torch.empty(1, dtype=torch.float32, device=a.device)
    grad = torch.empty_like(a) if want_grad else None
    ws = L.workspace(L.load().pd_mse_workspace_size(a.numel()), a.device)
    L.call("pd_mse", L.ptr(a), L.ptr(b), L.dtype_code(a.dtype), a.numel(), coeff, L.ptr(out), L.ptr(grad), L.ptr(ws),
           ws.numel(), L.stream())
    return out, grad


def kl(masked_logits, clean_logits, coeff=1.0, want_grad=False):
    rows, V = _flat_rows(masked_logits)
    out = torch.empty(1, dtype=torch.float32, device=masked_logits.device)
    grad = torch.empty_like(masked_logits) if want_grad else None
    ws = L.workspace(L.load().pd_kl_workspace_size(rows), masked_logits.device)
    L.call("pd_kl", L.ptr(masked_logits), L.ptr(clean_logits), L.dtype_code(masked_logits.dtype), rows, V, coeff,
           L.ptr(out), L.ptr(grad), L.ptr(ws), ws.numel(), L.stream())
    return out, grad


def gemm(a: torch.Tensor, b: torch.Tensor, *, trans_a=False, trans_b=False, out: torch.Tensor | None = None,
         out_dtype: torch.dtype | None = None, alpha=1.0, beta=0.0) -> torch.Tensor:
    """`alpha * op(a) @ op(b) + beta * out` for 2-D row-major tensors."""
    M = a.shape[1] if trans_a else a.shape[0]
    K = a.shape[0] if trans_a else a.shape[1]
    N = b.shape[0] if trans_b else b.shape[1]
    Kb = b.shape[1] if trans_b else b.shape[0]
    if K != Kb:
        raise L.PDError(f"gemm shape mismatch {tuple(a.shape)} {tuple(b.shape)}")
    if a.dtype != b.dtype:
        raise L.PDError("gemm operands must share a dtype")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or a.dtype, device=a.device)
    L.call("pd_gemm", L.dtype_code(a.dtype), M, N, K, L.ptr(a), a.shape[1], int(trans_a), L.ptr(b), b.shape[1],
           int(trans_b), L.ptr(out), N, L.dtype_code(out.dtype), alpha, beta, L.stream())
    return out


def route_uniform_k(key: Key, n_sites: int, n_positions: int, device, layout: int = L.LAYOUT_PARTITIONABLE):
    routes = torch.empty((n_sites, n_positions), dtype=torch.uint8, device=device)
    L.call("pd_route_uniform_k", key[0], key[1], n_positions, n_sites, layout, L.ptr(routes), L.stream())
    return routes


def route_static_p(key: Key, n_sites: int, p: float, n_positions: int, device, layout: int = L.LAYOUT_PARTITIONABLE):
    routes = torch.empty((n_sites, n_positions), dtype=torch.uint8, device=device)
    L.call("pd_route_static_p", key[0], key[1], n_positions, n_sites, p, layout, L.ptr(routes), L.stream())
    return routes


def router_topk(logits: torch.Tensor, k: int):
    T, E = logits.shape
    probs = torch.empty_like(logits)
    idx = torch.empty((T, k), dtype=torch.int32, device=logits.device)
    w = torch.empty((T, k), dtype=torch.float32, device=logits.device)
    L.call("pd_router_topk", L.ptr(logits), T, E, k, L.ptr(probs), L.ptr(idx), L.ptr(w), L.stream())
    return probs, idx, w


def routed_jobs(top_idx: torch.Tensor, n_experts: int):
    T, k = top_idx.shape
    n = T * k
    dev = top_idx.device
    sort_idx = torch.empty(n, dtype=torch.int32, device=dev)
    inv = torch.empty(n, dtype=torch.int32, device=dev)
    sizes = torch.empty(n_experts, dtype=torch.int32, device=dev)
    offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    ws = L.workspace(L.load().pd_routed_jobs_workspace_size(n, n_experts), dev)
    L.call("pd_routed_jobs", L.ptr(top_idx), T, k, n_experts, L.ptr(sort_idx), L.ptr(inv), L.ptr(sizes),
           L.ptr(offsets), L.ptr(ws), ws.numel(), L.stream())
    return sort_idx, inv, sizes, offsets


def gather_rows(src: torch.Tensor, idx: torch.Tensor, div: int) -> torch.Tensor:
    out = torch.empty((idx.numel(), src.shape[-1]), dtype=src.dtype, device=src.device)
    L.call("pd_gather_rows", L.ptr(src), L.dtype_code(src.dtype), src.shape[-1], L.ptr(idx), div, idx.numel(),
           L.ptr(out), L.stream())
    return out


def combine_jobs(y: torch.Tensor, inv: torch.Tensor, weights: torch.Tensor | None, T: int, k: int) -> torch.Tensor:
    out = torch.empty((T, y.shape[-1]), dtype=y.dtype, device=y.device)
    L.call("pd_combine_jobs", L.ptr(y), L.dtype_code(y.dtype), y.shape[-1], L.ptr(inv), L.ptr(weights), T, k,
           L.ptr(out), L.stream())
    return out


def grouped_gemm(lhs, rhs, offsets, *, trans_rhs=False, out_dtype=None):
    J, K = lhs.shape
    E = rhs.shape[0]
    N = rhs.shape[1] if trans_rhs else rhs.shape[2]
    out = torch.empty((J, N), dtype=out_dtype or lhs.dtype, device=lhs.device)
    L.call("pd_grouped_gemm", L.ptr(lhs), L.ptr(rhs), L.ptr(offsets), J, E, K, N, int(trans_rhs), L.ptr(out),
           L.dtype_code(out.dtype), L.stream())
    return out


def grouped_gemm_dw_kmajor(lhsT, doutT, offsets, n_groups: int, *, out_dtype=None):
    """`out[e] = lhsT[:, rows_e] @ doutT[:, rows_e]^T` from job-contiguous operands."""
    K, J = lhsT.shape
    N = doutT.shape[0]
    out = torch.empty((n_groups, K, N), dtype=out_dtype or lhsT.dtype, device=lhsT.device)
    L.call("pd_grouped_gemm_dw_kmajor", L.ptr(lhsT), L.ptr(doutT), L.ptr(offsets), J, n_groups, K, N, L.ptr(out),
           L.dtype_code(out.dtype), L.stream())
    return out


def grouped_gemm_dw(lhs, dout, offsets, n_groups: int, *, out_dtype=None):
    J, K = lhs.shape
    N = dout.shape[1]
    out = torch.empty((n_groups, K, N), dtype=out_dtype or lhs.dtype, device=lhs.device)
    L.call("pd_grouped_gemm_dw", L.ptr(lhs), L.ptr(dout), L.ptr(offsets), J, n_groups, K, N, L.ptr(out),
           L.dtype_code(out.dtype), L.stream())
    return out


def ci_mlp_fwd(x: torch.Tensor, weights, biases):
    """SiteMLP preactivations of bf16 `x` [..., d_0] with bf16 weights[i] [d_i, d_i+1] and
    biases[i] [d_i+1]. Returns (preact [..., d_n], workspace); the workspace holds the
    hidden activations and feeds `ci_mlp_bwd`."""
    rows, d0 = _flat_rows(x)
    dims = [d0] + [w.shape[1] for w in weights]
    for i, w in enumerate(weights):
        if w.shape[0] != dims[i] or biases[i].shape != (dims[i + 1],):
            raise L.PDError(f"ci_mlp layer {i}: weight {tuple(w.shape)} / bias {tuple(biases[i].shape)} mismatch")
    cdims = L.host_array(ctypes.c_int64, dims)
    out = torch.empty((*x.shape[:-1], dims[-1]), dtype=torch.bfloat16, device=x.device)
    ws = L.workspace(L.load().pd_ci_mlp_workspace_size(len(weights), cdims, rows), x.device)
    L.call("pd_ci_mlp_fwd", len(weights), cdims, rows, L.ptr(x), L.host_array(ctypes.c_void_p, map(L.ptr, weights)),
           L.host_array(ctypes.c_void_p, map(L.ptr, biases)), L.ptr(out), L.ptr(ws), ws.numel(), L.stream())
    return out, ws


def ci_mlp_bwd(x: torch.Tensor, weights, d_preact: torch.Tensor, ws: torch.Tensor, want_dx: bool):
    """Gradients of `ci_mlp_fwd` from bf16 `d_preact`, reusing its workspace: fp32
    d_weights and d_biases, and bf16 d_x (None unless asked)."""
    rows, d0 = _flat_rows(x)
    dims = [d0] + [w.shape[1] for w in weights]
    cdims = L.host_array(ctypes.c_int64, dims)
    dW = [torch.empty(w.shape, dtype=torch.float32, device=x.device) for w in weights]
    db = [torch.empty(w.shape[1], dtype=torch.float32, device=x.device) for w in weights]
    dx = torch.empty_like(x) if want_dx else None
    L.call("pd_ci_mlp_bwd", len(weights), cdims, rows, L.ptr(x), L.host_array(ctypes.c_void_p, map(L.ptr, weights)),
           L.ptr(d_preact), L.host_array(ctypes.c_void_p, map(L.ptr, dW)), L.host_array(ctypes.c_void_p, map(L.ptr, db)),
           L.ptr(dx), L.ptr(ws), ws.numel(), L.stream())
    return dW, db, dx


def ci_readout_fwd(h: torch.Tensor, params: torch.Tensor, base: torch.Tensor | None = None) -> torch.Tensor:
    """Component-activation readout of bf16 `h` [..., C] with fp32 params [7, C], added to
    bf16 `base` when given."""
    rows, C = _flat_rows(h)
    if params.shape != (7, C) or params.dtype != torch.float32:
        raise L.PDError("readout params must be fp32 [7, C]")
    out = torch.empty_like(h)
    L.call("pd_ci_readout_fwd", rows, C, L.ptr(h), L.ptr(params), L.ptr(base), L.ptr(out), L.stream())
    return out


def ci_readout_bwd(h: torch.Tensor, params: torch.Tensor, d_out: torch.Tensor, want_dh: bool = True):
    rows, C = _flat_rows(h)
    d_h = torch.empty_like(h) if want_dh else None
    d_params = torch.empty((7, C), dtype=torch.float32, device=h.device)
    ws = L.workspace(L.load().pd_ci_readout_workspace_size(rows, C), h.device)
    L.call("pd_ci_readout_bwd", rows, C, L.ptr(h), L.ptr(params), L.ptr(d_out), L.ptr(d_h), L.ptr(d_params), L.ptr(ws),
           ws.numel(), L.stream())
    return d_h, d_params


def faithfulness_fwd(W, V, U, w_sq_norms, mats_per_site: int, scale: float, keep_delta: bool):
    """Stacked faithfulness forward: W [n, d_out, d_in] (bf16/fp32), V fp32 [n, d_in, C],
    U fp32 [n, C, d_out], w_sq_norms fp32 [n / mats_per_site]. Returns (loss [1],
    site_errors, delta or None)."""
    n, d_out, d_in = W.shape
    C = V.shape[-1]
    if V.shape != (n, d_in, C) or U.shape != (n, C, d_out) or V.dtype != torch.float32 or U.dtype != torch.float32:
        raise L.PDError(f"faithfulness shapes: W {tuple(W.shape)} V {tuple(V.shape)} U {tuple(U.shape)} (fp32 V/U)")
    dev = W.device
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    site_err = torch.empty(n // mats_per_site, dtype=torch.float32, device=dev)
    delta = torch.empty((n, d_out, d_in), dtype=torch.float32, device=dev) if keep_delta else None
    ws = L.workspace(L.load().pd_faithfulness_workspace_size(n, d_in, d_out, C), dev)
    L.call("pd_faithfulness_fwd", n, mats_per_site, d_in, d_out, C, L.ptr(W), L.dtype_code(W.dtype), L.ptr(V), L.ptr(U),
           L.ptr(w_sq_norms), scale, L.ptr(loss), L.ptr(site_err), L.ptr(delta), L.ptr(ws), ws.numel(), L.stream())
    return loss, site_err, delta


def faithfulness_bwd(delta, V, U, w_sq_norms, mats_per_site: int, scale: float, d_loss: torch.Tensor | None):
    n, d_out, d_in = delta.shape
    C = V.shape[-1]
    dV = torch.empty_like(V)
    dU = torch.empty_like(U)
    L.call("pd_faithfulness_bwd", n, mats_per_site, d_in, d_out, C, L.ptr(delta), L.ptr(V), L.ptr(U), L.ptr(w_sq_norms),
           scale, L.ptr(d_loss), L.ptr(dV), L.ptr(dU), L.stream())
    return dV, dU


def masked_linear_fwd(x, V, U, mask, W=None, delta=None):
    """`pd_masked_linear_fwd` without route: (out, xV, acts) with acts = xV * (mask - delta)
    and, with a delta [T], out = acts @ U + delta * (x @ W^T)."""
    T, d_in = x.shape
    C, d_out = U.shape
    out = torch.empty((T, d_out), dtype=x.dtype, device=x.device)
    xV = torch.empty((T, C), dtype=x.dtype, device=x.device)
    acts = torch.empty((T, C), dtype=x.dtype, device=x.device)
    L.call("pd_masked_linear_fwd", L.dtype_code(x.dtype), T, d_in, d_out, C, L.ptr(x), L.ptr(V), L.ptr(U), L.ptr(W),
           L.ptr(mask), L.ptr(delta), None, L.ptr(out), L.ptr(xV), L.ptr(acts), L.stream())
    return out, xV, acts


def masked_linear_bwd(x, V, U, mask, xV, acts, g_out, *, W=None, delta=None, want_dx=False, want_dvu=True,
                      want_dmask=True, want_ddelta=False):
    """`pd_masked_linear_bwd` without route; each output optional. Returns
    (dx, dV, dU, dmask, d_delta); d_delta [T] needs W."""
    T, d_in = x.shape
    C, d_out = U.shape
    dx = torch.empty_like(x) if want_dx else None
    dV = torch.empty_like(V) if want_dvu else None
    dU = torch.empty_like(U) if want_dvu else None
    dm = torch.empty_like(mask) if want_dmask else None
    dd = torch.empty((T,), dtype=x.dtype, device=x.device) if want_ddelta else None
    dt = L.dtype_code(x.dtype)
    ws = L.workspace(L.load().pd_masked_linear_bwd_workspace_size(dt, T, d_out, C), x.device)
    L.call("pd_masked_linear_bwd", dt, T, d_in, d_out, C, L.ptr(x), L.ptr(V), L.ptr(U), L.ptr(W), L.ptr(mask),
           L.ptr(delta), None, L.ptr(xV), L.ptr(acts), L.ptr(g_out), L.ptr(dx), L.ptr(dV), L.ptr(dU), L.ptr(dm),
           L.ptr(dd), L.ptr(ws), ws.numel(), L.stream())
    return dx, dV, dU, dm, dd


def source_mask_fwd(ci, sources, rows_per_source: int):
    """m = ci + (1 - ci) s for ci [rows, C] and sources [rows / rows_per_source, C]."""
    rows, C = _flat_rows(ci)
    mask = torch.empty_like(ci)
    L.call("pd_source_mask_fwd", L.ptr(ci), L.dtype_code(ci.dtype), rows, C, L.ptr(sources),
           L.dtype_code(sources.dtype), rows_per_source, L.ptr(mask), L.stream())
    return mask


def source_mask_bwd(g_mask, ci, sources, rows_per_source: int, want_dci: bool = False):
    rows, C = _flat_rows(ci)
    d_src = torch.empty((rows // rows_per_source, C), dtype=torch.float32, device=ci.device)
    d_ci = torch.empty_like(ci) if want_dci else None
    ws = L.workspace(L.load().pd_source_mask_bwd_workspace_size(rows, C, rows_per_source), ci.device)
    L.call("pd_source_mask_bwd", L.ptr(g_mask), L.ptr(ci), L.dtype_code(ci.dtype), rows, C, L.ptr(sources),
           L.dtype_code(sources.dtype), rows_per_source, L.ptr(d_src), L.ptr(d_ci), L.ptr(ws), ws.numel(), L.stream())
    return d_src, d_ci


def source_ascend(opt: int, sources, grad, state_a=None, state_b=None, *, step_count=0.0, lr=1.0, beta1=0.9,
                  beta2=0.999, eps=1e-8, momentum=0.0, key: Key = (0, 0), layout: int = L.LAYOUT_PARTITIONABLE):
    """One projected ascent of `sources` in place (see pd_source_ascend)."""
    L.call("pd_source_ascend", opt, L.dtype_code(sources.dtype), sources.numel(), L.ptr(sources), L.ptr(grad),
           L.ptr(state_a), L.ptr(state_b), step_count, lr, beta1, beta2, eps, momentum, key[0], key[1], layout,
           L.stream())
    return sources

# ------------------------------------------------- around a language model's decomposed sites
def differentiated(*tensors: torch.Tensor | None) -> bool:
    """Whether a call on these has to go through its autograd function: one of them needs a
    gradient, or carries a forward-mode tangent (which the functions refuse; past them it
    would be lost without a word)."""
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and ((grad and t.requires_grad) or forward_ad.unpack_dual(t).tangent is not None):
            return True
    return False


def _one_device(name: str, first: torch.Tensor, labels: str, *others: torch.Tensor | None) -> torch.device:
    """The first tensor's device, which the others (named in `labels`) have to share."""
    device = first.device
    for i, t in enumerate(others):
        if t is not None and t.device != device:
            raise L.PDError(f"{name}: {labels.split()[i]} is on {t.device}, not {device}")
    if device.type != "cuda":
        raise L.PDError("pd kernels take GPU tensors")
    return device


def _strides(name: str, label: str, t: torch.Tensor) -> tuple[int, int]:
    """Row and head strides of [rows, heads, head_dim] as the attention kernels take them."""
    rows, heads, D = t.shape
    per = 16 // t.element_size()
    row = t.stride(0) if rows > 1 else heads * D
    head = t.stride(1) if heads > 1 else D
    if (D > 1 and t.stride(2) != 1) or row % per or head % per or t.data_ptr() % 16 or row * t.element_size() > 1 << 23:
        raise L.PDError(f"{name}: {label} needs a dense last axis and 16-byte aligned rows (8 MiB apart at most) and heads")
    return row, head


def _attention_checks(name: str, q, k, v, offsets, scale):
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise L.PDError(f"{name}: q [rows, heads, head_dim], k and v [rows, kv heads, head_dim], got "
                        f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in (torch.float32, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise L.PDError(f"{name}: q, k and v share one dtype, float32 or bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise L.PDError(f"{name}: {q.shape[1]} query heads are no multiple of {k.shape[1]} key heads")
    if q.shape[2] % 8 or not 8 <= q.shape[2] <= 128:
        raise L.PDError(f"{name}: head_dim is a multiple of 8 up to 128, got {q.shape[2]}")
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.numel() < 1 or not offsets.is_contiguous():
        raise L.PDError(f"{name}: offsets is a dense int32 vector of sequences + 1 row numbers")
    return q.shape[2]**-0.5 if scale is None else float(scale)


def _attention_args(name: str, q, k, v, offsets, scale: float, fill: bool) -> list:
    N, H, D = q.shape
    args = []
    for label, t in (("q", q), ("k", k), ("v", v)):
        args += [t.data_ptr(), *_strides(name, label, t)]
    return args + [L.dtype_code(q.dtype), N, H, k.shape[1], D, L.ptr(offsets), offsets.numel() - 1, scale, int(fill)]


def _stats_shape(q: torch.Tensor) -> tuple:
    return (2, q.shape[1], q.shape[0])


def _like_rows(name: str, label: str, t: torch.Tensor, q: torch.Tensor) -> torch.Tensor:
    if t.shape != q.shape or t.dtype != q.dtype:
        raise L.PDError(f"{name}: {label} is {tuple(t.shape)} {t.dtype}, not {tuple(q.shape)} {q.dtype}")
    return t


def packed_attention_fwd(q, k, v, offsets, *, scale: float | None = None, out: torch.Tensor | None = None,
                         want_saved: bool = False):
    """(out, saved) of causal attention over packed sequences: q [rows, H, head_dim], k and v
    [rows, KV, head_dim] (strided views will do), sequence s in rows offsets[s] ..
    offsets[s + 1] (int32, on the device). `scale`: head_dim^-0.5 by default. Rows of no
    sequence are zeros, or left as they were in an `out` that is given. saved: what the
    backward takes, (stats, out_rest), None unless wanted."""
    name = "packed_attention_fwd"
    scale = _attention_checks(name, q, k, v, offsets, scale)
    device = _one_device(name, q, "k v offsets out", k, v, offsets, out)
    fill = out is None
    out = torch.empty(q.shape, dtype=q.dtype, device=device) if fill else _like_rows(name, "out", out, q)
    stats = rest = None
    if want_saved:
        stats = torch.empty(_stats_shape(q), dtype=torch.float32, device=device)
        rest = torch.empty(q.shape, dtype=q.dtype, device=device) if q.dtype == torch.bfloat16 else None
    L.launch("pd_packed_attention_fwd", device, *_attention_args(name, q, k, v, offsets, scale, fill), L.ptr(out),
             L.ptr(rest), L.ptr(stats))
    return out, (stats, rest) if want_saved else None


def packed_attention_bwd(q, k, v, offsets, out, saved, d_out, *, scale: float | None = None):
    """(dq, dk, dv) from the forward's inputs, `out` and `saved`; zeros in rows of no
    sequence."""
    name = "packed_attention_bwd"
    scale = _attention_checks(name, q, k, v, offsets, scale)
    _like_rows(name, "out", out, q)
    _like_rows(name, "d_out", d_out, q)
    stats, rest = saved
    if (rest is None) != (q.dtype == torch.float32):
        raise L.PDError(f"{name}: the forward saves out_rest for bfloat16")
    if stats.dtype != torch.float32 or tuple(stats.shape) != _stats_shape(q):
        raise L.PDError(f"{name}: saved stats are the forward's, float32 {_stats_shape(q)}")
    if rest is not None:
        _like_rows(name, "out_rest", rest, q)
    device = _one_device(name, q, "k v offsets out stats out_rest d_out", k, v, offsets, out, stats, rest, d_out)
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v))
    ws = L.workspace(L.load().pd_packed_attention_bwd_workspace_size(q.shape[0], q.shape[1], k.shape[1], q.shape[2]),
                     device)
    L.launch("pd_packed_attention_bwd", device, *_attention_args(name, q, k, v, offsets, scale, True), L.ptr(out),
             L.ptr(rest), L.ptr(stats), L.ptr(d_out), L.ptr(dq), L.ptr(dk), L.ptr(dv), L.ptr(ws), ws.numel())
    return dq, dk, dv


def _norm_checks(name: str, x, weight, bias=None) -> tuple[int, int]:
    if x.dim() < 1 or x.shape[-1] == 0:
        raise L.PDError(f"{name}: x has no last axis to norm: {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise L.PDError(f"{name}: x is float32 or bfloat16, got {x.dtype}")
    for label, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (x.shape[-1],)):
            raise L.PDError(f"{name}: {label} is float32 [{x.shape[-1]}], got {t.dtype} {tuple(t.shape)}")
    return _flat_rows(x)


def layer_norm_fwd(x, weight=None, bias=None, *, eps: float = 1e-5, want_stats: bool = False):
    """(y, stats) over the last axis; stats fp32 [rows, 3] for the backward, None unless
    wanted."""
    rows, d = _norm_checks("layer_norm_fwd", x, weight, bias)
    device = _one_device("layer_norm_fwd", x, "weight bias", weight, bias)
    y = torch.empty_like(x)
    stats = torch.empty((rows, 3), dtype=torch.float32, device=device) if want_stats else None
    L.launch("pd_layer_norm_fwd", device, L.ptr(x), L.dtype_code(x.dtype), rows, d, L.ptr(weight), L.ptr(bias), eps,
             L.ptr(y), L.ptr(stats))
    return y, stats


def layer_norm_bwd(x, d_y, weight, stats, *, want_dx: bool = True, want_dweight: bool = True, want_dbias: bool = True):
    """(dx, dweight, dbias) from the forward's input and stats; None for those not wanted."""
    name = "layer_norm_bwd"
    rows, d = _norm_checks(name, x, weight)
    if d_y.shape != x.shape or d_y.dtype != x.dtype:
        raise L.PDError(f"{name}: d_y is {tuple(d_y.shape)} {d_y.dtype}, not {tuple(x.shape)} {x.dtype}")
    if stats.dtype != torch.float32 or tuple(stats.shape) != (rows, 3):
        raise L.PDError(f"{name}: stats is the forward's, float32 [rows, 3]")
    device = _one_device(name, x, "d_y weight stats", d_y, weight, stats)
    dx = torch.empty_like(x) if want_dx else None
    dw, db = (torch.empty(d, dtype=torch.float32, device=device) if want else None for want in (want_dweight, want_dbias))
    params = want_dweight or want_dbias
    ws = L.workspace(L.load().pd_layer_norm_bwd_workspace_size(rows, d), device) if params else None
    L.launch("pd_layer_norm_bwd", device, L.ptr(x), L.ptr(d_y), L.dtype_code(x.dtype), rows, d, L.ptr(weight),
             L.ptr(stats), L.ptr(dx), L.ptr(dw), L.ptr(db), L.ptr(ws), ws.numel() if params else 0)
    return dx, dw, db


def top_logits_kl(masked_logits, top_logits, top_indices, *, clean_lse=None, temperature: float = 1.0,
                  row_weight=None, want_kl: bool = True, want_grad: bool = False):
    """(kl, grad): per-position KL from the clean side's listed logits to the masked logits
    [..., V] (see `losses.top_logits_position_kl`), and row_weight (fp32 [...]; None: 1)
    times its gradient, from one read of the logits. None for those not wanted."""
    name = "top_logits_kl"
    z = masked_logits
    lead, V = z.shape[:-1], z.shape[-1] if z.dim() else 0
    if z.dtype not in (torch.float32, torch.bfloat16) or top_logits.dtype not in (torch.float32, torch.bfloat16):
        raise L.PDError(f"{name}: logits are float32 or bfloat16, got {z.dtype} and {top_logits.dtype}")
    if top_indices.dtype not in (torch.int32, torch.int64):
        raise L.PDError(f"{name}: indices are int32 or int64, got {top_indices.dtype}")
    k = top_logits.shape[-1] if top_logits.dim() else 0
    if top_logits.shape[:-1] != lead or top_indices.shape != top_logits.shape or not 1 <= k <= 1024:
        raise L.PDError(f"{name}: top logits and indices are [..., k], 1 <= k <= 1024, beside logits [..., V]; got "
                        f"{tuple(top_logits.shape)}, {tuple(top_indices.shape)}, {tuple(z.shape)}")
    if not 1 <= V <= 1 << 19:
        raise L.PDError(f"{name}: 1 to 2^19 logits a position, got {V}")
    for label, t in (("clean_lse", clean_lse), ("row_weight", row_weight)):
        if t is not None and (t.dtype != torch.float32 or t.shape != lead):
            raise L.PDError(f"{name}: {label} is float32 {tuple(lead)}, got {t.dtype} {tuple(t.shape)}")
    if not (math.isfinite(temperature) and temperature > 0):
        raise L.PDError(f"{name}: temperature must be positive and finite, got {temperature}")
    device = _one_device(name, z, "top_logits top_indices clean_lse row_weight", top_logits, top_indices, clean_lse,
                         row_weight)
    kl = torch.empty(lead, dtype=torch.float32, device=device) if want_kl else None
    grad = torch.empty_like(z) if want_grad else None
    rows = math.prod(lead)
    ws = L.workspace(L.load().pd_top_kl_workspace_size(rows, k), device) if want_kl else None
    if want_kl or want_grad:
        L.launch("pd_top_kl", device, L.ptr(z), L.dtype_code(z.dtype), rows, V, L.ptr(top_logits),
                 L.dtype_code(top_logits.dtype), L.ptr(top_indices), 8 * top_indices.element_size(), k,
                 L.ptr(clean_lse), temperature, L.ptr(row_weight), L.ptr(kl), L.ptr(grad), L.ptr(ws),
                 ws.numel() if want_kl else 0)
    return kl, grad


def route_scores_fwd(logits, k: int, *, sigmoid: bool = False, bias=None, n_groups: int = 1, top_groups: int = 1,
                     renormalize: bool = True, scale: float = 1.0):
    """(weights fp32 [T, k], top_idx int32 [T, k]) of logits [T, E], see `routed.experts.route_scores`."""
    name = "route_scores_fwd"
    T, E = _route_checks(name, logits, k, scale)
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (E,)):
        raise L.PDError(f"{name}: bias is float32 [{E}], got {bias.dtype} {tuple(bias.shape)}")
    if not 1 <= n_groups <= 64 or E % n_groups or not 1 <= top_groups <= n_groups or k > E // n_groups * top_groups:
        raise L.PDError(f"{name}: {top_groups} of {n_groups} equal groups (64 at most) of {E} experts have to hold {k}")
    device = _one_device(name, logits, "bias", bias)
    w = torch.empty((T, k), dtype=torch.float32, device=device)
    idx = torch.empty((T, k), dtype=torch.int32, device=device)
    L.launch("pd_route_scores_fwd", device, L.ptr(logits), L.dtype_code(logits.dtype), T, E, k, int(sigmoid), L.ptr(bias),
             n_groups, top_groups, int(renormalize), scale, L.ptr(w), L.ptr(idx))
    return w, idx


def route_scores_bwd(logits, top_idx, d_weights, *, sigmoid: bool = False, renormalize: bool = True, scale: float = 1.0):
    """d_logits from the forward's logits and choice."""
    name = "route_scores_bwd"
    k = top_idx.shape[-1] if top_idx.dim() else 0
    T, E = _route_checks(name, logits, k, scale)
    if top_idx.dtype != torch.int32 or d_weights.dtype != torch.float32 or tuple(top_idx.shape) != (T, k) or \
            d_weights.shape != top_idx.shape:
        raise L.PDError(f"{name}: top_idx int32 and d_weights float32 are [{T}, k], got {top_idx.dtype} "
                        f"{tuple(top_idx.shape)}, {d_weights.dtype} {tuple(d_weights.shape)}")
    device = _one_device(name, logits, "top_idx d_weights", top_idx, d_weights)
    d = torch.empty_like(logits)
    L.launch("pd_route_scores_bwd", device, L.ptr(logits), L.dtype_code(logits.dtype), T, E, k, int(sigmoid),
             int(renormalize), scale, L.ptr(top_idx), L.ptr(d_weights), L.ptr(d))
    return d


def _route_checks(name: str, logits, k: int, scale: float) -> tuple[int, int]:
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise L.PDError(f"{name}: logits are float32 or bfloat16 [T, E], got {logits.dtype} {tuple(logits.shape)}")
    T, E = logits.shape
    if not 1 <= E <= 1024 or not 1 <= k <= min(E, 64):
        raise L.PDError(f"{name}: up to 1024 experts and 64 of them chosen, got {k} of {E}")
    if not math.isfinite(scale):
        raise L.PDError(f"{name}: scale must be finite, got {scale}")
    return T, E


def _residual_checks(name: str, x, branch, y_dtype, post_norm, post_weight, gate, pre_weight, scale):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 16384:
        raise L.PDError(f"{name}: rows of 1 to 16384 columns, got {tuple(x.shape)}")
    d = x.shape[-1]
    if (x.dtype, y_dtype) not in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                  (torch.float32, torch.bfloat16)):
        raise L.PDError(f"{name}: stream and branch are bfloat16, float32, or a float32 stream with a bfloat16 branch, "
                        f"got {x.dtype}, {y_dtype}")
    if branch is not None and branch.shape != x.shape:
        raise L.PDError(f"{name}: branch is {tuple(branch.shape)}, not {tuple(x.shape)}")
    for label, t in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (d,)):
            raise L.PDError(f"{name}: {label} is float32 [{d}], got {t.dtype} {tuple(t.shape)}")
    if branch is None and (gate is not None or post_weight is not None):
        raise L.PDError(f"{name}: a gate or post_weight without a branch")
    if post_weight is not None and not post_norm:
        raise L.PDError(f"{name}: post_weight without the branch's norm")
    rows = math.prod(x.shape[:-1])
    gate_rows = 0
    if gate is not None:
        gate_rows = math.prod(gate.shape[:-1]) if gate.dim() else 0
        if gate.dtype not in (torch.float32, torch.bfloat16) or gate.dim() < 1 or gate.shape[-1] != d or \
                gate_rows < 1 and rows or gate_rows and rows % gate_rows:
            raise L.PDError(f"{name}: gate is float32 or bfloat16 [..., {d}] whose rows divide the {rows} rows, got "
                            f"{gate.dtype} {tuple(gate.shape)}")
    if not math.isfinite(scale):
        raise L.PDError(f"{name}: scale must be finite, got {scale}")
    return rows, d, gate_rows


def residual_norm_fwd(x, branch=None, *, post_norm: bool = True, post_weight=None, gate=None, pre_weight=None,
                      scale: float = 1.0, weight_offset: float = 0.0, eps: float = 1e-6, y_dtype=None,
                      want_stats: bool = False):
    """(stream, y, stats), see `norms.residual_norm`; stats fp32 [rows, 2] for the backward, None
    unless wanted. Without a branch stream is x itself and y its norm."""
    name = "residual_norm_fwd"
    y_dtype = branch.dtype if branch is not None else y_dtype or x.dtype
    post_norm = post_norm and branch is not None
    rows, d, gate_rows = _residual_checks(name, x, branch, y_dtype, post_norm, post_weight, gate, pre_weight, scale)
    device = _one_device(name, x, "branch post_weight gate pre_weight", branch, post_weight, gate, pre_weight)
    h = x if branch is None else torch.empty_like(x)
    y = torch.empty(x.shape, dtype=y_dtype, device=device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=device) if want_stats else None
    L.launch("pd_residual_norm_fwd", device, L.ptr(x), L.dtype_code(x.dtype), L.ptr(branch), L.dtype_code(y_dtype), rows, d,
             int(post_norm), L.ptr(post_weight), L.ptr(gate), L.dtype_code(gate.dtype) if gate is not None else 0, gate_rows,
             scale, L.ptr(pre_weight), weight_offset, eps, None if branch is None else L.ptr(h), L.ptr(y), L.ptr(stats))
    return h, y, stats


def residual_norm_bwd(stream, branch, stats, d_stream, d_y, *, post_norm: bool = True, post_weight=None, gate=None,
                      pre_weight=None, scale: float = 1.0, weight_offset: float = 0.0, y_dtype=None, want_dx: bool = True,
                      want_dbranch: bool = True, want_dpost: bool = True, want_dgate: bool = True, want_dpre: bool = True):
    """(dx, dbranch, dpost, dgate, dpre) from the forward's stream, branch and stats; None for those
    not wanted. d_stream or d_y None: zero."""
    name = "residual_norm_bwd"
    x = stream
    y_dtype = branch.dtype if branch is not None else y_dtype or x.dtype
    post_norm = post_norm and branch is not None
    rows, d, gate_rows = _residual_checks(name, x, branch, y_dtype, post_norm, post_weight, gate, pre_weight, scale)
    for label, t, dt in (("d_stream", d_stream, x.dtype), ("d_y", d_y, y_dtype)):
        if t is not None and (t.shape != x.shape or t.dtype != dt):
            raise L.PDError(f"{name}: {label} is {tuple(t.shape)} {t.dtype}, not {tuple(x.shape)} {dt}")
    if stats.dtype != torch.float32 or tuple(stats.shape) != (rows, 2):
        raise L.PDError(f"{name}: stats is the forward's, float32 [rows, 2]")
    device = _one_device(name, x, "branch stats d_stream d_y post_weight gate pre_weight", branch, stats, d_stream, d_y,
                         post_weight, gate, pre_weight)
    dx = torch.empty_like(x) if want_dx else None
    db = torch.empty_like(branch) if want_dbranch and branch is not None else None
    # sums over no rows are zero; the entry point writes those of the weights itself
    dg = (torch.zeros_like if not rows else torch.empty_like)(gate) if want_dgate and gate is not None else None
    dpost = torch.empty(d, dtype=torch.float32, device=device) if want_dpost and post_norm else None
    dpre = torch.empty(d, dtype=torch.float32, device=device) if want_dpre else None
    params = dpost is not None or dpre is not None
    nbytes = L.load().pd_residual_norm_bwd_workspace_size(rows, d, gate_rows, int(params), int(dg is not None))
    ws = L.workspace(nbytes, device) if nbytes else None
    L.launch("pd_residual_norm_bwd", device, L.ptr(x), L.dtype_code(x.dtype), L.ptr(branch), L.dtype_code(y_dtype), rows, d,
             int(post_norm), L.ptr(post_weight), L.ptr(gate), L.dtype_code(gate.dtype) if gate is not None else 0, gate_rows,
             scale, L.ptr(pre_weight), weight_offset, L.ptr(stats), L.ptr(d_stream), L.ptr(d_y), L.ptr(dx), L.ptr(db),
             L.ptr(dpost), L.ptr(dg), L.ptr(dpre), L.ptr(ws), ws.numel() if nbytes else 0)
    return dx, db, dpost, dg, dpre


def _ce_checks(name: str, act, head, targets):
    if act.dim() != 2 or head.dim() != 2 or act.shape[1] != head.shape[1] or targets.shape != act.shape[:1]:
        raise L.PDError(f"{name}: act [N, d], head [V, d] and targets [N], got {tuple(act.shape)}, {tuple(head.shape)}, "
                        f"{tuple(targets.shape)}")
    if act.dtype not in (torch.float32, torch.bfloat16) or head.dtype != act.dtype:
        raise L.PDError(f"{name}: act and head share one dtype, float32 or bfloat16, got {act.dtype}, {head.dtype}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise L.PDError(f"{name}: targets are int32 or int64, got {targets.dtype}")
    if head.shape[0] < 1 or head.shape[1] < 1 or (act.dtype == torch.bfloat16 and head.shape[1] % 8):
        raise L.PDError(f"{name}: V >= 1 and d >= 1 (bfloat16: a multiple of 8), got head {tuple(head.shape)}")
    device = _one_device(name, act, "head targets", head, targets)
    N, d = act.shape
    return device, [L.dtype_code(act.dtype), N, d, head.shape[0]]


def _ce_args(act, head, targets, ignore_index: int) -> list:
    return [L.ptr(act), L.ptr(head), L.ptr(targets), 8 * targets.element_size(), int(ignore_index)]


def streamed_cross_entropy_fwd(act, head, targets, *, ignore_index: int = -100, want_stats: bool = False):
    """(loss fp32 [N], stats) of act [N, d] @ head[V, d]^T against targets [N]; stats fp32 [N, 2] for the
    backward, None unless wanted (see `losses.streamed_position_cross_entropy`)."""
    name = "streamed_cross_entropy_fwd"
    device, sizes = _ce_checks(name, act, head, targets)
    loss = torch.empty(act.shape[0], dtype=torch.float32, device=device)
    stats = torch.empty((act.shape[0], 2), dtype=torch.float32, device=device) if want_stats else None
    ws = L.workspace(L.load().pd_streamed_ce_fwd_workspace_size(*sizes), device)
    L.launch("pd_streamed_ce_fwd", device, *sizes, *_ce_args(act, head, targets, ignore_index), L.ptr(loss), L.ptr(stats),
             L.ptr(ws), ws.numel())
    return loss, stats


def streamed_cross_entropy_bwd(act, head, targets, stats, g, *, ignore_index: int = -100, want_dact: bool = True,
                               want_dhead: bool = True):
    """(d_act, d_head) of sum g_i loss_i from the forward's stats, g fp32 [N]; None for those not wanted."""
    name = "streamed_cross_entropy_bwd"
    device, sizes = _ce_checks(name, act, head, targets)
    N = act.shape[0]
    if stats.dtype != torch.float32 or tuple(stats.shape) != (N, 2) or g.dtype != torch.float32 or tuple(g.shape) != (N,):
        raise L.PDError(f"{name}: stats float32 [{N}, 2] and g float32 [{N}], got {stats.dtype} {tuple(stats.shape)}, "
                        f"{g.dtype} {tuple(g.shape)}")
    _one_device(name, act, "stats g", stats, g)
    if not N:
        return torch.empty_like(act) if want_dact else None, torch.zeros_like(head) if want_dhead else None
    da = torch.empty_like(act) if want_dact else None
    dh = torch.empty_like(head) if want_dhead else None
    if want_dact or want_dhead:
        ws = L.workspace(L.load().pd_streamed_ce_bwd_workspace_size(*sizes, int(want_dact)), device)
        L.launch("pd_streamed_ce_bwd", device, *sizes, *_ce_args(act, head, targets, ignore_index), L.ptr(stats), L.ptr(g),
                 L.ptr(da), L.ptr(dh), L.ptr(ws), ws.numel())
    return da, dh


def streamed_cross_entropy_kept_fwd(act, head, targets, *, ignore_index: int = -100):
    """(loss fp32 [N], kept): the forward that leaves the softmax in 16 bits (fp32: the
    logits) for `streamed_cross_entropy_kept_bwd`, which then forms no logits again. kept (2 or 4 bytes for each
    position and entry of the vocabulary) is None where it would take 2 GiB, or a bf16 head does: nothing has run then."""
    name = "streamed_cross_entropy_kept_fwd"
    device, sizes = _ce_checks(name, act, head, targets)
    nbytes = L.load().pd_streamed_ce_kept_size(*sizes)
    if not nbytes:
        return None, None
    loss = torch.empty(act.shape[0], dtype=torch.float32, device=device)
    kept = torch.empty(nbytes, dtype=torch.uint8, device=device)
    ws = L.workspace(L.load().pd_streamed_ce_kept_workspace_size(*sizes, 0, 0), device)
    L.launch("pd_streamed_ce_kept_fwd", device, *sizes, *_ce_args(act, head, targets, ignore_index), L.ptr(loss), L.ptr(kept),
             nbytes, L.ptr(ws), ws.numel())
    return loss, kept


def streamed_cross_entropy_kept_bwd(act, head, targets, kept, g, *, ignore_index: int = -100, want_dact: bool = True,
                                    want_dhead: bool = True):
    """(d_act, d_head) of sum g_i loss_i from what the forward kept, g fp32 [N]; None for those not wanted. The
    workspace is as large as kept again."""
    name = "streamed_cross_entropy_kept_bwd"
    device, sizes = _ce_checks(name, act, head, targets)
    N = act.shape[0]
    if kept.dtype != torch.uint8 or kept.numel() != L.load().pd_streamed_ce_kept_size(*sizes) or not kept.numel():
        raise L.PDError(f"{name}: kept is the forward's, got {kept.dtype} {tuple(kept.shape)}")
    if g.dtype != torch.float32 or tuple(g.shape) != (N,):
        raise L.PDError(f"{name}: g is float32 [{N}], got {g.dtype} {tuple(g.shape)}")
    _one_device(name, act, "kept g", kept, g)
    da = torch.empty_like(act) if want_dact else None
    dh = torch.empty_like(head) if want_dhead else None
    if want_dact or want_dhead:
        ws = L.workspace(L.load().pd_streamed_ce_kept_workspace_size(*sizes, int(want_dact), int(want_dhead)), device)
        L.launch("pd_streamed_ce_kept_bwd", device, *sizes, *_ce_args(act, head, targets, ignore_index), L.ptr(kept),
                 kept.numel(), L.ptr(g), L.ptr(da), L.ptr(dh), L.ptr(ws), ws.numel())
    return da, dh


def streamed_cross_entropy(act, head, targets, *, ignore_index: int = -100, row_weight=None, want_dact: bool = False,
                           want_dhead: bool = False):
    """(loss, d_act, d_head): per-position cross entropy (see `losses.streamed_position_cross_entropy`) and
    row_weight (fp32 [N]; None: 1) times its gradients; None for those not wanted."""
    name = "streamed_cross_entropy"
    N = act.shape[0] if act.dim() else 0
    if row_weight is not None and (row_weight.dtype != torch.float32 or tuple(row_weight.shape) != (N,)):
        raise L.PDError(f"{name}: row_weight is float32 [{N}], got {row_weight.dtype} {tuple(row_weight.shape)}")
    if not (want_dact or want_dhead):
        return streamed_cross_entropy_fwd(act, head, targets, ignore_index=ignore_index)[0], None, None
    device, sizes = _ce_checks(name, act, head, targets)
    if row_weight is None:
        row_weight = torch.ones(N, dtype=torch.float32, device=device)
    _one_device(name, act, "row_weight", row_weight)
    loss = torch.empty(N, dtype=torch.float32, device=device)
    if not N:
        return loss, torch.empty_like(act) if want_dact else None, torch.zeros_like(head) if want_dhead else None
    da = torch.empty_like(act) if want_dact else None
    dh = torch.empty_like(head) if want_dhead else None
    ws = L.workspace(L.load().pd_streamed_ce_train_workspace_size(*sizes, int(want_dact), int(want_dhead)), device)
    L.launch("pd_streamed_ce_train", device, *sizes, *_ce_args(act, head, targets, ignore_index), L.ptr(row_weight),
             L.ptr(loss), L.ptr(da), L.ptr(dh), L.ptr(ws), ws.numel())
    return loss, da, dh
