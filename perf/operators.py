"""The calls that the operators around the decomposed sites of a language-model target are
measured on: causal attention over packed sequences, layer norm, and the KL to a teacher's
top logits.

`listed()` and `draw(rng)` give cases (dicts of plain values), `prepare(case, seed)` what a
program holds before the call, `run(state)` one pass: the framework's calls where `own` is
set, elementary torch operations in 32 bits otherwise. `work(case)` gives the bytes and
operations a pass cannot do without and `exact(case, seed)` its outputs in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
REST_MIN = 2.0**-20  # probability outside the listed logits below this counts as none


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one short request of a few prompts, forward only: latency
        dict(name="attn_small", kind="attn", lengths="17,1,40,5,33", rows=96, H=12, KV=12, D=64, dtype="bf16",
             train=False),
        # a training batch of the 4-layer LM target's size (16 x 512 tokens, 12 heads of 64),
        # documents of different lengths packed, padding behind the last
        dict(name="attn_packed_train", kind="attn", lengths="512,1301,77,900,2048,33,1,640,1500,1117", rows=8192, H=12,
             KV=12, D=64, dtype="bf16", train=True),
        # one long prompt, forward only, four query heads to a key head
        dict(name="attn_long", kind="attn", lengths="16384", rows=16384, H=16, KV=4, D=128, dtype="bf16",
             train=False),
        # long documents with grouped heads, forward and backward: the largest training call
        dict(name="attn_long_train", kind="attn", lengths="5003,2048,1,1140", rows=8192, H=32, KV=8, D=128,
             dtype="bf16", train=True),
        # the check of a target in full precision, an uneven head width
        dict(name="attn_fp32_train", kind="attn", lengths="700,3,801", rows=1504, H=8, KV=2, D=80, dtype="fp32",
             train=True),
        # a short request's norm at the LM target's width: latency
        dict(name="norm_small", kind="norm", rows=96, d=768, dtype="bf16", affine="both", train=False),
        # a training batch of wide activations
        dict(name="norm_train", kind="norm", rows=16384, d=4096, dtype="bf16", affine="both", train=True),
        # fp32 activations of the residual MLP's width over an odd number of rows
        dict(name="norm_fp32_train", kind="norm", rows=5003, d=1000, dtype="fp32", affine="both", train=True),
        # a few positions of a scoring pass over the LM target's vocabulary
        dict(name="top_kl_small", kind="top_kl", rows=33, V=50277, k=32, dtype="bf16", rest=False, tau=1.0,
             fused=False),
        # the LM step's positions: loss and gradient in one call, weighted positions
        dict(name="top_kl_50277", kind="top_kl", rows=8192, V=50277, k=64, dtype="bf16", rest=True, tau=1.0,
             fused=True),
        # a large vocabulary inside a caller's own autograd model, softened
        dict(name="top_kl_autograd_131072", kind="top_kl", rows=2048, V=131072, k=128, dtype="bf16", rest=True,
             tau=2.0, fused=False),
        # fp32 logits
        dict(name="top_kl_fp32", kind="top_kl", rows=1500, V=32000, k=20, dtype="fp32", rest=False, tau=1.0,
             fused=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "norm", "top_kl"])
    if kind == "attn":
        train, dtype = rng.random() < 0.6, rng.choice(["bf16", "bf16", "bf16", "fp32"])
        KV = rng.choice([1, 2, 4, 8, 12])
        H = KV * rng.choice([r for r in (1, 2, 3, 4, 8) if 4 <= KV * r <= 32])
        D = rng.choice([64, 64, 128, 128, 80, 96, 40])
        while True:
            total = _log_int(rng, 1, 2000 if dtype == "fp32" else 8000)
            left, lengths = total, []
            while left:
                lengths.append(min(left, _log_int(rng, 1, total)))
                left -= lengths[-1]
                if len(lengths) == 400:
                    lengths.append(left)
                    break
            case = dict(kind="attn", lengths=",".join(map(str, lengths)), rows=total + rng.choice([0, 0, 1, 50]), H=H,
                        KV=KV, D=D, dtype=dtype, train=train)
            # gradients of scores that have one key each are zero: nothing to compare
            if work(case)["flops"] <= 5e11 and (max(lengths) > 1 or not train):
                return case
    if kind == "norm":
        d = rng.choice([64, 768, 1000, 1024, 2048, 4096, 5120, 8192, _log_int(rng, 33, 9000)])
        rows = _log_int(rng, 1, 6e7 / d)
        return dict(kind="norm", rows=rows, d=d, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    affine=rng.choice(["both", "both", "weight", "none"]), train=rng.random() < 0.7)
    V = rng.choice([1000, 32000, 50277, 65536, 131072, _log_int(rng, 500, 200000)])
    rest = rng.random() < 0.5
    return dict(kind="top_kl", rows=_log_int(rng, 1, 2e8 / V), V=V, k=_log_int(rng, 8 if rest else 1, 200),
                dtype=rng.choice(["bf16", "bf16", "fp32"]), rest=rest, tau=rng.choice([1.0, 1.0, 2.0, 0.7]),
                fused=rng.random() < 0.5)


# ----------------------------------------------------------------------------------- inputs
def _lengths(case):
    return [int(s) for s in case["lengths"].split(",")]


def prepare(case, seed):
    dev, dt = "cuda", DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def rand(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=gen).mul_(scale)

    if case["kind"] == "attn":
        ends = [0]
        for n in _lengths(case):
            ends.append(ends[-1] + n)
        N, H, KV, D = case["rows"], case["H"], case["KV"], case["D"]
        s = dict(offsets=torch.tensor(ends, dtype=torch.int32, device=dev))
        if case["train"]:
            s["q"] = rand(N, H, D).to(dt).requires_grad_()
            s["k"] = rand(N, KV, D).to(dt).requires_grad_()
            s["v"] = rand(N, KV, D).to(dt).requires_grad_()
            s["g"] = rand(N, H, D).to(dt)
        else:  # the views of one projection's output
            qkv = rand(N, (H + 2 * KV) * D).to(dt)
            s["q"] = qkv[:, :H * D].view(N, H, D)
            s["k"] = qkv[:, H * D:(H + KV) * D].view(N, KV, D)
            s["v"] = qkv[:, (H + KV) * D:].view(N, KV, D)
    elif case["kind"] == "norm":
        d = case["d"]
        # a residual stream: channels of different scales around a common offset
        s = dict(x=(rand(case["rows"], d) * (0.5 + rand(d).abs_()) + 0.5).to(dt), weight=None, bias=None)
        if case["affine"] != "none":
            s["weight"] = rand(d, scale=0.2) + 1.0
        if case["affine"] == "both":
            s["bias"] = rand(d, scale=0.1)
        if case["train"]:
            s["g"] = rand(case["rows"], d).to(dt)
            s["leaves"] = [t.requires_grad_() for t in (s["x"], s["weight"], s["bias"]) if t is not None]
    else:
        rows, V, k = case["rows"], case["V"], min(case["k"], case["V"])
        # probabilities fall as a power of their rank, as a language model's do
        clean = torch.empty(rows, V, device=dev).exponential_(generator=gen).mul_(1.6)
        top = clean.topk(k, dim=-1)
        s = dict(top=top.values.to(dt), idx=top.indices.to(torch.int32), tau=case["tau"], lse=None)
        if case["rest"]:
            s["lse"] = torch.logsumexp(clean / case["tau"], -1)
            # as the stored logits are rounded, their mass is kept at most the whole
            s["lse"] = torch.maximum(s["lse"], torch.logsumexp(s["top"].float() / case["tau"], -1))
        s["z"] = clean.add_(rand(rows, V, scale=0.7)).to(dt)
        s["g"] = torch.rand(rows, device=dev, generator=gen) / rows
        if not case["fused"]:
            s["z"].requires_grad_()
    return dict(s, case=case)


# ------------------------------------------------------------------------------- the passes
def run(state):
    return {"attn": _run_attn, "norm": _run_norm, "top_kl": _run_top_kl}[state["case"]["kind"]](state)


def _run_attn(s):
    q, k, v, offsets = s["q"], s["k"], s["v"], s["offsets"]
    if own:
        from param_decomp_amd.attention import packed_attention

        out = packed_attention(q, k, v, offsets)
        return (out, *torch.autograd.grad(out, (q, k, v), s["g"])) if s["case"]["train"] else out
    with torch.no_grad():
        return _plain_attn(q, k, v, offsets, s.get("g"))


def _run_norm(s):
    x, w, b = s["x"], s["weight"], s["bias"]
    if own:
        from param_decomp_amd.norms import layer_norm

        y = layer_norm(x, w, b, eps=EPS)
        return (y, *torch.autograd.grad(y, s["leaves"], s["g"])) if s["case"]["train"] else y
    with torch.no_grad():
        return _plain_norm(x, w, b, s.get("g"))


def _run_top_kl(s):
    z, top, idx, lse, tau, g = (s[n] for n in ("z", "top", "idx", "lse", "tau", "g"))
    if own:
        from param_decomp_amd import losses, ops

        if s["case"]["fused"]:
            return ops.top_logits_kl(z, top, idx, clean_lse=lse, temperature=tau, row_weight=g, want_grad=True)
        kl = losses.top_logits_position_kl(z, top, idx, clean_lse=lse, temperature=tau)
        return (kl, *torch.autograd.grad(kl, z, g))
    with torch.no_grad():
        return _plain_top_kl(z, top, idx, lse, tau, g)


# ------------------------------------------------------------------- plain forms, in 32 bits
def _plain_attn(q, k, v, offsets, g):
    N, H, D = q.shape
    KV, dt = k.shape[1], q.dtype
    pos = torch.arange(N, device=q.device)
    seq = torch.searchsorted(offsets, pos.to(offsets.dtype), right=True)  # 1 .. sequences for the rows of one
    held = (seq >= 1) & (seq < offsets.numel())
    allowed = (seq[:, None] == seq[None, :]) & (pos[:, None] >= pos[None, :]) & held[:, None]
    qf, kf, vf = (t.float().transpose(0, 1).reshape(KV, -1, N, D) for t in (q, k, v))  # [KV, H / KV or 1, N, D]
    scale = D**-0.5
    s = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale).masked_fill_(~allowed, -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    p = s.div_(s.sum(-1, keepdim=True).clamp_(min=1e-30))
    o = torch.matmul(p, vf)
    rows = lambda t, heads: t.reshape(heads, N, D).transpose(0, 1).to(dt).contiguous()  # noqa: E731
    if g is None:
        return rows(o, H)
    gf = g.float().transpose(0, 1).reshape(KV, -1, N, D)
    dv = torch.matmul(p.transpose(-1, -2), gf).sum(1)
    ds = torch.matmul(gf, vf.transpose(-1, -2)).sub_((gf * o).sum(-1, keepdim=True)).mul_(p)
    del p, s
    dq = torch.matmul(ds, kf).mul_(scale)
    dk = torch.matmul(ds.transpose(-1, -2), qf).sum(1).mul_(scale)
    return rows(o, H), rows(dq, H), rows(dk, KV), rows(dv, KV)


def _plain_norm(x, w, b, g):
    xf = x.float()
    xc = xf - xf.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xh = xc * rstd
    y = xh if w is None else xh * w
    y = (y if b is None else y + b).to(x.dtype)
    if g is None:
        return y
    gf = g.float()
    gw = gf if w is None else gf * w
    dx = (rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))).to(x.dtype)
    out = [y, dx]
    if w is not None:
        out.append((gf * xh).sum(0, dtype=F64).float())
    if b is not None:
        out.append(gf.sum(0, dtype=F64).float())
    return tuple(out)


def _plain_top_kl(z, top, idx, lse, tau, g):
    # a row's sums and logarithms in 64 bits: kl is a small difference of them
    zf = z.float() / tau
    t = top.double() / tau
    at = idx.long()
    zmax = zf.amax(-1, keepdim=True)
    e = (zf - zmax).exp_()
    total = e.sum(-1, keepdim=True, dtype=F64)
    logq = zf.gather(1, at).double() - zmax - total.log()
    if lse is None:
        logp = t - torch.logsumexp(t, -1, keepdim=True)
        p = logp.exp()
        kl = (p * (logp - logq)).sum(-1)
        mass = p.sum(-1, keepdim=True)
        grad = e.mul_((mass / total).float())
    else:
        logp = t - lse[:, None].double()
        p = logp.exp()
        rest = 1.0 - p.sum(-1, keepdim=True)
        rest = torch.where((rest < REST_MIN) | (at.shape[1] == z.shape[1]), torch.zeros_like(rest), rest)
        # the sum over the rest leaves the listed entries out itself: no difference of two sums
        others = zf.scatter(1, at, -math.inf)
        omax = others.amax(-1, keepdim=True).clamp_(min=-1e30)
        eo = (others - omax).exp_()
        so = eo.sum(-1, keepdim=True, dtype=F64)
        log_q_rest = (omax - zmax) + so.log() - total.log()
        part = torch.where(rest > 0, rest * (rest.clamp(min=1e-30).log() - log_q_rest), torch.zeros_like(rest))
        kl = (p * (logp - logq)).sum(-1) + part[:, 0]
        grad = e.mul_(((p.sum(-1, keepdim=True) + rest) / total).float())
        grad.sub_(eo.mul_(torch.where(rest > 0, rest / so, torch.zeros_like(rest)).float()))
    grad.scatter_add_(1, at, -p.float())
    return kl.float(), grad.mul_(g[:, None] / tau).to(z.dtype)


# ------------------------------------------------------------------------------------ work
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "attn":
        pairs = sum(n * (n + 1) // 2 for n in _lengths(case))
        qo = case["rows"] * case["H"] * case["D"] * e
        kv = case["rows"] * case["KV"] * case["D"] * e
        # q k^T and p v; backward dp, dq, dk and dv
        return {"bytes": (2 if case["train"] else 1) * (2 * qo + 2 * kv),
                "flops": (12 if case["train"] else 4) * pairs * case["H"] * case["D"]}
    if case["kind"] == "norm":
        n = case["rows"] * case["d"]
        par = {"both": 2, "weight": 1, "none": 0}[case["affine"]] * case["d"] * 4
        return {"bytes": (4 * n * e + 2 * par) if case["train"] else (2 * n * e + par),
                "flops": (20 if case["train"] else 8) * n}
    n, k = case["rows"] * case["V"], min(case["k"], case["V"])
    return {"bytes": 2 * n * e + case["rows"] * (k * (e + 4) + 8), "flops": 8 * n}


# ------------------------------------------------------------------------ outputs in 64 bits
def exact(case, seed):
    s = prepare(case, seed)

    def attn():
        q, k, v = (s[n].detach() for n in ("q", "k", "v"))
        N, H, D = q.shape
        rep = H // k.shape[1]
        outs = [torch.zeros(t.shape, dtype=F64, device=q.device) for t in ((q, q, k, v) if case["train"] else (q,))]
        first = 0
        for n in _lengths(case):  # one sequence and head at a time, as if it were alone
            at = slice(first, first + n)
            first += n
            above = torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1)
            for h in range(H):
                Q, K, V = q[at, h].double(), k[at, h // rep].double(), v[at, h // rep].double()
                S = (Q @ K.T / math.sqrt(D)).masked_fill_(above, -math.inf)
                P = torch.softmax(S, -1)
                outs[0][at, h] = P @ V
                if case["train"]:
                    G = s["g"][at, h].double()
                    dP = G @ V.T
                    dS = P * (dP - (P * dP).sum(-1, keepdim=True)) / math.sqrt(D)
                    outs[1][at, h] = dS @ K
                    outs[2][at, h // rep] += dS.T @ Q
                    outs[3][at, h // rep] += P.T @ G
        return tuple(outs) if case["train"] else outs[0]

    def norm():
        x = s["x"].detach().double()
        w = torch.ones(case["d"], dtype=F64, device=x.device) if s["weight"] is None else s["weight"].detach().double()
        var, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
        sd = (var + EPS).sqrt()
        xh = (x - mean) / sd
        y = xh * w
        if s["bias"] is not None:
            y = y + s["bias"].detach().double()
        if not case["train"]:
            return y
        g = s["g"].double()
        a = g * w
        out = [y, (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True)) / sd]
        if s["weight"] is not None:
            out.append((g * xh).sum(0))
        if s["bias"] is not None:
            out.append(g.sum(0))
        return tuple(out)

    def top_kl():
        z, tau, at = s["z"].detach(), case["tau"], s["idx"].long()
        kl, grad = [], []
        for r in range(0, z.shape[0], 1024):
            zz, aa = z[r:r + 1024].double() / tau, at[r:r + 1024]
            logq = torch.log_softmax(zz, -1)
            t = s["top"][r:r + 1024].double() / tau
            target = torch.zeros_like(zz)
            if s["lse"] is None:
                p = torch.softmax(t, -1)
                kl.append((p * (p.log() - logq.gather(1, aa))).sum(-1))
            else:
                p = (t - s["lse"][r:r + 1024, None].double()).exp()
                rest = 1 - p.sum(-1, keepdim=True)
                rest = torch.where((rest < REST_MIN) | (aa.shape[1] == zz.shape[1]), torch.zeros_like(rest), rest)
                qrest = logq.scatter(1, aa, -math.inf)
                lrest = torch.logsumexp(qrest, -1, keepdim=True)
                kl.append((p * (p.log() - logq.gather(1, aa))).sum(-1) +
                          torch.where(rest > 0, rest * (rest.log() - lrest), torch.zeros_like(rest))[:, 0])
                target += torch.where(rest > 0, rest * (qrest - lrest).exp(), torch.zeros_like(qrest))
            target.scatter_add_(1, aa, p)
            # the row's whole target mass times q, less the target
            grad.append((logq.exp() * target.sum(-1, keepdim=True) - target) * (s["g"][r:r + 1024, None].double() / tau))
        return torch.cat(kl), torch.cat(grad)

    with torch.no_grad():
        return {"attn": attn, "norm": norm, "top_kl": top_kl}[case["kind"]]()
