"""The calls that a training step of a language-model or mixture-of-experts target makes beside
its decomposed sites, as they are measured: cross entropy over a vocabulary whose logits are
never kept, AdamW over many tensors, the router's choice by scores, and the norms around a
residual branch.

`listed()` and `draw(rng)` give cases (dicts of plain values), `prepare(case, seed)` what a
program holds before the call, `run(state)` one pass: the framework's calls where `own` is
set, elementary torch operations in 32 bits otherwise. `work(case)` gives the bytes and
operations a pass cannot do without and `exact(case, seed)` its outputs in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

F32, F64, I64 = torch.float32, torch.float64, torch.int64
FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
QBLOCK = 256  # values that share a scale in 8-bit states
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
STEP0 = 700  # steps that an optimizer has behind it


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the loss of a few positions of a short text under the LM target: latency
        dict(name="ce_score", kind="ce", N=33, d=768, V=50277, skip=0, dtype="bf16", form="score"),
        # a training batch of the 4-layer LM target (16 x 512 positions), every position weighted by the caller
        dict(name="ce_lm_train", kind="ce", N=8192, d=768, V=50277, skip=0, dtype="bf16", form="autograd"),
        # wide activations over a large vocabulary, a quarter of the positions a prompt that does
        # not count; loss and gradients in one call: the largest
        dict(name="ce_wide_train", kind="ce", N=4096, d=4096, V=131072, skip=1024, dtype="bf16", form="fused"),
        # the check of a target in full precision, odd sizes
        dict(name="ce_fp32_train", kind="ce", N=1003, d=1000, V=32003, skip=100, dtype="fp32", form="autograd"),
        # the components of a toy target: latency
        dict(name="adamw_toy", kind="adamw", sizes="100*2,500,2000*2,77,1,4096", bits=32, grad="fp32", copy=False),
        # V and U of the LM target's 24 sites and their bf16 copies for the next step
        dict(name="adamw_lm_32", kind="adamw", sizes="786432*32,3145728*8,12582912*8", bits=32, grad="fp32", copy=True),
        # V and U of the 4-layer mixture's expert sites, states in 8 bits
        dict(name="adamw_moe_8", kind="adamw", sizes="11010048*24", bits=8, grad="bf16", copy=True),
        # a short request's rows through the mixture target's router: latency
        dict(name="route_small", kind="route", T=17, E=42, k=8, scoring="softmax", bias=False, groups=1, top=1,
             renorm=True, dtype="fp32", train=False),
        # a training batch with balanced sigmoid scores and limited groups
        dict(name="route_train", kind="route", T=8192, E=256, k=8, scoring="sigmoid", bias=True, groups=8, top=4,
             renorm=True, dtype="bf16", train=True),
        # many rows, softmax weights as they are
        dict(name="route_long", kind="route", T=131072, E=128, k=8, scoring="softmax", bias=False, groups=1, top=1,
             renorm=False, dtype="fp32", train=True),
        # a short request's block at the LM target's width: latency
        dict(name="norm_small", kind="norm", rows=96, d=768, stream="bf16", dtype="bf16", gate="none", post=False,
             train=False),
        # a training batch of wide activations, norms on both sides of the branch, a gate for each sequence
        dict(name="norm_train", kind="norm", rows=16384, d=4096, stream="bf16", dtype="bf16", gate="seq", post=True,
             train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["ce", "adamw", "route", "norm"])
    if kind == "ce":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        most = 2e11 if dtype == "fp32" else 2e12
        while True:
            N, d, V = _log_int(rng, 1, 20000), rng.choice([512, 768, 1024, 2048, 4096, 8 * _log_int(rng, 8, 600)]), \
                rng.choice([1000, 32000, 50277, 65536, 131072, _log_int(rng, 300, 160000)])
            if dtype == "fp32":
                d = rng.choice([d, _log_int(rng, 33, 3000)])
            if 2 * N * d * V <= most:
                return dict(kind="ce", N=N, d=d, V=V, skip=rng.choice([0, 0, N // 5, N // 2]), dtype=dtype,
                            form=rng.choice(["score", "autograd", "autograd", "fused"]))
    if kind == "adamw":
        total, sizes = _log_int(rng, 100, 1.5e8), []
        while total > 0 and len(sizes) < 70:
            sizes.append(min(total, _log_int(rng, 1, total)) if len(sizes) < 69 else total)
            total -= sizes[-1]
        return dict(kind="adamw", sizes=",".join(map(str, sizes)), bits=rng.choice([32, 8]),
                    grad=rng.choice(["fp32", "bf16"]), copy=rng.random() < 0.5)
    if kind == "route":
        E = rng.choice([8, 16, 42, 64, 72, 128, 160, 256, 256, 384, 512])
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0])
        top = rng.randint(1, groups)
        k = rng.randint(1, min(16, E // groups * top))
        return dict(kind="route", T=_log_int(rng, 1, 1.6e7 / E), E=E, k=k, scoring=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, groups=groups, top=top, renorm=rng.random() < 0.6,
                    dtype=rng.choice(["bf16", "fp32"]), train=rng.random() < 0.7)
    stream, dtype = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32")])
    d = rng.choice([64, 768, 1000, 1024, 2048, 4096, 5120, 8192, _log_int(rng, 33, 9000)])
    rows = _log_int(rng, 1, 6e7 / d)
    return dict(kind="norm", rows=rows, d=d, stream=stream, dtype=dtype,
                gate=rng.choice(["none", "channel", "seq", "full"]), post=rng.random() < 0.6, train=rng.random() < 0.7)


# ----------------------------------------------------------------------------------- inputs
def _sizes(case):
    out = []
    for s in case["sizes"].split(","):
        n, _, times = s.partition("*")
        out += [int(n)] * int(times or 1)
    return out


def _up(n):
    return -(-n // QBLOCK) * QBLOCK


def _sequences(rows):
    """Sequences of one length that the rows are cut into."""
    return next(s for s in (16, 8, 5, 4, 3, 2, 1) if rows % s == 0)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def rand(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=gen).mul_(scale)

    if case["kind"] == "ce":
        N, d, V, dt = case["N"], case["d"], case["V"], DTYPES[case["dtype"]]
        head = rand(V, d, scale=1.5 / math.sqrt(d))
        targets = torch.randint(V, (N,), device=dev, generator=gen)
        act = rand(N, d)
        known = torch.rand(N, 1, device=dev, generator=gen) < 0.5  # positions whose target the model expects
        act += torch.where(known, 4.0 * head[targets], torch.zeros_like(act))
        if case["skip"]:
            targets[torch.randperm(N, device=dev, generator=gen)[:case["skip"]]] = -100
        s = dict(act=act.to(dt), head=head.to(dt), targets=targets)
        s["g"] = (0.5 + torch.rand(N, device=dev, generator=gen)) / N
        if case["form"] == "autograd":
            s["act"].requires_grad_()
            s["head"].requires_grad_()
    elif case["kind"] == "adamw":
        sizes, starts = _sizes(case), [0]
        for n in sizes:
            starts.append(starts[-1] + _up(n))
        total = starts[-1]
        held = torch.zeros(total, dtype=torch.bool, device=dev)
        flat_p, flat_g = rand(total, scale=0.05), rand(total, scale=1e-3)
        m, v = rand(total, scale=3e-4), torch.empty(total, device=dev).exponential_(generator=gen).mul_(1e-6)
        for n, at in zip(sizes, starts):
            held[at:at + n] = True
        for t in (flat_p, flat_g, m, v):
            t.mul_(held)
        del held

        def cut(t, per=1):
            return [t[at // per:at // per + -(-n // per)] for n, at in zip(sizes, starts)]

        flat_g = flat_g.to(DTYPES[case["grad"]])
        s = dict(flat=dict(p=flat_p, g=flat_g), p=cut(flat_p), g=cut(flat_g), key=(int(seed) & 0x7FFFFFFF, 11),
                 step=torch.full((1,), STEP0, dtype=torch.int32, device=dev), copies=None)
        state = dict(step=s["step"])
        if case["bits"] == 8:
            for name, t in (("m", m), ("v", v.sqrt_())):
                top = t.view(-1, QBLOCK).abs().amax(-1)
                codes = (t.view(-1, QBLOCK) * (448.0 / top.clamp(min=1e-30))[:, None]).clamp_(-448.0, 448.0).to(FP8)
                s["flat"][name], s["flat"][name + "_scale"] = codes.view(-1), top / 448.0
                state[name], state[name + "_scale"] = cut(codes.view(-1)), cut(s["flat"][name + "_scale"], QBLOCK)
        else:
            s["flat"].update(m=m, v=v)
            state.update(m=cut(m), v=cut(v))
        if case["copy"]:
            s["flat"]["copy"] = flat_p.to(torch.bfloat16)
            s["copies"] = cut(s["flat"]["copy"])
        s["state"] = state
    elif case["kind"] == "route":
        T, E, dt = case["T"], case["E"], DTYPES[case["dtype"]]
        s = dict(logits=(rand(T, E, scale=1.5) + rand(E, scale=0.7)).to(dt), bias=None)
        if case["bias"]:
            s["bias"] = rand(E, scale=0.1)
        if case["train"]:
            s["logits"].requires_grad_()
            s["g"] = rand(T, case["k"])
    else:
        rows, d = case["rows"], case["d"]
        xt, bt = DTYPES[case["stream"]], DTYPES[case["dtype"]]
        # a residual stream of channels of different scales, and a branch's output
        s = dict(x=(rand(rows, d) * (0.5 + rand(d).abs_())).to(xt), branch=rand(rows, d, scale=0.6).to(bt),
                 pre=rand(d, scale=0.2) + 1.0, post=rand(d, scale=0.2) + 1.0 if case["post"] else None, gate=None)
        seqs = {"none": 0, "channel": 1, "seq": _sequences(rows), "full": rows}[case["gate"]]
        if seqs:
            s["gate"] = rand(seqs, d, scale=0.5).add_(0.3).to(bt if case["gate"] == "full" else F32)
            if case["gate"] == "channel":
                s["gate"] = s["gate"][0].clone()
        if case["train"]:
            s["gh"], s["gy"] = rand(rows, d).to(xt), rand(rows, d).to(bt)
            s["leaves"] = [s[n].requires_grad_() for n in ("x", "branch", "post", "gate", "pre") if s[n] is not None]
    return dict(s, case=case)


# ------------------------------------------------------------------------------- the passes
def run(state):
    return {"ce": _run_ce, "adamw": _run_adamw, "route": _run_route, "norm": _run_norm}[state["case"]["kind"]](state)


def _run_ce(s):
    act, head, targets, g, form = s["act"], s["head"], s["targets"], s["g"], s["case"]["form"]
    if own:
        from param_decomp_amd import losses, ops

        if form == "fused":
            return ops.streamed_cross_entropy(act, head, targets, row_weight=g, want_dact=True, want_dhead=True)
        loss = losses.streamed_position_cross_entropy(act, head, targets)
        return (loss, *torch.autograd.grad(loss, (act, head), g)) if form == "autograd" else loss
    with torch.no_grad():
        return _plain_ce(act, head, targets, None if form == "score" else g)


def _run_adamw(s):
    case, flat = s["case"], s["flat"]
    if own:
        from param_decomp_amd.optim import AdamW

        opt = s.get("optimizer")
        if opt is None:  # the one that the program keeps
            opt = s["optimizer"] = AdamW(s["p"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY,
                                         state_bits=case["bits"], key=s["key"], copies=s["copies"], state=s["state"])
        opt.step(s["g"])
    else:
        _plain_adamw(s)
    return dict(step=s["step"], **{n: t for n, t in flat.items() if n != "g"})


def _run_route(s):
    case, logits, bias = s["case"], s["logits"], s["bias"]
    if own:
        from param_decomp_amd.routed import experts

        w, idx = experts.route_scores(logits, case["k"], scoring=case["scoring"], bias=bias, n_groups=case["groups"],
                                      top_groups=case["top"], renormalize=case["renorm"], scale=2.5)
        return (w, idx, *torch.autograd.grad(w, logits, s["g"])) if case["train"] else (w, idx)
    with torch.no_grad():
        return _plain_route(s)


def _run_norm(s):
    if own:
        from param_decomp_amd.norms import residual_norm

        out = residual_norm(s["x"], s["branch"], post_weight=s["post"], post_norm=s["case"]["post"], gate=s["gate"],
                            pre_weight=s["pre"], scale=0.5, eps=EPS)
        return (*out, *torch.autograd.grad(out, s["leaves"], (s["gh"], s["gy"]))) if s["case"]["train"] else out
    with torch.no_grad():
        return _plain_norm(s)


# ------------------------------------------------------------------- plain forms, in 32 bits
def _plain_ce(act, head, targets, g):
    N, V = act.shape[0], head.shape[0]
    counts = (targets >= 0) & (targets < V)
    at = torch.where(counts, targets, torch.zeros_like(targets))[:, None]
    af, hf = act.float(), head.float()
    z = torch.matmul(af, hf.t())
    top = z.amax(-1, keepdim=True)
    target = z.gather(1, at) - top
    e = z.sub_(top).exp_()
    total = e.sum(-1, keepdim=True, dtype=F64)
    loss = torch.where(counts, (total.log() - target.double())[:, 0], torch.zeros(N, dtype=F64, device=z.device))
    if g is None:
        return loss.float()
    e.div_(total.float())
    # p - 1 at the target, where p may be near 1, from the loss
    e.scatter_(1, at, torch.expm1(-loss).float()[:, None])
    e.mul_(torch.where(counts, g, torch.zeros_like(g))[:, None])
    return loss.float(), torch.matmul(e, hf).to(act.dtype), torch.matmul(e.t(), af).to(head.dtype)


MASK = 0xFFFFFFFF


def _threefry(k0, k1, x0, x1):
    """Threefry-2x32 of 20 rounds over int64 tensors that hold 32-bit words."""
    ks = (k0, k1, k0 ^ k1 ^ 0x1BD11BDA)
    x0, x1 = (x0 + k0) & MASK, (x1 + k1) & MASK
    for i, rot in enumerate((13, 15, 26, 6, 17, 29, 16, 24) * 2 + (13, 15, 26, 6)):
        x0 = (x0 + x1) & MASK
        x1 = (((x1 << rot) & MASK) | (x1 >> (32 - rot))) ^ x0
        if i % 4 == 3:
            n = i // 4 + 1
            x0, x1 = (x0 + ks[n % 3]) & MASK, (x1 + ks[(n + 1) % 3] + n) & MASK
    return x0, x1


def _to_fp8(a, bits, floor):
    """Magnitudes up to 448 rounded to e4m3 values, up with the probability of their fraction (16 bits
    of it); `floor`: what is not zero does not become zero."""
    normal = ((a.view(torch.int32) + (bits << 4).int()) >> 20 << 20).view(F32)
    small = torch.floor(a * 512.0 + bits.float() / 65536.0) / 512.0
    q = torch.where(a >= 2.0**-6, normal, small)
    return torch.where((a > 0) & (q == 0), torch.full_like(q, 2.0**-9), q) if floor else q


def _plain_adamw(s):
    flat, case = s["flat"], s["case"]
    p, g, step = flat["p"], flat["g"].float(), s["step"]
    step += 1
    t = step.double()
    c1, c2 = -torch.expm1(t * math.log(BETA1)), -torch.expm1(t * math.log(BETA2))
    if case["bits"] == 8:
        wide = lambda n: (flat[n].float().view(-1, QBLOCK) * flat[n + "_scale"][:, None]).view(-1)  # noqa: E731
        m, v = wide("m"), wide("v").square_()
    else:
        m, v = flat["m"], flat["v"]
    m.add_(g - m, alpha=1 - BETA1)
    v.add_(g * g - v, alpha=1 - BETA2)
    root = v.sqrt()
    p.sub_(p * (LR * DECAY) + m * (LR / c1).float() / (root / c2.sqrt().float() + ADAM_EPS))
    if case["copy"]:
        flat["copy"].copy_(p)
    if case["bits"] == 8:
        zero = torch.zeros((), dtype=I64, device=p.device)
        k0, k1 = _threefry(zero + s["key"][0], zero + s["key"][1], zero, step[0].long())
        pair = torch.arange(p.numel() // 2, device=p.device)
        bits = torch.stack(_threefry(k0, k1, pair >> 32, pair & MASK), -1).view(-1)  # a word for each value
        del pair
        for name, x, b in (("m", m, bits & 0xFFFF), ("v", root, bits >> 16)):
            top = x.view(-1, QBLOCK).abs().amax(-1)
            a = (x.view(-1, QBLOCK).abs() * (448.0 / top.clamp(min=2.0**-100))[:, None]).clamp_(max=448.0).view(-1)
            flat[name].copy_(torch.copysign(_to_fp8(a, b, name == "v"), x))
            flat[name + "_scale"].copy_(top / 448.0)


def _largest(keys, n):
    """Indices of the n largest along the last axis, ties to the lowest index."""
    return keys.sort(dim=-1, descending=True, stable=True).indices[..., :n]


def _plain_route(s):
    case, logits = s["case"], s["logits"].double()  # scores next to each other decide the choice
    T, E = logits.shape
    softmax = case["scoring"] == "softmax"
    score = torch.softmax(logits, -1) if softmax else torch.sigmoid(logits)
    key = logits if s["bias"] is None and case["groups"] == 1 else score
    if s["bias"] is not None:
        key = key + s["bias"].double()
    if case["groups"] > 1:
        grouped = key.view(T, case["groups"], -1)
        best = _largest(grouped.gather(2, _largest(grouped, 2)).sum(-1), case["top"])
        allowed = torch.zeros(T, case["groups"], dtype=torch.bool, device=key.device).scatter_(1, best, True)
        key = grouped.masked_fill(~allowed[..., None], -math.inf).view(T, E)
    idx = _largest(key, case["k"])
    chosen = score.gather(1, idx)
    total = chosen.sum(-1, keepdim=True) if case["renorm"] else 1.0
    w = chosen / total * 2.5
    out = [w.float(), idx.int()]
    if case["train"]:
        g = s["g"].double()
        gc = (g - (g * w).sum(-1, keepdim=True) / 2.5 if case["renorm"] else g) * 2.5 / total
        if softmax:
            d = torch.zeros_like(score).scatter_(1, idx, gc * chosen)
            d.sub_(score * d.sum(-1, keepdim=True))
        else:
            d = torch.zeros_like(score).scatter_(1, idx, gc * chosen * (1.0 - chosen))
        out.append(d.to(s["logits"].dtype))
    return tuple(out)


def _plain_norm(s):
    case, x, b = s["case"], s["x"].float(), s["branch"].float()
    rows, d = x.shape

    def over(gate):  # the gate of each row
        return gate.float().view(-1, 1, d).expand(-1, rows // (gate.numel() // d), -1).reshape(rows, d)

    n = b
    if case["post"]:
        rb = torch.rsqrt((b * b).mean(-1, keepdim=True) + EPS)
        bh = b * rb
        n = bh * s["post"]
    h = x + (0.5 * n if s["gate"] is None else 0.5 * over(s["gate"]) * n)
    ho = h.to(s["x"].dtype)
    h = ho.float()  # the stream as it is stored is what is normed
    rh = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    hh = h * rh
    y = (hh * s["pre"]).to(s["branch"].dtype)
    if not case["train"]:
        return ho, y
    gy = s["gy"].float()
    a = gy * s["pre"]
    dx = s["gh"].float() + rh * (a - hh * (a * hh).mean(-1, keepdim=True))
    dn = 0.5 * dx
    out = {"pre": (gy * hh).sum(0, dtype=F64).float()}
    if s["gate"] is not None:
        gate = s["gate"]
        dg = (dn * n).view(-1, rows // (gate.numel() // d), d).sum(1, dtype=F64)
        out["gate"] = dg.view(gate.shape).to(gate.dtype)
        dn = dn * over(gate)
    if case["post"]:
        out["post"] = (dn * bh).sum(0, dtype=F64).float()
        a = dn * s["post"]
        dn = rb * (a - bh * (a * bh).mean(-1, keepdim=True))
    grads = [dx.to(s["x"].dtype), dn.to(s["branch"].dtype), out.get("post"), out.get("gate"), out["pre"]]
    return (ho, y, *(t for t in grads if t is not None))


# ------------------------------------------------------------------------------------ work
def work(case):
    if case["kind"] == "ce":
        e = 2 if case["dtype"] == "bf16" else 4
        N, n = case["N"], case["N"] - case["skip"]
        both = (case["N"] + case["V"]) * case["d"] * e
        train = case["form"] != "score"
        return {"bytes": (2 if train else 1) * both + 16 * N, "flops": max(1, (6 if train else 2) * n * case["d"] * case["V"])}
    if case["kind"] == "adamw":
        n = sum(_sizes(case))
        state = 16 if case["bits"] == 32 else 4 + 16 / QBLOCK
        return {"bytes": n * (8 + (4 if case["grad"] == "fp32" else 2) + state + (2 if case["copy"] else 0)),
                "flops": 15 * n}
    if case["kind"] == "route":
        e = 2 if case["dtype"] == "bf16" else 4
        n, k = case["T"] * case["E"], case["T"] * case["k"]
        return {"bytes": (2 if case["train"] else 1) * n * e + k * (12 if case["train"] else 8), "flops": 8 * n}
    n = case["rows"] * case["d"]
    xe, be = (2 if case[t] == "bf16" else 4 for t in ("stream", "dtype"))
    gate = {"none": 0, "channel": 4 * case["d"], "seq": 4 * case["d"] * _sequences(case["rows"]), "full": be * n}[case["gate"]]
    par = gate + 4 * case["d"] * (2 if case["post"] else 1)
    times = 2 if case["train"] else 1
    return {"bytes": times * (2 * n * (xe + be) + par), "flops": (30 if case["train"] else 12) * n}


# ------------------------------------------------------------------------ outputs in 64 bits
def exact(case, seed):
    s = prepare(case, seed)

    def ce():
        act, head, targets = s["act"].detach(), s["head"].detach().double(), s["targets"]
        losses, dact, dhead = [], [], torch.zeros_like(head)
        for r in range(0, case["N"], 2048):
            a, t = act[r:r + 2048].double(), targets[r:r + 2048]
            logp = torch.log_softmax(a @ head.T, -1)
            on = t != -100
            hot = torch.zeros_like(logp)
            hot[on, t[on]] = 1.0
            losses.append(-(hot * logp.nan_to_num(neginf=-1e300)).sum(-1))
            if case["form"] != "score":
                dz = (logp.exp() - hot) * (s["g"][r:r + 2048].double() * on)[:, None]
                dact.append(dz @ head)
                dhead += dz.T @ a
        return torch.cat(losses) if case["form"] == "score" else (torch.cat(losses), torch.cat(dact), dhead)

    def adamw():
        flat = s["flat"]
        p, g = flat["p"].double(), flat["g"].double()
        if case["bits"] == 8:
            m = flat["m"].double() * flat["m_scale"].double().repeat_interleave(QBLOCK)
            v = (flat["v"].double() * flat["v_scale"].double().repeat_interleave(QBLOCK)) ** 2
        else:
            m, v = flat["m"].double(), flat["v"].double()
        t = STEP0 + 1
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g * g
        del g
        p = p - LR * (DECAY * p + (m / (1 - BETA1**t)) / ((v / (1 - BETA2**t)).sqrt() + ADAM_EPS))
        out = dict(step=None, p=p)
        if case["copy"]:
            out["copy"] = p
        if case["bits"] == 32:
            return dict(out, m=m, v=v)
        for name, x in (("m", m), ("v", v.sqrt())):  # what the codes round, and their scales
            scale = x.view(-1, QBLOCK).abs().amax(-1) / 448
            out[name + "_scale"] = scale
            out[name] = (x.view(-1, QBLOCK) / scale.clamp(min=1e-300)[:, None]).view(-1)
        return out

    def route():
        x = s["logits"].detach().double().requires_grad_()
        T, E = x.shape
        with torch.enable_grad():
            p = 1 / (1 + (-x).exp()) if case["scoring"] == "sigmoid" else (x - x.logsumexp(-1, keepdim=True)).exp()
            with torch.no_grad():
                key = p if s["bias"] is None else p + s["bias"].double()
                size = E // case["groups"]
                best = key.view(T, -1, size).topk(min(2, size), -1).values.sum(-1)
                number = torch.arange(case["groups"], device=x.device)
                before = (best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None]) &
                                                                  (number[None, :] < number[:, None]))
                allowed = (before.sum(-1) < case["top"]).repeat_interleave(size, 1)
                idx = torch.where(allowed, key, -math.inf).sort(dim=-1, descending=True, stable=True).indices[:, :case["k"]]
            c = p.gather(1, idx)
            w = 2.5 * c / c.sum(-1, keepdim=True) if case["renorm"] else 2.5 * c
            grad = torch.autograd.grad(w, x, s["g"].double())[0] if case["train"] else None
        return (w.detach(), None, grad) if case["train"] else (w.detach(), None)

    def norm():
        x, b = s["x"].detach().double(), s["branch"].detach().double()
        rows, d = x.shape
        one = torch.ones(d, dtype=F64, device=x.device)
        wide = lambda n: None if s[n] is None else s[n].detach().double()  # noqa: E731
        post, pre, gate = wide("post"), wide("pre"), wide("gate")
        G = one[None] if gate is None else gate.reshape(-1, d)
        of = torch.arange(rows, device=x.device) // (rows // G.shape[0])
        rb = (b.square().mean(-1, keepdim=True) + EPS).sqrt()
        bn = b / rb if post is not None else b
        n = bn * (one if post is None else post)
        h = x + 0.5 * G[of] * n
        hs = h.to(s["x"].dtype).double()
        rh = (hs.square().mean(-1, keepdim=True) + EPS).sqrt()
        hn = hs / rh
        if not case["train"]:
            return h, hn * pre
        gy = s["gy"].double()
        u = gy * pre
        dx = s["gh"].double() + (u - hn * (u * hn).mean(-1, keepdim=True)) / rh
        dn = dx * 0.5 * G[of]
        if post is None:
            db = dn
        else:
            u = dn * post
            db = (u - bn * (u * bn).mean(-1, keepdim=True)) / rb
        out = [h, hn * pre, dx, db]
        if post is not None:
            out.append((dn * bn).sum(0))
        if gate is not None:
            out.append(torch.zeros_like(G).index_add_(0, of, 0.5 * dx * n).view(gate.shape))
        out.append((gy * hn).sum(0))
        return tuple(out)

    with torch.no_grad():
        return {"ce": ce, "adamw": adamw, "route": route, "norm": norm}[case["kind"]]()
