"""The two ends of a policy with memory, as cases that can be timed and compared.

* ``lce``   softmax cross entropy of a linear head over action bins or a vocabulary, from the hidden
  states and the head's weight: the loss of imitation, or the log-probabilities alone that a policy
  loss takes as its old or reference ones;
* ``mem``   linear attention with a decay for each head along a rollout, cut where an episode
  starts, with its gradients;
* ``step``  the same for the single step of an acting policy, its state updated in place.

``run`` computes them in plain torch, or, where ``own`` is true, by the package's operators.
"""

import math

import torch

own = False

DEV = "cuda:0"
CHUNK = 64                    # steps that the plain form of the attention takes at once
F16_SCALE = 4096.0            # a loss with float16 heads is scaled, as mixed precision does it


def listed():
    return [
        # a minibatch of nine compass actions behind the example's trunk: launch latency
        _lce("lce_2560x64x9", 2560, 64, 9, bias=True),
        # one step of the benchmark workload's agents, 5 x 5 acceleration bins
        _lce("lce_256000x64x25_bf16", 256000, 64, 25, "bfloat16", bias=True),
        # sequences of tokens, an odd vocabulary, padded ends masked
        _lce("lce_8x1023x1024x50001_bf16", 8 * 1023, 1024, 50001, "bfloat16", seqs=8, mask=True),
        # few rows of a long vocabulary in float32
        _lce("lce_96x1024x131072", 96, 1024, 131072),
        # odd widths in float16, a bias
        _lce("lce_2047x1000x32003_f16", 2047, 1000, 32003, "float16", bias=True),
        # log-probabilities of single tokens, as an acting policy records them
        _lce("lce_logp_16x1024x131072_bf16", 16, 1024, 131072, "bfloat16", grad=False),
        # the smallest rollout's agents (64 envs x 4) act: launch latency
        _step("step_64x4", 256, 2, 32, 32),
        # the benchmark workload's agents act
        _step("step_16000x16_bf16", 256000, 2, 32, 32, "bfloat16"),
        # a rollout of the benchmark workload, trained on
        _mem("mem_32x16000x16_bf16_grad", 32, 256000, 2, 32, 32, "bfloat16", grad=True),
        # long episodes of 24 envs x 4 agents, odd length
        _mem("mem_4095x96_bf16_grad", 4095, 96, 4, 64, 64, "bfloat16", grad=True, state=True),
        # odd widths in float32
        _mem("mem_1023x64_grad", 1023, 64, 4, 40, 72, grad=True, state=True),
        # two long sequences taken in at once
        _mem("mem_32769x2_bf16", 32769, 2, 8, 128, 128, "bfloat16", state=True, starts=False),
    ]


def _named(name, case):
    return dict(case, name=name) if name else case


def _lce(name, rows, dim, width, dtype="float32", seqs=0, mask=False, bias=False, grad=True):
    return _named(name, {"kind": "lce", "rows": rows, "dim": dim, "width": width, "dtype": dtype,
                         "seqs": seqs, "mask": mask, "bias": bias, "grad": grad})


def _mem(name, T, batch, heads, dk, dv, dtype="float32", grad=False, state=False, starts=True):
    return _named(name, {"kind": "mem", "T": T, "batch": batch, "heads": heads, "dk": dk, "dv": dv,
                         "dtype": dtype, "grad": grad, "state": state, "starts": starts})


def _step(name, batch, heads, dk, dv, dtype="float32", starts=True):
    return _named(name, {"kind": "step", "batch": batch, "heads": heads, "dk": dk, "dv": dv,
                         "dtype": dtype, "starts": starts})


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("lce", "lce", "mem", "mem", "step"))
    dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
    if kind == "lce":
        V, D = _log(rng, 2, 140_000), _log(rng, 16, 2048)
        rows = _log(rng, 1, max(2, min(260_000, 200_000_000 // V, 200_000_000_000 // (V * D),
                                       130_000_000 // D)))
        seqs = rng.choice((0, 0, rng.randint(1, 8)))
        seqs = seqs if rows >= 4 * seqs else 0
        return _lce("", rows // seqs * seqs if seqs else rows, D, V, dtype, seqs,
                    bool(seqs) and rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.8)
    H = rng.choice((1, 2, 3, 4, 8))
    dk, dv = ((rng.choice((16, 32, 64, 128)),) * 2 if rng.random() < 0.6 else
              (rng.randint(1, 128), rng.randint(1, 128)))
    if kind == "step":
        return _step("", _log(rng, 1, max(2, min(256_000, 500_000_000 // (H * dk * dv)))), H, dk, dv,
                     dtype, rng.random() < 0.5)
    T = _log(rng, 1, 33_000)
    batch = _log(rng, 1, max(2, min(60_000, 100_000_000 // (T * H * max(dk, dv)),
                                    250_000_000 // (H * dk * dv))))
    return _mem("", T, batch, H, dk, dv, dtype, rng.random() < 0.6, rng.random() < 0.6,
                rng.random() < 0.6)


# ------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1) + 29)
    dt = getattr(torch, case["dtype"])
    s = {"case": case}

    def rn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV).mul_(scale).to(dt)
    if case["kind"] == "lce":
        n, D, V, seqs = case["rows"], case["dim"], case["width"], case["seqs"]
        lead = (seqs, n // seqs) if seqs else (n,)
        # a head in training: logits of a few units
        h, s["weight"] = rn(*lead, D), rn(V, D, scale=2.0 / math.sqrt(D))
        s["bias"] = rn(V, scale=0.5) if case["bias"] else None
        t = torch.randint(0, V, lead, generator=g, device=DEV)
        s["mask"] = None
        if case["mask"]:  # sequences end before their padding does, which holds anything
            L = lead[1]
            ends = torch.randint(max(1, L // 2), L + 1, (seqs, 1), generator=g, device=DEV)
            s["mask"] = torch.arange(L, device=DEV) < ends
            h = torch.where(s["mask"][..., None], h, math.nan)
            t = torch.where(s["mask"], t, -100)
        s["hidden"], s["targets"] = h, t
        return s
    H, dk, dv, B = case["heads"], case["dk"], case["dv"], case["batch"]
    # half-lives from a few steps to a few hundred
    s["log_decay"] = torch.log1p(-torch.exp2(-torch.linspace(2.0, 8.0, H, device=DEV)))
    if case["kind"] == "step":
        s["q"], s["k"], s["v"] = rn(B, H, dk), rn(B, H, dk), rn(B, H, dv)
        s["starts"] = torch.rand(B, generator=g, device=DEV) < 0.02 if case["starts"] else None
        s["state"] = torch.randn(B, H, dk, dv, generator=g, device=DEV)
        return s
    T = case["T"]
    s["q"], s["k"], s["v"] = rn(T, B, H, dk), rn(T, B, H, dk), rn(T, B, H, dv)
    s["starts"] = torch.rand(T, B, generator=g, device=DEV) < 0.01 if case["starts"] else None
    s["state"] = torch.randn(B, H, dk, dv, generator=g, device=DEV) if case["state"] else None
    if case["grad"]:
        s["g_out"] = rn(T, B, H, dv)
        s["g_state"] = torch.randn(B, H, dk, dv, generator=g, device=DEV) * 0.1 if case["state"] else None
    return s


# -------------------------------------------------------------------------- the operators


def run(s):
    return {"lce": _run_lce, "mem": _run_mem, "step": _run_step}[s["case"]["kind"]](s)


def _run_lce(s):
    c = s["case"]
    up = F16_SCALE if c["dtype"] == "float16" else 1.0
    if own:
        from swarp_amd import linear_cross_entropy
        leaves = [s["hidden"], s["weight"]] + ([s["bias"]] if c["bias"] else [])
        if not c["grad"]:
            with torch.no_grad():
                r = linear_cross_entropy(s["hidden"], s["weight"], s["targets"], s["bias"], s["mask"])
            return {"loss": r.loss, "logp": r.logp}
        leaves = [t.detach().requires_grad_(True) for t in leaves]
        r = linear_cross_entropy(leaves[0], leaves[1], s["targets"],
                                 leaves[2] if c["bias"] else None, s["mask"])
        (r.loss * up if up != 1.0 else r.loss).backward()
        return {"loss": r.loss.detach(), "logp": r.logp, "grads": [t.grad for t in leaves]}
    n, D, V = c["rows"], c["dim"], c["width"]
    h, w = s["hidden"].reshape(n, D).float(), s["weight"].float()
    on = s["mask"].reshape(n, 1) if c["mask"] else torch.ones(n, 1, dtype=torch.bool, device=DEV)
    h = torch.where(on, h, 0.0)
    z = h @ w.t()
    if c["bias"]:
        z += s["bias"].float()
    at = s["targets"].reshape(n, 1).clamp(min=0)
    z -= z.amax(-1, keepdim=True)
    za = z.gather(-1, at)
    e = torch.exp_(z)
    total = e.sum(-1, keepdim=True)
    logp = torch.where(on, za - torch.log(total), 0.0)
    count = on.sum().clamp(min=1)
    out = {"loss": -logp.sum() / count, "logp": logp.view(s["targets"].shape)}
    if not c["grad"]:
        return out
    weight = on.float() * (up / count)
    d = e.mul_(weight / total)
    d.scatter_add_(-1, at, -weight)
    grads = [(d @ w).to(s["hidden"].dtype).view(s["hidden"].shape), (d.t() @ h).to(s["weight"].dtype)]
    if c["bias"]:
        grads.append(d.sum(0).to(s["bias"].dtype))
    return dict(out, grads=grads)


def _run_step(s):
    c = s["case"]
    if own:
        from swarp_amd import decay_attention_step
        out = decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["starts"])
        return {"out": out, "state": s["state"]}
    S = s["state"] * torch.exp(s["log_decay"])[:, None, None]
    if c["starts"]:
        S = torch.where(s["starts"][:, None, None, None], 0.0, S)
    S += s["k"].float()[..., :, None] * s["v"].float()[..., None, :]
    s["state"].copy_(S)
    out = (s["q"].float()[..., :, None] * S).sum(-2) * c["dk"] ** -0.5
    return {"out": out.to(s["v"].dtype), "state": s["state"]}


def _rows(x):
    """[T, B, H, D] as [B H, T, D] in float32."""
    return x.float().permute(1, 2, 0, 3).reshape(-1, x.shape[0], x.shape[3])


def _back(x, like):
    """[B H, T, D] as `like` [T, B, H, D] and of its type."""
    T, B, H, D = like.shape
    return x.to(like.dtype).view(B, H, T, D).permute(2, 0, 1, 3).contiguous()


def _run_mem(s):
    c = s["case"]
    if own:
        from swarp_amd import decay_attention
        if not c["grad"]:
            r = decay_attention(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["starts"])
            return {"out": r.out, "state": r.state}
        x = [t.detach().requires_grad_(True) for t in
             [s["q"], s["k"], s["v"]] + ([s["state"]] if c["state"] else [])]
        r = decay_attention(*x[:3], s["log_decay"], x[3] if c["state"] else None, s["starts"])
        if c["state"]:
            d = torch.autograd.grad((r.out, r.state), x, (s["g_out"], s["g_state"]))
        else:
            d = torch.autograd.grad(r.out, x, s["g_out"])
        return {"out": r.out.detach(), "state": r.state.detach(), "grads": list(d)}
    T, B, H, dk, dv = c["T"], c["batch"], c["heads"], c["dk"], c["dv"]
    n, scale = B * H, dk ** -0.5
    q, k, v = _rows(s["q"]) * scale, _rows(s["k"]), _rows(s["v"])
    ld = s["log_decay"].repeat(B)[:, None]                       # [n, 1]
    ep = torch.zeros(n, T + 1, dtype=torch.int32, device=DEV)    # the episode of each step; first: of the state
    if c["starts"]:
        ep[:, 1:] = torch.cumsum(s["starts"].t(), 1).to(torch.int32).repeat_interleave(H, 0)
    S = s["state"].reshape(n, dk, dv) if c["state"] else torch.zeros(n, dk, dv, device=DEV)
    out, kept = torch.empty_like(v), []
    for a in range(0, T, CHUNK):
        b = min(T, a + CHUNK)
        A, w, u, whole = _weights(ld, ep[:, a:b + 1])
        qc, kc, vc = q[:, a:b], k[:, a:b], v[:, a:b]
        out[:, a:b] = torch.matmul(torch.matmul(qc, kc.transpose(1, 2)) * A, vc) + torch.matmul(qc * w, S)
        if c["grad"]:
            kept.append(S)
        S = whole * S + torch.matmul((kc * u).transpose(1, 2), vc)
    res = {"out": _back(out, s["v"]), "state": S.view(B, H, dk, dv)}
    if not c["grad"]:
        return res
    do = _rows(s["g_out"])
    dS = s["g_state"].reshape(n, dk, dv) if c["state"] else torch.zeros(n, dk, dv, device=DEV)
    dq, dk_, dv_ = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for a in reversed(range(0, T, CHUNK)):
        b = min(T, a + CHUNK)
        A, w, u, whole = _weights(ld, ep[:, a:b + 1])
        qc, kc, vc, dc = q[:, a:b], k[:, a:b], v[:, a:b], do[:, a:b]
        P = torch.matmul(qc, kc.transpose(1, 2)) * A
        dP = torch.matmul(dc, vc.transpose(1, 2)) * A
        S0 = kept.pop()
        dq[:, a:b] = (torch.matmul(dP, kc) + w * torch.matmul(dc, S0.transpose(1, 2))) * scale
        dk_[:, a:b] = torch.matmul(dP.transpose(1, 2), qc) + u * torch.matmul(vc, dS.transpose(1, 2))
        dv_[:, a:b] = torch.matmul(P.transpose(1, 2), dc) + u * torch.matmul(kc, dS)
        dS = whole * dS + torch.matmul((qc * w).transpose(1, 2), dc)
    grads = [_back(dq, s["q"]), _back(dk_, s["k"]), _back(dv_, s["v"])]
    return dict(res, grads=grads + ([dS.view(B, H, dk, dv)] if c["state"] else []))


def _weights(ld, ep):
    """Of a chunk of L steps whose episodes are ep[:, 1:]: step i's weight at step t [n, L, L], the
    entering state's at step t [n, L, 1], step i's in the leaving state [n, L, 1] and the entering
    state's there [n, 1, 1]."""
    L = ep.shape[1] - 1
    t = torch.arange(L, device=DEV)
    here, before, last = ep[:, 1:], ep[:, :1], ep[:, -1:]
    A = torch.exp(ld[..., None] * (t[:, None] - t).clamp(min=0))
    A = torch.where((here[:, :, None] == here[:, None]) & (t[:, None] >= t), A, 0.0)
    w = torch.where(here == before, torch.exp(ld * (t + 1)), 0.0)
    u = torch.where(here == last, torch.exp(ld * (L - 1 - t)), 0.0)
    whole = torch.where(before == last, torch.exp(ld * L), 0.0)
    return A, w[..., None], u[..., None], whole[..., None]


# ------------------------------------------------------------------------- what it costs


def work(case):
    size = {"float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
    if case["kind"] == "lce":
        n, D, V = case["rows"], case["dim"], case["width"]
        on = 0.75 * n if case["mask"] else n  # sequences end between a half and the whole
        passes = 2 if case["grad"] else 1
        return {"bytes": int(passes * size * (D * (V + n) + (V if case["bias"] else 0)) + 13 * n),
                "flops": int((6 if case["grad"] else 2) * on * D * V)}
    n, dk, dv = case["batch"] * case["heads"], case["dk"], case["dv"]
    if case["kind"] == "step":
        return {"bytes": n * (2 * 4 * dk * dv + 2 * size * (dk + dv)), "flops": n * 5 * dk * dv}
    states = 4 * n * dk * dv * ((1 + case["state"]) + (2 * case["state"] if case["grad"] else 0))
    tokens = case["T"] * n * size * 2 * (dk + dv) + (case["T"] * case["batch"] if case["starts"] else 0)
    if case["grad"]:
        tokens += case["T"] * n * size * 2 * (dk + dv)
    return {"bytes": states + tokens, "flops": case["T"] * n * dk * dv * (16 if case["grad"] else 4)}


# ------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    """What ``run`` returns, from the definitions in float64 (gradients by differentiation)."""
    if case["kind"] == "mem" and case["T"] ** 2 * case["batch"] * case["heads"] > 150_000_000_000:
        return None
    s = prepare(case, seed)
    return {"lce": _exact_lce, "mem": _exact_mem, "step": _exact_step}[case["kind"]](s)


def _exact_lce(s):
    c = s["case"]
    on = s["mask"] if c["mask"] else torch.ones_like(s["targets"], dtype=torch.bool)
    x = [s["hidden"].double(), s["weight"].double()] + ([s["bias"].double()] if c["bias"] else [])
    x = [t.requires_grad_(c["grad"]) for t in x]
    z = x[0][on] @ x[1].t()
    if c["bias"]:
        z = z + x[2]
    logp_on = z.gather(-1, s["targets"][on][:, None])[:, 0] - torch.logsumexp(z, -1)
    loss = -logp_on.sum() / max(1, int(on.sum()))
    logp = torch.zeros(on.shape, dtype=torch.float64, device=DEV)
    logp[on] = logp_on.detach()
    out = {"loss": loss.detach(), "logp": logp}
    if c["grad"]:
        out["grads"] = list(torch.autograd.grad(loss * (F16_SCALE if c["dtype"] == "float16" else 1.0), x))
    return out


def _exact_step(s):
    keep = torch.exp(s["log_decay"].double())[:, None, None]
    if s["case"]["starts"]:
        keep = keep * (~s["starts"]).double()[:, None, None, None]
    S = s["state"].double() * keep + torch.einsum("bhi,bhj->bhij", s["k"].double(), s["v"].double())
    return {"out": torch.einsum("bhi,bhij->bhj", s["q"].double(), S) / math.sqrt(s["case"]["dk"]),
            "state": S}


def _exact_mem(s):
    """Every step against every earlier one, a few sequences (or a block of their rows) at a time."""
    c = s["case"]
    T, B, H, dk, dv = c["T"], c["batch"], c["heads"], c["dk"], c["dv"]
    t = torch.arange(T, device=DEV)
    at_once = max(1, 40_000_000 // (T * T))
    rows = T if c["grad"] else max(1, min(T, 40_000_000 // T))
    names = ["q", "k", "v"] + (["state"] if c["state"] else [])
    out = torch.empty(T, B, H, dv, dtype=torch.float64, device=DEV)
    state = torch.empty(B, H, dk, dv, dtype=torch.float64, device=DEV)
    grads = [torch.empty(s[k].shape, dtype=torch.float64, device=DEV) for k in names] if c["grad"] else []
    for h in range(H):
        g = s["log_decay"][h].double()
        for a in range(0, B, at_once):
            cut = slice(a, min(B, a + at_once))

            def part(k, source=s, cut=cut, h=h):
                x = source[k]
                return (x[cut, h] if k.endswith("state") else x[:, cut, h].transpose(0, 1)).double()
            x = [part(k).requires_grad_(c["grad"]) for k in names]
            q, k, v = x[:3]
            ep = torch.zeros(q.shape[0], T, dtype=torch.int64, device=DEV)
            if c["starts"]:
                ep = torch.cumsum(s["starts"][:, cut].t().long(), 1)
            pieces = []
            for r in range(0, T, rows):
                tr = t[r:r + rows, None]
                w = torch.exp(g * (tr - t).clamp(min=0)) * (tr >= t)
                w = w * (ep[:, r:r + rows, None] == ep[:, None, :])
                o = ((q[:, r:r + rows] @ k.transpose(1, 2).contiguous()) * w) @ v
                if c["state"]:
                    first = torch.exp(g * (tr + 1)) * (ep[:, r:r + rows, None] == 0)
                    o = o + first * (q[:, r:r + rows] @ x[3])
                pieces.append(o / math.sqrt(dk))
            o = torch.cat(pieces, 1)
            u = torch.exp(g * (T - 1 - t))[:, None] * (ep == ep[:, -1:])[..., None]
            S = (k * u).transpose(1, 2).contiguous() @ v
            if c["state"]:
                S = S + torch.exp(g * T) * (ep[:, -1] == 0)[:, None, None] * x[3]
            out[:, cut, h], state[cut, h] = o.detach().transpose(0, 1), S.detach()
            if not c["grad"]:
                continue
            if c["state"]:
                d = torch.autograd.grad((o, S), x, (part("g_out"), part("g_state")))
            else:
                d = torch.autograd.grad(o, x, part("g_out"))
            for name, to, y in zip(names, grads, d):
                if name == "state":
                    to[cut, h] = y
                else:
                    to[:, cut, h] = y.transpose(0, 1)
    res = {"out": out, "state": state}
    return dict(res, grads=grads) if c["grad"] else res
