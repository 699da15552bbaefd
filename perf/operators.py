"""The operators of a policy update, as cases that can be timed and compared.

What follows a rollout of the simulator when a policy is trained on it:

* ``gae``    generalised advantage estimation of a rollout's rewards and values (and the adjoint
  of that scan, for a loss that is differentiated through the rewards);
* ``cat``    the clipped policy loss with KL and entropy terms of a categorical head -- action
  bins of an agent, or tokens of a vocabulary -- and its gradient;
* ``gauss``  the same loss of a diagonal Gaussian head over the agents' continuous actions;
* ``adamw``  one AdamW step over all tensors of a policy, its moments in 32 bits or in 8.

``run`` computes them in plain torch, or, where ``own`` is true, by the package's operators.
"""

import math

import torch

own = False

DEV = "cuda:0"
GROUP = 256                   # elements that share an exponent in an 8-bit moment
LR, B1, B2, EPS, WD = 3e-4, 0.9, 0.999, 1e-8, 0.01
CLIP = 0.2
F16_SCALE = 4096.0            # a loss with float16 heads is scaled, as mixed precision does it
STEP = 10                     # the optimizer step that is timed


def listed():
    return [
        # the smallest rollout of the repository (64 envs x 4 agents, 10 steps): launch latency
        _gae("gae_10x64x4", 10, 64, 4),
        # a rollout of the benchmark workload, 32 steps of 16000 envs x 16 agents
        _gae("gae_32x16000x16", 32, 16000, 16),
        # long episodes kept row by row, odd length, bootstrapped at time limits, with the adjoint
        _gae("gae_rows_96x4095_grad", 4095, 24, 4, layout="rows", grad=True, final=True),
        # continuous accelerations of the benchmark workload, a standard deviation per dimension
        _gauss("gauss_8192000x2", 16000 * 16 * 32, 2),
        # quadrotors' four thrusts, a network's own standard deviations in bfloat16, dead agents
        # masked, a KL term towards a reference policy
        _gauss("gauss_1048573x4_bf16", 1048573, 4, dtype="bfloat16", rows_std=True, mask=True,
               ref=True),
        # a minibatch of nine compass actions: launch latency
        _cat("cat_2560x9", 2560, 9),
        # 5 x 5 acceleration bins of the benchmark workload, unavailable actions at -inf
        _cat("cat_4096000x25_bf16", 16000 * 16 * 16, 25, dtype="bfloat16", ban=True),
        # sequences of tokens, an odd vocabulary, padded ends masked, KL towards a reference
        _cat("cat_8x1023x50001_bf16", 8 * 1023, 50001, dtype="bfloat16", seqs=8, mask=True,
             ref=True),
        # few rows of a long vocabulary in float32
        _cat("cat_96x131072", 96, 131072, ref=True),
        # a small policy: 12 tensors, gradient norm clipped: launch latency
        _adamw("adamw_12x70k", 12, 70_000, clip=True),
        # a large policy in float32
        _adamw("adamw_48x100m", 48, 100_000_000),
        # a larger one in bfloat16 with its moments in 8 bits
        _adamw("adamw_48x150m_bf16_8bit", 48, 150_000_000, dtype="bfloat16", bits=8),
    ]


def _named(name, case):
    return dict(case, name=name) if name else case


def _gae(name, T, envs, agents, layout="time", grad=False, final=False, dtype="float32"):
    return _named(name, {"kind": "gae", "T": T, "envs": envs, "agents": agents, "layout": layout,
                         "grad": grad, "final": final, "dtype": dtype})


def _gauss(name, rows, dim, dtype="float32", rows_std=False, mask=False, ref=False):
    return _named(name, {"kind": "gauss", "rows": rows, "dim": dim, "dtype": dtype,
                         "rows_std": rows_std, "mask": mask, "ref": ref})


def _cat(name, rows, width, dtype="float32", seqs=0, mask=False, ref=False, ban=False):
    return _named(name, {"kind": "cat", "rows": rows, "width": width, "dtype": dtype,
                         "seqs": seqs, "mask": mask, "ref": ref, "ban": ban})


def _adamw(name, tensors, total, dtype="float32", bits=32, clip=False):
    return _named(name, {"kind": "adamw", "tensors": tensors, "total": total, "dtype": dtype,
                         "bits": bits, "clip": clip})


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("gae", "gauss", "cat", "cat", "adamw"))
    if kind == "gae":
        T, A = _log(rng, 1, 4500), _log(rng, 1, 64)
        most = max(1, 8_000_000 // (T * A))
        return _gae("", T, _log(rng, 1, min(16000, most)), A, rng.choice(("time", "time", "rows")),
                    rng.random() < 0.4, rng.random() < 0.3,
                    "float64" if rng.random() < 0.2 else "float32")
    if kind == "gauss":
        D = rng.choice((1, 2, 2, 3, 4, 4, 6, 9, 17, 40))
        return _gauss("", _log(rng, 200, 16_000_000 // D), D,
                      rng.choice(("float32", "float32", "bfloat16", "float16")),
                      rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)
    if kind == "cat":
        V = _log(rng, 2, 150_000)
        rows = _log(rng, 16, min(4_000_000, 200_000_000 // V))
        seqs = rng.choice((0, 0, rng.randint(1, 8)))
        return _cat("", rows // seqs * seqs if seqs else rows, V,
                    rng.choice(("float32", "bfloat16", "bfloat16", "float16")), seqs,
                    rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.3)
    dtype = rng.choice(("float32", "float32", "bfloat16"))
    bits = rng.choice((32, 8))
    return _adamw("", rng.randint(1, 60), _log(rng, 5_000, 60_000_000), dtype, bits,
                  bits == 32 and rng.random() < 0.5)


# ------------------------------------------------------------------------------- inputs


def _sizes(case):
    """Element counts of a policy's tensors: square-ish matrices, each with its bias."""
    n = case["tensors"]
    w = max(1, int(math.sqrt(2.0 * case["total"] / n)))
    return [w * (w + k % 3) if k % 2 == 0 else w + k % 5 for k in range(n)]


def _slots(sizes):
    """Where each tensor's moments start in the flat state, and its length."""
    at, n = [], 0
    for s in sizes:
        at.append(n)
        n += -(-s // GROUP) * GROUP
    return at, n


def _coefs(case):
    """(kl, entropy) of the loss."""
    return (0.05 if case["ref"] else 0.0), 0.01


def _apart(d):
    """Log ratios kept 1e-3 away from the clip bounds: the gradient jumps there, and either side
    of the jump is a right answer for a ratio that is a rounding away from it."""
    lo, hi = math.log(1 - CLIP), math.log(1 + CLIP)
    d = torch.where((d - lo).abs() < 1e-3, torch.full_like(d, lo - 1e-3), d)
    return torch.where((d - hi).abs() < 1e-3, torch.full_like(d, hi + 1e-3), d)


def _row_inputs(case, g, logp, shape):
    """The per-row inputs of a policy loss beside the actions: ``logp`` is the current one."""
    n = logp.numel()

    def rn(s):
        return torch.randn(n, generator=g, device=DEV) * s
    d = _apart(rn(0.12).double())
    x = {"old_logp": (logp.double() - d).float().view(shape), "advantages": rn(1.0).view(shape),
         "ref_logp": (logp.double() + rn(0.3).double()).float().view(shape) if case["ref"] else None,
         "mask": None}
    if case["mask"]:
        x["mask"] = (torch.rand(n, generator=g, device=DEV) < 0.8).view(shape)
        # what a masked row holds is nobody's: an unfinished episode's advantage may be anything
        x["advantages"] = torch.where(x["mask"], x["advantages"], math.nan)
    return x


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1) + 17)
    s = {"case": case}
    if case["kind"] == "gae":
        T, E, A, dt = case["T"], case["envs"], case["agents"], getattr(torch, case["dtype"])
        rows = case["layout"] == "rows"

        def shape(t, *lead):
            return (*lead, t) if rows else (t, *lead)

        def rn(*sh):
            return torch.randn(*sh, generator=g, device=DEV).to(dt)
        s["rewards"], s["values"] = rn(*shape(T, E, A)) * 0.1, rn(*shape(T + 1, E, A))
        s["terminated"] = torch.rand(shape(T, E), generator=g, device=DEV) < 0.01
        s["truncated"] = torch.rand(shape(T, E), generator=g, device=DEV) < 0.01
        s["final_values"] = rn(*shape(T, E, A)) if case["final"] else None
        if case["grad"]:
            s["g_adv"], s["g_ret"] = rn(*shape(T, E, A)), rn(*shape(T, E, A))
        return s
    if case["kind"] == "adamw":
        sizes = _sizes(case)
        at, n = _slots(sizes)
        dt = getattr(torch, case["dtype"])
        s["params"] = [(torch.randn(k, generator=g, device=DEV) * 0.02).to(dt) for k in sizes]
        s["grads"] = [(torch.randn(k, generator=g, device=DEV) * 1e-3).to(dt) for k in sizes]
        s["seed"] = int(torch.randint(1 << 30, (1,), generator=g, device=DEV))
        m = torch.randn(n, generator=g, device=DEV) * 3e-4
        v = torch.rand(n, generator=g, device=DEV) * 2e-6
        for k, a in zip(sizes, at):  # the padding behind a tensor is zero
            m[a + k:a + -(-k // GROUP) * GROUP] = 0
            v[a + k:a + -(-k // GROUP) * GROUP] = 0
        if case["bits"] == 8:
            half = torch.full((n,), 1 << 15, dtype=torch.int32, device=DEV)
            s["m"], s["m_base"] = _pack(m, half, True)
            s["v"], s["v_base"] = _pack(v, half, False)
        else:
            s["m"], s["v"], s["m_base"], s["v_base"] = m, v, None, None
        return s
    n, dt = case["rows"], getattr(torch, case["dtype"])
    if case["kind"] == "gauss":
        D = case["dim"]
        mean = (torch.randn(n, D, generator=g, device=DEV) * 0.5).to(dt)
        ls = (torch.randn((n, D) if case["rows_std"] else (D,), generator=g, device=DEV) * 0.2
              - 0.7).to(dt)
        z = torch.randn(n, D, generator=g, device=DEV)
        act = mean.float() + ls.float().exp() * z
        q = (act.double() - mean.double()) * torch.exp(-ls.double())
        logp = (-0.5 * q * q - ls.double() - 0.5 * math.log(2 * math.pi)).sum(-1)
        s.update(mean=mean, log_std=ls, actions=act, **_row_inputs(case, g, logp, (n,)))
        return s
    V = case["width"]
    # a policy in training: a few likely actions, a long tail
    shape = (case["seqs"], n // case["seqs"]) if case["seqs"] else (n,)
    full = (shape[0], shape[1] + 1, V) if case["seqs"] else (n, V)
    x = torch.randn(full, generator=g, device=DEV, dtype=torch.float32) * 2.0
    if case["ban"]:  # actions that are not open to an agent; the first always is
        x[..., 1:].masked_fill_(torch.rand(*full[:-1], V - 1, generator=g, device=DEV) < 0.15,
                                -math.inf)
    x = x.to(dt)
    # the last position of a sequence predicts nothing: a view, not a copy, goes on
    x = x[:, :-1] if case["seqs"] else x
    rows = x.reshape(n, V).float()
    u = torch.rand(n, V, generator=g, device=DEV).clamp_(1e-12, 1 - 1e-7)
    act = torch.argmax(rows - torch.log(-torch.log(u)), dim=-1)
    del u
    logp = (rows.gather(-1, act[:, None])[:, 0] - torch.logsumexp(rows, -1))
    s.update(logits=x, **_row_inputs(case, g, logp, shape))
    s["actions"] = act.view(shape)
    if case["mask"]:
        s["actions"] = torch.where(s["mask"], s["actions"], -100)
    return s


# -------------------------------------------------------------------------- the operators


def run(s):
    return {"gae": _run_gae, "gauss": _run_gauss, "cat": _run_cat,
            "adamw": _run_adamw}[s["case"]["kind"]](s)


def _run_gae(s):
    c = s["case"]
    dim = -1 if c["layout"] == "rows" else 0
    flags = (s["terminated"], s["truncated"])
    if own:
        from swarp_amd import gae
        if not c["grad"]:
            adv, ret = gae(s["rewards"], s["values"], *flags, s["final_values"], gamma=0.99,
                           lam=0.95, time_dim=dim)
            return {"advantages": adv, "returns": ret}
        x = [s["rewards"], s["values"]] + ([s["final_values"]] if c["final"] else [])
        x = [t.detach().requires_grad_(True) for t in x]
        adv, ret = gae(x[0], x[1], *flags, x[2] if c["final"] else None, gamma=0.99, lam=0.95,
                       time_dim=dim)
        d = torch.autograd.grad((adv, ret), x, (s["g_adv"], s["g_ret"]))
        return {"advantages": adv.detach(), "returns": ret.detach(), "grads": list(d)}
    r, v = s["rewards"].movedim(dim, 0), s["values"].movedim(dim, 0)
    term = s["terminated"].movedim(dim, 0)[..., None]
    trunc = s["truncated"].movedim(dim, 0)[..., None]
    fin = s["final_values"].movedim(dim, 0) if c["final"] else None
    nxt = v[1:] if fin is None else torch.where(trunc, fin, v[1:])
    delta = r + 0.99 * torch.where(term, 0.0, nxt) - v[:-1]
    carry = (0.99 * 0.95 * (~(term | trunc)).to(r.dtype)).expand_as(r)
    adv = _scan(delta.flip(0), carry.flip(0)).flip(0)
    out = {"advantages": adv.movedim(0, dim), "returns": (adv + v[:-1]).movedim(0, dim)}
    if not c["grad"]:
        return out
    g_a, g_r = s["g_adv"].movedim(dim, 0), s["g_ret"].movedim(dim, 0)
    before = torch.cat([torch.zeros_like(carry[:1]), carry[:-1]])
    G = _scan(g_a + g_r, before)
    dv = torch.zeros_like(v)
    dv[:-1] = g_r - G
    dv[1:] += 0.99 * torch.where(term if fin is None else term | trunc, 0.0, G)
    grads = [G, dv] + ([0.99 * torch.where(trunc & ~term, G, 0.0)] if c["final"] else [])
    return dict(out, grads=[t.movedim(0, dim) for t in grads])


def _scan(d, c):
    """x_t = d_t + c_t x_{t-1} along the first axis, by doubling."""
    d, c, k = d.clone(), c.clone(), 1
    while k < d.shape[0]:
        d[k:], c[k:] = d[k:] + c[k:] * d[:-k], c[k:] * c[:-k]
        k *= 2
    return d


def _surrogate(s, logp, entropy):
    """Per-row weight, d(loss)/d(logp) / weight, and the loss and its means from the rows'
    log-probabilities and entropies (float32)."""
    c = s["case"]
    kl_c, ent_c = _coefs(c)
    old, adv = s["old_logp"].reshape(-1), s["advantages"].reshape(-1)
    ref = s["ref_logp"].reshape(-1) if c["ref"] else old
    on = s["mask"].reshape(-1) if c["mask"] else torch.ones_like(old, dtype=torch.bool)
    w = on.float() / on.sum().clamp(min=1)
    ratio = torch.exp(logp - old)
    bounded = ratio.clamp(1 - CLIP, 1 + CLIP)
    first, second = ratio * adv, bounded * adv
    e = ref - logp
    kl = torch.expm1(e) - e
    per_row = -torch.minimum(first, second) + kl_c * kl - ent_c * entropy
    g = torch.where(first <= second, -first, 0.0) - kl_c * torch.expm1(e)

    def mean(x):
        return (torch.where(on, x, 0.0) * w).sum()
    out = {"loss": mean(per_row), "entropy": mean(entropy), "kl": mean(kl),
           "clip_fraction": mean((second < first).float()),
           "logp": torch.where(on, logp, 0.0).view(s["old_logp"].shape)}
    w = w * F16_SCALE if c["dtype"] == "float16" else w
    return on[:, None], w[:, None], torch.where(on, g, 0.0)[:, None], out


def _call(s, op, *heads):
    """The package's loss and its backward pass to the heads."""
    kl_c, ent_c = _coefs(s["case"])
    heads = [h.detach().requires_grad_(True) for h in heads]
    r = op(*heads, s["actions"], s["old_logp"], s["advantages"], s["ref_logp"], s["mask"],
           clip=CLIP, kl_coef=kl_c, entropy_coef=ent_c)
    (r.loss * F16_SCALE if s["case"]["dtype"] == "float16" else r.loss).backward()
    return {"loss": r.loss.detach(), "entropy": r.entropy, "kl": r.kl,
            "clip_fraction": r.clip_fraction, "logp": r.logp, "grads": [h.grad for h in heads]}


def _run_gauss(s):
    if own:
        from swarp_amd import gaussian_policy_loss
        return _call(s, gaussian_policy_loss, s["mean"], s["log_std"])
    c = s["case"]
    mean, ls = s["mean"].float(), s["log_std"].float()
    inv = torch.exp(-ls)
    z = (s["actions"] - mean) * inv
    logp = (-0.5 * z * z - ls - 0.5 * math.log(2 * math.pi)).sum(-1)
    entropy = (ls + 0.5 * math.log(2 * math.pi * math.e)).sum(-1).expand(c["rows"])
    on, w, g, out = _surrogate(s, logp, entropy)
    ent_c = _coefs(c)[1]
    d_mean = torch.where(on, w * g * z * inv, 0.0)
    d_ls = torch.where(on, w * (g * (z * z - 1.0) - ent_c), 0.0)
    d_ls = d_ls if c["rows_std"] else d_ls.sum(0)
    return dict(out, grads=[d_mean.to(s["mean"].dtype), d_ls.to(s["log_std"].dtype)])


def _run_cat(s):
    if own:
        from swarp_amd import categorical_policy_loss
        return _call(s, categorical_policy_loss, s["logits"])
    c = s["case"]
    x = s["logits"].reshape(c["rows"], c["width"]).float()
    z = x - x.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    p, lp = e / total, z - torch.log(total)
    lp0 = torch.where(p > 0, lp, 0.0)
    entropy = -(p * lp0).sum(-1)
    at = s["actions"].reshape(-1, 1).clamp(min=0)
    on, w, g, out = _surrogate(s, lp.gather(-1, at)[:, 0], entropy)
    ent_c = _coefs(c)[1]
    d = p * (w * ent_c * (lp0 + entropy[:, None]) - w * g)
    d.scatter_add_(-1, at, w * g)
    return dict(out, grads=[torch.where(on, d, 0.0).to(s["logits"].dtype).view(s["logits"].shape)])


def _run_adamw(s):
    c = s["case"]
    at, n = _slots(_sizes(c))
    if own:
        from swarp_amd import AdamWState, adamw_step
        state = AdamWState(s["m"], s["v"], s["m_base"], s["v_base"], None)
        norm = adamw_step(s["params"], s["grads"], state, STEP, lr=LR, betas=(B1, B2), eps=EPS,
                          weight_decay=WD, max_grad_norm=1.0 if c["clip"] else None,
                          seed=s["seed"])
        m, v = state.moments()
        return {"params": list(s["params"]), "m": m, "v": v, "norm": norm}
    norm, scale = None, None
    if c["clip"]:
        norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
        scale = (1.0 / (norm + 1e-6)).clamp(max=1.0)
    b1, b2 = _f32(B1), _f32(B2)
    a1, a2 = _f32(1 - B1), _f32(1 - B2)
    lr_t, v_t = LR / (1 - B1 ** STEP), 1 / math.sqrt(1 - B2 ** STEP)
    for p, g, a in zip(s["params"], s["grads"], at):
        k, pad = p.numel(), -(-p.numel() // GROUP) * GROUP
        g, w = g.float(), p.float()
        g = g if scale is None else g * scale
        m, v = _moments(s, a, pad)
        m = m[:k] * b1 + g * a1
        v = v[:k] * b2 + g * g * a2
        w = w * (1 - LR * WD) - lr_t * (m / (v.sqrt() * v_t + EPS))
        if c["bits"] == 8:
            m, v = (torch.cat([t, t.new_zeros(pad - k)]) for t in (m, v))
            r = _hash(a, pad, s["seed"])
            s["m"][a:a + pad], s["m_base"][a // GROUP:(a + pad) // GROUP] = _pack(m, r >> 16 & 0xffff, True)
            s["v"][a:a + pad], s["v_base"][a // GROUP:(a + pad) // GROUP] = _pack(v, r & 0xffff, False)
        else:
            s["m"][a:a + k], s["v"][a:a + k] = m, v
        if p.dtype == torch.bfloat16:  # stochastic: an update is mostly below half a step
            r = _mix(_hash(a, pad, s["seed"])[:k]) & 0xffff
            bits = w.view(torch.int32)
            p.copy_(((bits + r) & -65536).view(torch.float32).to(torch.bfloat16))
        else:
            p.copy_(w)
    m, v = _moments(s, 0, n)
    return {"params": list(s["params"]), "m": m, "v": v, "norm": norm}


def _f32(x):
    """The float32 nearest to x."""
    return float(torch.tensor(x, dtype=torch.float32))


def _moments(s, a, k):
    """Both moments of k elements from a on, as the values that they stand for."""
    if s["case"]["bits"] == 32:
        return s["m"][a:a + k], s["v"][a:a + k]
    g = slice(a // GROUP, (a + k) // GROUP)
    return _unpack(s["m"][a:a + k], s["m_base"][g], True), _unpack(s["v"][a:a + k], s["v_base"][g], False)


def _mix(x):
    """One round of multiply and shift over 32-bit integers (they wrap)."""
    x = x * _i32(0xBB67AE85)
    x = x ^ (x >> 15 & 0x1ffff)
    x = x * _i32(0xA54FF53B)
    return x ^ (x >> 16 & 0xffff)


def _i32(x):
    return x - (1 << 32) if x >= 1 << 31 else x


def _hash(a, k, seed):
    """32 random bits of elements a .. a + k of the flat state."""
    x = torch.arange(a, a + k, dtype=torch.int64, device=DEV).to(torch.int32)
    return _mix(x * _i32(0x9E3779B1) + _i32(seed & 0xffffffff))


def _pack(x, r, signed):
    """8-bit codes of x and the base of each group: the top bits of the float -- (sign,) exponent
    counted from the group's base, three of mantissa -- after adding 16 random bits r below."""
    reach, top = (15, 127) if signed else (31, 255)
    bits = x.view(torch.int32)
    mag = (bits & 0x7fffffff).clamp(max=0x7ff00000).view(-1, GROUP)
    most = (mag.amax(-1) + 0xfffff) >> 20
    base = ((most >> 3) - reach).clamp(min=0)
    code = ((mag + (r.view(-1, GROUP) << 4 | 8)) >> 20) - (base[:, None] << 3)
    code = torch.maximum(code, torch.zeros_like(code) if signed else (mag > 0).int()).clamp(max=top)
    if signed:
        code = code | (bits.view(-1, GROUP) >> 24 & 128)
    return code.view(-1).to(torch.uint8), base.to(torch.uint8)


def _unpack(code, base, signed):
    q = code.view(-1, GROUP).int()
    low = q & 127 if signed else q
    bits = torch.where(low > 0, (low + (base.int()[:, None] << 3)) << 20, 0)
    if signed:
        bits = bits | (q & 128) << 24
    return bits.view(-1).view(torch.float32)


# ------------------------------------------------------------------------- what it costs


def work(case):
    size = {"float32": 4, "float64": 8, "bfloat16": 2, "float16": 2}[case["dtype"]]
    if case["kind"] == "gae":
        n = case["T"] * case["envs"] * case["agents"]
        flags = 2 * case["T"] * case["envs"]
        arrays = 4 + case["final"] + (4 + case["final"] if case["grad"] else 0)
        return {"bytes": n * size * arrays + flags * (1 + case["grad"]),
                "flops": n * (8 + 6 * case["grad"])}
    if case["kind"] == "adamw":
        n = sum(_sizes(case))
        if case["bits"] == 8:  # codes read and written, and written out as values
            return {"bytes": n * (3 * size + 4 + 8), "flops": 30 * n}
        return {"bytes": n * (3 * size + 16), "flops": 15 * n}
    n = case["rows"]
    row = 4 + 4 + 4 + (4 if case["ref"] else 0) + (1 if case["mask"] else 0)
    if case["kind"] == "gauss":
        D = case["dim"]
        return {"bytes": n * (row + D * (2 * size + 4 + (2 * size if case["rows_std"] else 0))),
                "flops": n * (20 + 14 * D)}
    return {"bytes": n * (row + 8 + 2 * case["width"] * size), "flops": 12 * n * case["width"]}


# ------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    """What ``run`` returns, from the definitions in float64 (gradients by differentiation)."""
    s = prepare(case, seed)
    return {"gae": _exact_gae, "gauss": _exact_loss, "cat": _exact_loss,
            "adamw": _exact_adamw}[case["kind"]](s)


def _exact_gae(s):
    c = s["case"]
    dim = -1 if c["layout"] == "rows" else 0
    x = [s[k].double().movedim(dim, 0).contiguous().requires_grad_(c["grad"])
         for k in ("rewards", "values", "final_values") if s[k] is not None]
    r, v = x[0], x[1]
    stop = s["terminated"].movedim(dim, 0)[..., None].expand_as(r)
    cut = s["truncated"].movedim(dim, 0)[..., None].expand_as(r)
    nxt = torch.where(cut, x[2], v[1:]) if c["final"] else v[1:]
    delta = r + 0.99 * torch.where(stop, torch.zeros_like(nxt), nxt) - v[:-1]
    ends = stop | cut
    # the definition, backwards in time
    rows, a = [None] * c["T"], torch.zeros_like(delta[0])
    for t, (d, e) in reversed(list(enumerate(zip(delta.unbind(0), ends.unbind(0))))):
        a = d + torch.where(e, torch.zeros_like(a), 0.99 * 0.95 * a)
        rows[t] = a
    adv = torch.stack(rows)
    ret = adv + v[:-1]

    def back(t):
        return t.detach().movedim(0, dim)
    out = {"advantages": back(adv), "returns": back(ret)}
    if c["grad"]:
        g = [s[k].double().movedim(dim, 0) for k in ("g_adv", "g_ret")]
        out["grads"] = [back(t) for t in torch.autograd.grad((adv, ret), x, g)]
    return out


def _exact_loss(s):
    c = s["case"]
    kl_c, ent_c = _coefs(c)
    on = s["mask"] if c["mask"] else torch.ones_like(s["old_logp"], dtype=torch.bool)
    if c["kind"] == "gauss":
        heads = [s[k].double().requires_grad_(True) for k in ("mean", "log_std")]
        var = torch.exp(2 * heads[1])
        sq = (s["actions"].double() - heads[0]) ** 2 / var
        logp = -0.5 * (sq + torch.log(2 * math.pi * var)).sum(-1)
        entropy = (0.5 * torch.log(2 * math.pi * math.e * var)).sum(-1).expand_as(logp)
    else:
        heads = [s["logits"].double().requires_grad_(True)]
        lsm = torch.log_softmax(heads[0], -1)
        logp = lsm.gather(-1, s["actions"].clamp(min=0)[..., None])[..., 0]
        safe = torch.where(torch.isinf(lsm), torch.zeros_like(lsm), lsm)
        entropy = -(torch.exp(lsm) * safe).sum(-1)
    logp_on, entropy_on, old = logp[on], entropy[on], s["old_logp"].double()[on]
    adv = s["advantages"].double()[on]
    e = (s["ref_logp"].double()[on] if c["ref"] else old) - logp_on
    ratio = torch.exp(logp_on - old)
    low = torch.where(adv >= 0, torch.clamp(ratio, max=1 + CLIP), torch.clamp(ratio, min=1 - CLIP))
    kl = torch.special.expm1(e) - e
    n = max(1, int(on.sum()))
    loss = (-low * adv + kl_c * kl - ent_c * entropy_on).sum() / n
    grads = torch.autograd.grad(loss * (F16_SCALE if c["dtype"] == "float16" else 1.0), heads)
    clipped = ((adv > 0) & (ratio > 1 + CLIP)) | ((adv < 0) & (ratio < 1 - CLIP))
    return {"loss": loss.detach(), "entropy": entropy_on.detach().sum() / n,
            "kl": kl.detach().sum() / n, "clip_fraction": clipped.double().sum() / n,
            "logp": torch.where(on, logp.detach(), torch.zeros_like(old[:1])), "grads": list(grads)}


def _exact_adamw(s):
    c = s["case"]
    at, n = _slots(_sizes(c))
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in s["grads"]))
    scale = min(1.0, 1.0 / (norm + 1e-6)) if c["clip"] else 1.0
    m0, v0 = (t.double() for t in _moments(s, 0, n))
    params, ms, vs = [], torch.zeros_like(m0), torch.zeros_like(v0)
    for p, g, a in zip(s["params"], s["grads"], at):
        k, g = p.numel(), g.double() * scale
        m = B1 * m0[a:a + k] + (1 - B1) * g
        v = B2 * v0[a:a + k] + (1 - B2) * g ** 2
        ms[a:a + k], vs[a:a + k] = m, v
        update = m / (1 - B1 ** STEP) / (torch.sqrt(v / (1 - B2 ** STEP)) + EPS)
        params.append(p.double() - LR * (update + WD * p.double()))
    if c["bits"] == 8:  # moments rounded at random have no value of their own
        return {"params": params, "m": None, "v": None, "norm": None}
    return {"params": params, "m": ms, "v": vs,
            "norm": torch.tensor(norm, dtype=torch.float64) if c["clip"] else None}
