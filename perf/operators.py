"""The gated delta rule, its single-token step and the RMS norm around them, as cases that can be timed and checked.

A case is one call of a public entry point: ``gated_delta_rule`` (forward, or forward
and backward), ``gated_delta_step``, ``add_rms_norm`` (forward and backward) or
``add_rms_norm_fp8``.  Where ``own`` is false the same operators are computed in plain
torch.  Heads are the framework's (d = 128), 16 of them unless a case says otherwise;
sequence lengths are those of the benchmark's configs and of the harness's sweep, and
ragged ones between them.
"""

import math

import torch

own = False

DH = 128
EPS = 1e-6
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _rule(name, dtype, B, T, Hk, Hv, train=False, seqs=0, state=False):
    """B sequences of T tokens, or (seqs > 0, B = 1) T tokens packed from that many
    sequences; Hk heads of q and k serve Hv heads of v; state: an initial state is given
    and the final one wanted."""
    return {"name": name, "op": "rule", "dtype": dtype, "B": B, "T": T, "Hk": Hk, "Hv": Hv, "train": train, "seqs": seqs,
            "state": state}


def listed():
    return [
        # a short prompt at the harness sweep's shortest length, state kept for decoding: latency counts
        _rule("rule_bf16_T512", "bf16", 1, 512, 16, 16, state=True),
        # prefill at the benchmark's headline length: few heads, a long axis
        _rule("rule_bf16_T16384", "bf16", 1, 16384, 16, 16, state=True),
        # a packed batch of ragged prompts (one of a single token among them), each q/k head shared by two v heads
        _rule("rule_bf16_packed_T12289", "bf16", 1, 12289, 8, 16, seqs=23, state=True),
        # a training step over a batch, forward and backward: the largest
        _rule("train_bf16_B4_T4096", "bf16", 4, 4096, 16, 16, train=True),
        # a training step on packed sequences with shared heads and carried states
        _rule("train_bf16_packed_T6001", "bf16", 1, 6001, 8, 16, train=True, seqs=7, state=True),
        # full precision, ragged, forward and backward (gradient checks, small models)
        _rule("train_f32_B2_T1537", "f32", 2, 1537, 4, 4, train=True, state=True),
        # decoding one sequence: the smallest call of the rule's kind
        {"name": "step_bf16_N1", "op": "step", "dtype": "bf16", "N": 1, "pool": 4, "Hk": 16, "Hv": 16},
        # decoding a serving batch out of a larger pool of states, some rows padding, shared heads
        {"name": "step_bf16_N203", "op": "step", "dtype": "bf16", "N": 203, "pool": 256, "Hk": 8, "Hv": 16},
        # the residual stream's norm in a training step at the layer's width, forward and backward
        {"name": "norm_bf16_16384x2048", "op": "norm", "dtype": "bf16", "rows": 16384, "D": 2048, "residual": True},
        # q's norm by heads in a training step: short rows, no residual, full precision
        {"name": "norm_f32_24592x128", "op": "norm", "dtype": "f32", "rows": 24592, "D": 128, "residual": False},
        # one token's norm before a product in 8 bits: the smallest call
        {"name": "norm8_bf16_1x2048", "op": "norm8", "dtype": "bf16", "rows": 1, "D": 2048, "residual": True},
        # a prompt's norm before a product in 8 bits, a row count that no tile divides
        {"name": "norm8_bf16_12289x4096", "op": "norm8", "dtype": "bf16", "rows": 12289, "D": 4096, "residual": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rule", "rule", "train", "train", "step", "norm", "norm8"])
    if op in ("rule", "train"):
        train, f32 = op == "train", rng.random() < 0.3
        B = rng.choice([1, 1, 2, 3, 5])
        Hk = rng.choice([1, 2, 4, 8, 16])
        Hv = Hk * rng.choice([1, 1, 2, 3]) if Hk < 16 else 16
        top = (3074 if f32 else 16384) if train else (8192 if f32 else 16384)
        T = _log_int(rng, 1, top // B)
        seqs = rng.choice([0, 0, 0, 2, 9, 31]) if B == 1 and T > 1 else 0
        c = _rule("", "f32" if f32 else "bf16", B, T, Hk, min(Hv, 16), train, min(seqs, T), rng.random() < 0.5)
        if c["Hv"] % Hk:
            c["Hv"] = Hk
    elif op == "step":
        N, Hk = _log_int(rng, 1, 256), rng.choice([1, 4, 8, 16])
        c = {"op": "step", "dtype": rng.choice(["bf16", "bf16", "f32"]), "N": N, "pool": N + rng.randrange(1, 33), "Hk": Hk,
             "Hv": Hk * rng.choice([1, 2]) if Hk < 16 else 16}
    elif op == "norm":
        D = rng.choice([128, 128, 512, 1000, 2048, 4096, 5120, 8192])
        c = {"op": "norm", "dtype": rng.choice(["bf16", "bf16", "f32"]), "rows": _log_int(rng, 1, 33554432 // D), "D": D,
             "residual": rng.random() < 0.7}
    else:
        D = rng.choice([128, 512, 1000, 2048, 4096, 5120, 8192])
        c = {"op": "norm8", "dtype": rng.choice(["bf16", "bf16", "f32"]), "rows": _log_int(rng, 1, 50331648 // D), "D": D,
             "residual": rng.random() < 0.7}
    c.pop("name", None)
    return c


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _unit(x):
    return x / (x.square().sum(-1, keepdim=True) + EPS).sqrt()


def _rule_inputs(g, lead, Hk, Hv, dt):
    """q, k of unit length, v behind a SiLU, g = -a softplus(x + b) with a in [1, 16] and
    softplus(b) in [0.001, 0.1] by heads, beta a sigmoid: what the projections of such a
    layer give (heads that forget within a few tokens and heads that hardly do)."""
    silu = torch.nn.functional.silu
    q, k = (_unit(silu(_randn(g, *lead, Hk, DH))).to(dt) for _ in range(2))
    v = silu(_randn(g, *lead, Hv, DH)).to(dt)
    a = 1 + 15 * torch.rand(Hv, generator=g, device="cuda")
    sp = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(Hv, generator=g, device="cuda"))
    gate = -a * torch.nn.functional.softplus(_randn(g, *lead, Hv) + torch.log(torch.expm1(sp)))
    return q, k, v, gate, torch.sigmoid(_randn(g, *lead, Hv))


def _lengths(case, seed):
    """The lengths of the packed sequences: at least 1 each, the first of them 1, T in all."""
    n, T = case["seqs"], case["T"]
    r = torch.rand(n, generator=torch.Generator().manual_seed(seed)) + 0.05
    lens = (r / r.sum() * (T - n)).long() + 1
    lens[0] = 1
    lens[-1] += T - int(lens.sum())
    return lens.tolist()


def prepare(case, seed):
    g, dt = torch.Generator(device="cuda").manual_seed(seed), _DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "rule":
        B, T, Hk, Hv = case["B"], case["T"], case["Hk"], case["Hv"]
        s["in"] = dict(zip(("q", "k", "v", "g", "beta"), _rule_inputs(g, (B, T), Hk, Hv, dt)))
        n = case["seqs"] or B
        if case["state"]:
            s["in"]["state"] = _randn(g, n, Hv, DH, DH) * 0.1
        s["lens"] = _lengths(case, seed) if case["seqs"] else None
        if case["seqs"]:
            s["cu"] = torch.tensor([0] + s["lens"], device="cuda").cumsum(0).to(torch.int32)
        if case["train"]:
            for t in s["in"].values():
                t.requires_grad_(True)
            s["do"] = _randn(g, B, T, Hv, DH).to(dt)
            s["ds"] = _randn(g, n, Hv, DH, DH) * 0.1 if case["state"] else None
    elif case["op"] == "step":
        N, pool = case["N"], case["pool"]
        s["in"] = dict(zip(("q", "k", "v", "g", "beta"), _rule_inputs(g, (N,), case["Hk"], case["Hv"], dt)))
        s["pool"] = _randn(g, pool, case["Hv"], DH, DH) * 0.1
        at = torch.randperm(pool, generator=g, device="cuda")[:N].to(torch.int32)
        if N >= 8:
            at[5::8] = -1                       # padding of the batch
        s["at"] = at
    else:
        rows, D = case["rows"], case["D"]
        s["x"] = _randn(g, rows, D).to(dt)
        s["res"] = (_randn(g, rows, D) * 2).to(dt) if case["residual"] else None
        s["w"] = (1 + 0.1 * _randn(g, D)).to(dt)
        if case["op"] == "norm":
            for t in (s["x"], s["res"], s["w"]):
                if t is not None:
                    t.requires_grad_(True)
            s["dy"] = _randn(g, rows, D).to(dt)
            s["dh"] = _randn(g, rows, D).to(dt) if case["residual"] else None
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _pad_index(lens):
    """Rows of the packed tokens laid out as [sequences, longest], and which of them are real."""
    n, most = len(lens), max(lens)
    lens_t = torch.tensor(lens, device="cuda")
    at = torch.arange(most, device="cuda")[None]
    real = at < lens_t[:, None]
    rows = (lens_t.cumsum(0) - lens_t)[:, None] + at
    return torch.where(real, rows, 0), real


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular a [..., n, n], n a power of two: the
    inverses of the diagonal blocks, joined two by two."""
    n = a.shape[-1]
    inv, b = torch.ones_like(a[..., :1]).unsqueeze(-1), 1        # [..., blocks, b, b]
    while b < n:
        low = torch.stack([a[..., i + b:i + 2 * b, i:i + b] for i in range(0, n, 2 * b)], -3)
        x, y = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        top = torch.cat([x, torch.zeros_like(x)], -1)
        inv, b = torch.cat([top, torch.cat([-(y @ (low @ x)), y], -1)], -2), 2 * b
    return inv.squeeze(-3)


def _plain_chunks(q, k, v, g, beta, state, scale):
    """The rule over [B, H, T, .] in fp32, 64 tokens at a time: all that does not depend
    on the state at once, then the states one chunk after the other (one product each),
    then the outputs at once.  Sums of g in 64 bits."""
    B, H, T, _ = q.shape
    C = 64
    pad = -T % C
    n = (T + pad) // C
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, pad)).view(B, H, n, C, DH) for t in (q, k, v))
    g, beta = (torch.nn.functional.pad(t, (0, pad)).view(B, H, n, C) for t in (g, beta))
    G = g.double().cumsum(-1)
    low = torch.ones(C, C, dtype=torch.bool, device=q.device).tril()
    D = torch.where(low, G[..., :, None] - G[..., None, :], -math.inf).exp().float()
    decay, rest, whole = G.exp().float(), (G[..., -1:] - G).exp().float(), G[..., -1].exp().float()
    kt = k.transpose(-1, -2)
    A = ((k @ kt) * D * beta[..., :, None]).tril(-1)
    inv = _unit_lower_inverse(A)
    w = inv @ (k * (beta * decay)[..., None])
    u = inv @ (v * beta[..., None])
    kr = (k * rest[..., None]).transpose(-1, -2)
    move = whole[..., None, None] * torch.eye(DH, device=q.device) - kr @ w
    add = kr @ u
    S = state if state is not None else torch.zeros(B, H, DH, DH, device=q.device)
    each = []
    for m, a in zip(move.unbind(2), add.unbind(2)):
        each.append(S)
        S = m @ S + a
    S0 = torch.stack(each, 2)
    u = u - w @ S0
    o = (((q * decay[..., None]) @ S0) + ((q @ kt) * D) @ u) * scale
    return o.reshape(B, H, T + pad, DH)[:, :, :T], S


def _plain_rule(t, lens, dt):
    Hv, share = t["v"].shape[2], t["v"].shape[2] // t["q"].shape[2]
    x = {n: t[n].float() for n in ("q", "k", "v", "g", "beta")}
    for n in ("q", "k"):
        x[n] = x[n].repeat_interleave(share, 2)
    if lens is not None:
        rows, real = _pad_index(lens)
        x = {n: a[0][rows] * real.view(*real.shape, *([1] * (a.dim() - 2))) for n, a in x.items()}
    o, S = _plain_chunks(*(x[n].transpose(1, 2) for n in ("q", "k", "v", "g", "beta")), t.get("state"), DH ** -0.5)
    o = o.transpose(1, 2)
    if lens is not None:
        o = o[real][None]                       # the packed order again
    return o.to(dt), S


def _plain_step(t, pool, at, dt):
    share = t["v"].shape[1] // t["q"].shape[1]
    q, k = (t[n].float().repeat_interleave(share, 1) for n in ("q", "k"))
    real = (at >= 0) & (at < pool.shape[0])
    rows = torch.where(real, at, 0).long()
    S = pool[rows] * t["g"].exp()[..., None, None]
    u = (t["v"].float() - (S * k[..., None]).sum(-2)) * t["beta"][..., None]
    S = S + k[..., None] * u[..., None, :]
    o = (S * q[..., None]).sum(-2) * DH ** -0.5
    pool[rows[real]] = S[real]
    return (o * real[:, None, None]).to(dt)


def _plain_norm(x, res, w):
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    f = h.float()
    return f * (f.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float(), h


def run(state):
    case = state["case"]
    if case["op"] == "rule":
        t = state["in"]
        if own:
            from gsa_gdn_benchmarkstudy_amd import gated_delta_rule

            o, S = gated_delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], initial_state=t.get("state"),
                                    output_final_state=case["state"], cu_seqlens=state.get("cu"))
        else:
            o, S = _plain_rule(t, state["lens"], _DTYPES[case["dtype"]])
        out = {"o": o}
        if case["state"]:
            out["final"] = S
        if case["train"]:
            outs, grads = ([o, S], [state["do"], state["ds"]]) if case["state"] else ([o], [state["do"]])
            out |= {"d" + n: d for n, d in zip(t, torch.autograd.grad(outs, list(t.values()), grads))}
        return {n: a.detach() for n, a in out.items()}
    if case["op"] == "step":
        t = state["in"]
        if own:
            from gsa_gdn_benchmarkstudy_amd import gated_delta_step

            o = gated_delta_step(t["q"], t["k"], t["v"], t["g"], t["beta"], state["pool"], state_indices=state["at"])
        else:
            o = _plain_step(t, state["pool"], state["at"], _DTYPES[case["dtype"]])
        return {"o": o, "pool": state["pool"]}
    x, res, w = state["x"], state["res"], state["w"]
    if case["op"] == "norm":
        if own:
            from gsa_gdn_benchmarkstudy_amd import add_rms_norm

            y, h = add_rms_norm(x, w, residual=res, eps=EPS)
        else:
            y, h = _plain_norm(x, res, w)
            y = y.to(x.dtype)
        if res is None:
            dx, dw = torch.autograd.grad(y, [x, w], state["dy"])
            return {"y": y.detach(), "dx": dx, "dw": dw}
        dx, dres, dw = torch.autograd.grad([y, h], [x, res, w], [state["dy"], state["dh"]])
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dres": dres, "dw": dw}
    if own:
        from gsa_gdn_benchmarkstudy_amd import add_rms_norm_fp8

        y, scale, h = add_rms_norm_fp8(x, w, residual=res, eps=EPS)
    else:
        y, h = _plain_norm(x, res, w)
        scale = y.abs().amax(-1) / 448
        scale = torch.where(scale == 0, 1.0, scale)
        y = (y / scale[:, None]).to(torch.float8_e4m3fn)
    return {"y": y, "scale": scale, "h": h}


def work(case):
    size = {"bf16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "rule":
        n, Hk, Hv = case["B"] * case["T"], case["Hk"], case["Hv"]
        states = (case["seqs"] or case["B"]) * Hv * DH * DH * 4 * 2 if case["state"] else 0
        ends = n * (2 * Hk + 2 * Hv) * DH * size + n * Hv * 8 + states           # q, k, v, o; g, beta; the states
        flops = 6 * DH * DH * n * Hv
        if case["train"]:
            ends += n * (2 * Hk + 2 * Hv) * DH * size + n * Hv * 8 + states      # dq, dk, dv, do; dg, dbeta; the states'
            flops += 14 * DH * DH * n * Hv
        return {"bytes": ends, "flops": flops}
    if case["op"] == "step":
        real = case["N"] - (len(range(5, case["N"], 8)) if case["N"] >= 8 else 0)
        per = case["Hv"] * DH * DH
        io = case["N"] * ((2 * case["Hk"] + 2 * case["Hv"]) * DH * size + case["Hv"] * 8)
        return {"bytes": 2 * 4 * real * per + io, "flops": 6 * real * per}
    n, D, r = case["rows"] * case["D"], case["D"], case["residual"]
    if case["op"] == "norm":                     # forward x (res), y (h); backward dy (dh), dx (dres)
        return {"bytes": n * size * (8 if r else 4) + 2 * D * size, "flops": 12 * n}
    return {"bytes": n * (size * (3 if r else 1) + (1 if r else 1 + size)) + case["rows"] * 4 + D * size, "flops": 6 * n}


# ---------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_rule(x, S, do, dS, scale):
    """One batch of equally long sequences, token by token: x of q, k, v [n, T, H, 128], g,
    beta [n, T, H], S [n, H, 128, 128], all in 64 bits; with do (and dS) the gradients too."""
    T = x["q"].shape[1]
    a = x["g"].exp()
    states, out, us = [], [], []
    for t in range(T):
        k, b = x["k"][:, t], x["beta"][:, t, :, None]
        if do is not None:
            states.append(S)
        P = S * a[:, t, :, None, None]
        u = b * (x["v"][:, t] - torch.einsum("nhkv,nhk->nhv", P, k))
        S = P + k[..., None] * u[..., None, :]
        out.append(scale * torch.einsum("nhkv,nhk->nhv", S, x["q"][:, t]))
        us.append(u)
    o, final = torch.stack(out, 1), S
    if do is None:
        return o, final, None
    d = {n: torch.zeros_like(v) for n, v in x.items()}
    for t in reversed(range(T)):
        q, k, v, b = x["q"][:, t], x["k"][:, t], x["v"][:, t], x["beta"][:, t, :, None]
        P, u = states[t] * a[:, t, :, None, None], us[t]
        S = P + k[..., None] * u[..., None, :]
        d["q"][:, t] = scale * torch.einsum("nhkv,nhv->nhk", S, do[:, t])
        dS = dS + scale * q[..., None] * do[:, t, :, None, :]
        du = torch.einsum("nhkv,nhk->nhv", dS, k)
        d["k"][:, t] = torch.einsum("nhkv,nhv->nhk", dS, u) - torch.einsum("nhkv,nhv->nhk", P, b * du)
        d["v"][:, t] = b * du
        d["beta"][:, t] = (du * (v - torch.einsum("nhkv,nhk->nhv", P, k))).sum(-1)
        dP = dS - k[..., None] * (b * du)[..., None, :]
        d["g"][:, t] = (dP * P).sum((-1, -2))
        dS = dP * a[:, t, :, None, None]
        states[t] = None
    return o, final, d | {"state": dS}


def _exact_case_rule(s, case):
    share, Hk = case["Hv"] // case["Hk"], case["Hk"]
    x = {n: s["in"][n].detach().double() for n in ("q", "k", "v", "g", "beta")}
    for n in ("q", "k"):
        x[n] = x[n].repeat_interleave(share, 2)
    init = s["in"]["state"].detach().double() if case["state"] else None
    lens = s["lens"] or [case["T"]] * case["B"]
    # sequences padded behind their ends with tokens that change nothing (k, v, beta, g of 0)
    n, most, b0 = len(lens), max(lens), 0
    where = []
    for i, L in enumerate(lens):
        where.append((0, b0, L) if s["lens"] else (i, 0, L))
        b0 += L if s["lens"] else 0

    def padded(t):
        r = torch.zeros(n, most, *t.shape[2:], dtype=torch.float64, device="cuda")
        for i, (b, at, L) in enumerate(where):
            r[i, :L] = t[b, at:at + L]
        return r

    def packed(t):
        if not s["lens"]:
            return t
        return torch.cat([t[i, :L] for i, (_, _, L) in enumerate(where)])[None]

    x = {name: padded(t) for name, t in x.items()}
    do = padded(s["do"].double()) if case["train"] else None
    zero = torch.zeros(n, case["Hv"], DH, DH, dtype=torch.float64, device="cuda")
    parts = []
    step = max(1, 64 * 4096 // (most * case["Hv"])) if case["train"] else n     # the states of all tokens at once: 34 GB at most
    for i in range(0, n, step):
        sl = slice(i, i + step)
        dS = (s["ds"].double() if case["state"] else zero)[sl] if case["train"] else None
        parts.append(_exact_rule({a: t[sl] for a, t in x.items()}, (init if init is not None else zero)[sl],
                                 do[sl] if do is not None else None, dS, DH ** -0.5))
    out = {"o": packed(torch.cat([p[0] for p in parts]))}
    if case["state"]:
        out["final"] = torch.cat([p[1] for p in parts])
    if case["train"]:
        d = {a: torch.cat([p[2][a] for p in parts]) for a in parts[0][2]}
        for a in ("q", "k"):
            d[a] = d[a].unflatten(2, (Hk, share)).sum(3)
        out |= {"d" + a: packed(d[a]) for a in ("q", "k", "v", "g", "beta")}
        if case["state"]:
            out["dstate"] = d["state"]
    return out


def exact(case, seed):
    if case["op"] == "rule" and case["T"] * (4 if case["train"] else 1) > 32000:
        return None                              # a loop over tokens of more than 20 s
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rule":
            return _exact_case_rule(s, case)
        if case["op"] == "step":
            share = case["Hv"] // case["Hk"]
            x = {n: t.double() for n, t in s["in"].items()}
            q, k = (x[n].repeat_interleave(share, 1) for n in ("q", "k"))
            pool, o = s["pool"].double(), torch.zeros_like(x["v"])
            for i, at in enumerate(s["at"].tolist()):
                if at < 0:
                    continue
                P = pool[at] * x["g"][i].exp()[:, None, None]
                u = x["beta"][i][:, None] * (x["v"][i] - (P.transpose(-1, -2) @ k[i][..., None]).squeeze(-1))
                pool[at] = P + k[i][..., None] * u[:, None]
                o[i] = DH ** -0.5 * (pool[at].transpose(-1, -2) @ q[i][..., None]).squeeze(-1)
            return {"o": o, "pool": pool}
        x, w = s["x"].double(), s["w"].double()
        h = x if s["res"] is None else (x + s["res"].double()).to(s["x"].dtype).double()   # the stream as it is kept
        r = (h.square().mean(-1, keepdim=True) + EPS) ** -0.5
        y = h * r * w
        if case["op"] == "norm8":
            return {"y": None, "scale": y.abs().amax(-1) / 448, "h": h}
        dy = s["dy"].double()
        dn = dy * w
        dx = r * (dn - h * r * (dn * h * r).mean(-1, keepdim=True))
        if s["res"] is None:
            return {"y": y, "dx": dx, "dw": (dy * h * r).sum(0)}
        dx = dx + s["dh"].double()
        return {"y": y, "h": h, "dx": dx, "dres": dx, "dw": (dy * h * r).sum(0)}
