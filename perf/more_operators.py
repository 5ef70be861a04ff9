"""Linear attention with a decay for each head, attention in a sliding window, and the single-token
steps of both, as cases that can be timed and checked.

A case is one call of a public entry point: ``linear_attention`` or ``window_attention``
(forward, or forward and backward), ``linear_attention_step`` or ``window_attention_step``.
Where ``own`` is false the same operators are computed in plain torch.  Heads are the
framework's (d = 128), 16 of them unless a case says otherwise; sequence lengths are those of
the benchmark's configs and of the harness's sweep, and ragged ones between them.
"""

import math

import torch

own = False

DH = 128
SCALE = DH ** -0.5
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _linear(name, dtype, B, T, Hk, Hv, train=False, seqs=0, state=False):
    """B sequences of T tokens, or (seqs > 0, B = 1) T tokens packed from that many
    sequences; Hk heads of q and k serve Hv heads of v; state: an initial state is given
    and the final one wanted."""
    return {"name": name, "op": "linear", "dtype": dtype, "B": B, "T": T, "Hk": Hk, "Hv": Hv, "train": train, "seqs": seqs,
            "state": state}


def _window(name, dtype, B, T, H, Hkv, W, S, train=False, seqs=0):
    """The same of H query heads on Hkv heads of keys: a window of W tokens and the first S."""
    return {"name": name, "op": "window", "dtype": dtype, "B": B, "T": T, "H": H, "Hkv": Hkv, "W": W, "S": S, "train": train,
            "seqs": seqs}


def listed():
    return [
        # prefill at the benchmark's headline length: few heads, a long axis, state kept for decoding
        _linear("linear_bf16_T16384", "bf16", 1, 16384, 16, 16, state=True),
        # a packed batch of ragged prompts (one of a single token among them), each q/k head shared by two v heads
        _linear("linear_bf16_packed_T12289", "bf16", 1, 12289, 8, 16, seqs=23, state=True),
        # a training step over a batch, forward and backward, the decays learned
        _linear("linear_train_bf16_B4_T4096", "bf16", 4, 4096, 16, 16, train=True),
        # full precision, ragged, forward and backward with carried states (gradient checks, small models)
        _linear("linear_train_f32_B2_T1537", "f32", 2, 1537, 4, 4, train=True, state=True),
        # decoding one sequence: the smallest call
        {"name": "linear_step_bf16_N1", "op": "linear_step", "dtype": "bf16", "N": 1, "pool": 4, "Hk": 16, "Hv": 16},
        # decoding a serving batch out of a larger pool of states, some rows padding, shared heads
        {"name": "linear_step_bf16_N203", "op": "linear_step", "dtype": "bf16", "N": 203, "pool": 256, "Hk": 8, "Hv": 16},
        # prefill at the headline length with a long window, four query heads to a key head: the largest
        _window("window_bf16_T16384_W4096", "bf16", 1, 16384, 16, 4, 4096, 4),
        # a packed batch of ragged prompts with a short window
        _window("window_bf16_packed_T12289_W512", "bf16", 1, 12289, 16, 16, 512, 4, seqs=23),
        # a training step over a batch, forward and backward
        _window("window_train_bf16_B4_T4096_W1024", "bf16", 4, 4096, 16, 4, 1024, 4, train=True),
        # full precision, ragged, forward and backward, more first tokens than a tile
        _window("window_train_f32_B2_T1537_W256", "f32", 2, 1537, 4, 2, 256, 70, train=True),
        # decoding one sequence: latency counts
        {"name": "window_step_bf16_N1_W1024", "op": "window_step", "dtype": "bf16", "N": 1, "pool": 4, "H": 16, "Hkv": 4, "W": 1024, "S": 4,
         "more": 0},
        # decoding a serving batch out of a larger pool of caches, short sequences and rows of padding among it
        {"name": "window_step_bf16_N61_W2048", "op": "window_step", "dtype": "bf16", "N": 61, "pool": 64, "H": 16, "Hkv": 4, "W": 2048, "S": 4,
         "more": 60},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_step", "window", "window", "window_step"])
    f32 = rng.random() < 0.3
    dtype = "f32" if f32 else "bf16"
    if op in ("linear", "window"):
        train = rng.random() < 0.5
        B = rng.choice([1, 1, 2, 3, 5])
        top = (3074 if f32 else 16384) if train else (6001 if f32 else 16384)
        T = _log_int(rng, 1, top // B)
        seqs = min(rng.choice([0, 0, 0, 2, 9, 31]), T) if B == 1 and T > 1 else 0
        few = rng.choice([1, 2, 4, 8, 16])
        many = few * rng.choice([1, 1, 2, 3, 4]) if few < 8 else 16
        if op == "linear":
            c = _linear("", dtype, B, T, few, many, train, seqs, rng.random() < 0.5)
        else:
            W = min(_log_int(rng, 1, 4096), 16384 * 1024 // (B * T) if train or f32 else 4096)
            c = _window("", dtype, B, T, many, few, W, rng.choice([0, 0, 1, 4, 4, 33, 130]), train, seqs)
    elif op == "linear_step":
        N, Hk = _log_int(rng, 1, 256), rng.choice([1, 4, 8, 16])
        c = {"op": op, "dtype": dtype, "N": N, "pool": N + rng.randrange(1, 33), "Hk": Hk, "Hv": Hk * rng.choice([1, 2]) if Hk < 16 else 16}
    else:
        N, Hkv, W = _log_int(rng, 1, 96), rng.choice([1, 2, 4, 8]), _log_int(rng, 16, 4096)
        N = max(1, min(N, 64 * 2048 * 4 // (W * Hkv) // (2 if f32 else 1)))
        c = {"op": op, "dtype": dtype, "N": N, "pool": N + rng.randrange(1, 5), "H": Hkv * rng.choice([1, 2, 4, 8]), "Hkv": Hkv, "W": W,
             "S": rng.choice([0, 1, 4, 33]), "more": rng.choice([0, 7, 60])}
    c.pop("name", None)
    return c


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _decays(g, H):
    """Log decays from -0.7 to -0.004 by heads (half a token to 256 tokens of memory), none alike."""
    at = (torch.arange(H, device="cuda") + torch.rand(H, generator=g, device="cuda")) / H
    return -torch.exp2(-8 * at)


def _linear_inputs(g, lead, Hk, Hv, dt):
    """q and k behind a SiLU, as such layers take them."""
    q, k = (torch.nn.functional.silu(_randn(g, *lead, Hk, DH)).to(dt) for _ in range(2))
    return {"q": q, "k": k, "v": _randn(g, *lead, Hv, DH).to(dt), "g": _decays(g, Hv)}


def _lengths(case, seed):
    """The lengths of the packed sequences: at least 1 each, the first of them 1, T in all."""
    n, T = case["seqs"], case["T"]
    r = torch.rand(n, generator=torch.Generator().manual_seed(seed)) + 0.05
    lens = (r / r.sum() * (T - n)).long() + 1
    lens[0] = 1
    lens[-1] += T - int(lens.sum())
    return lens.tolist()


def _rows_of_pool(g, N, pool):
    at = torch.randperm(pool, generator=g, device="cuda")[:N].to(torch.int32)
    if N >= 8:
        at[5::8] = -1                            # padding of the batch
    return at


def prepare(case, seed):
    g, dt = torch.Generator(device="cuda").manual_seed(seed), _DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("linear", "window"):
        B, T = case["B"], case["T"]
        if case["op"] == "linear":
            s["in"] = _linear_inputs(g, (B, T), case["Hk"], case["Hv"], dt)
            n = case["seqs"] or B
            if case["state"]:
                s["in"]["state"] = _randn(g, n, case["Hv"], DH, DH)
            s["ds"] = _randn(g, n, case["Hv"], DH, DH) if case["train"] and case["state"] else None
        else:
            s["in"] = {n: _randn(g, B, T, case[h], DH).to(dt) for n, h in (("q", "H"), ("k", "Hkv"), ("v", "Hkv"))}
        s["lens"] = _lengths(case, seed) if case["seqs"] else None
        s["cu"] = torch.tensor([0] + s["lens"], device="cuda").cumsum(0).to(torch.int32) if case["seqs"] else None
        if case["train"]:
            for t in s["in"].values():
                t.requires_grad_(True)
            s["do"] = _randn(g, B, T, case.get("Hv") or case["H"], DH).to(dt)
        return s
    N, pool = case["N"], case["pool"]
    s["at"] = _rows_of_pool(g, N, pool)
    if case["op"] == "linear_step":
        s["in"] = _linear_inputs(g, (N,), case["Hk"], case["Hv"], dt)
        s["pool"] = _randn(g, pool, case["Hv"], DH, DH)
        return s
    s["in"] = {n: _randn(g, N, case[h], DH).to(dt) for n, h in (("q", "H"), ("k", "Hkv"), ("v", "Hkv"))}
    rows = case["S"] + case["W"] + case["more"]
    s["caches"] = [_randn(g, pool, rows, case["Hkv"], DH).to(dt) for _ in range(2)]
    # most sequences are longer than the window, a quarter are not; lengths have no common step
    far = torch.rand(N, generator=g, device="cuda") < 0.75
    at = torch.rand(N, generator=g, device="cuda")
    s["pos"] = torch.where(far, case["W"] + at * 8 * case["W"], at * (case["W"] + case["S"])).to(torch.int64)
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


def _unpacked(x, lens):
    """Packed rows [1, T, ...] as [sequences, longest, ...] with zeros behind each sequence."""
    rows, real = _pad_index(lens)
    return [a[0][rows] * real.view(*real.shape, 1, 1) for a in x], real


def _plain_linear(t, lens, dt):
    """Chunks of 64 tokens: what each adds to the state at once, the states before all chunks as one
    product with the decays between chunks, then the outputs at once.  Decays in 64 bits."""
    share, Hv = t["v"].shape[2] // t["q"].shape[2], t["v"].shape[2]
    q, k, v = t["q"].float().repeat_interleave(share, 2), t["k"].float().repeat_interleave(share, 2), t["v"].float()
    real = None
    if lens is not None:
        (q, k, v), real = _unpacked((q, k, v), lens)
    B, T = v.shape[:2]
    C, g = 64, t["g"].double()
    n = (T + C - 1) // C
    q, k, v = (torch.nn.functional.pad(a, (0, 0, 0, 0, 0, n * C - T)).view(B, n, C, Hv, DH).permute(0, 3, 1, 2, 4) for a in (q, k, v))
    i = torch.arange(C, device=v.device, dtype=torch.float64)
    gap = i[:, None] - i
    D = torch.where(gap >= 0, (g[:, None, None] * gap.clamp_min(0)).exp(), 0.0).float()            # [Hv, C, C]
    c = torch.arange(n + 1, device=v.device, dtype=torch.float64)
    gap = c[:, None] - c
    # the state before chunk c: the initial one and what chunks 0 .. c - 1 add, each decayed by the chunks between
    between = torch.where(gap >= 0, (g[:, None, None] * C * gap.clamp_min(0)).exp(), 0.0).float()   # [Hv, n + 1, n + 1]
    rest = (g[:, None] * (C - 1 - i)).exp().float()[:, None, :, None]
    add = (k * rest).transpose(-1, -2) @ v                                                         # [B, Hv, n, d, d]
    first = t["state"] if "state" in t else torch.zeros(B, Hv, DH, DH, device=v.device)
    add = torch.cat([first.unsqueeze(2), add], 2).flatten(-2)
    S0 = (between @ add).unflatten(-1, (DH, DH))[:, :, :n]
    o = (q * (g[:, None] * (i + 1)).exp().float()[:, None, :, None]) @ S0 + ((q @ k.transpose(-1, -2)) * D[:, None]) @ v
    o = (o * SCALE).permute(0, 2, 3, 1, 4).reshape(B, n * C, Hv, DH)[:, :T]
    # the final state: every token and the initial state, decayed to the sequence's own end
    end = torch.full((B,), T, device=v.device) if lens is None else torch.tensor(lens, device=v.device)
    last = (end - 1) // C                                                                          # the chunk with the last token
    left = (end - 1 - last * C).double()                                                           # its index there
    pick = last.view(B, 1, 1, 1, 1)
    kl, vl = (torch.take_along_dim(a, pick, 2).squeeze(2) for a in (k, v))
    w = torch.where(i <= left[:, None, None], (g[:, None] * (left[:, None, None] - i).clamp_min(0)).exp(), 0.0).float()
    Sl = torch.take_along_dim(S0, pick, 2).squeeze(2)
    final = Sl * (g * (left[:, None] + 1)).exp().float()[..., None, None] + (kl * w[..., None]).transpose(-1, -2) @ vl
    return (o if real is None else o[real][None]).to(dt), final


def _plain_window(t, lens, W, S, dt):
    """Blocks of queries against their own block of keys, the one before and the first S tokens."""
    q, k, v = (t[n].float() for n in ("q", "k", "v"))
    real = None
    if lens is not None:
        (q, k, v), real = _unpacked((q, k, v), lens)
    B, T, H, _ = q.shape
    Hkv = k.shape[2]
    C = min(T, max(W, 64))
    n = (T + C - 1) // C
    q, k, v = (torch.nn.functional.pad(a, (0, 0, 0, 0, 0, n * C - T)).view(B, n, C, Hkv, -1, DH).permute(0, 3, 1, 4, 2, 5) for a in (q, k, v))
    q = q.flatten(3, 4)                                                                            # [B, Hkv, n, share * C, d]
    S = min(S, T)

    def keys(a):
        a = a.squeeze(3)
        before = torch.nn.functional.pad(a, (0, 0, 0, 0, 1, 0))[:, :, :n]
        first = a.flatten(2, 3)[:, :, None, :S].expand(-1, -1, n, -1, -1)
        return torch.cat([first, before, a], 3) if n > 1 else a

    k, v = keys(k), keys(v)
    at = torch.arange(n * C, device=q.device).view(n, C, 1)
    block = at[:, :1] - C + torch.arange(2 * C, device=q.device)                                   # [n, 1, 2 C]
    if n > 1:
        first = torch.arange(S, device=q.device).expand(n, 1, S)
        seen = torch.cat([first <= at, (block <= at) & (block > at - W) & (block >= S)], -1)       # a first token counts once
    else:
        pos = torch.arange(C, device=q.device)
        seen = (pos <= at) & ((pos > at - W) | (pos < S))
    seen = seen.repeat(1, H // Hkv, 1)
    s = (q @ k.transpose(-1, -2) * SCALE).masked_fill(~seen, -math.inf)
    p = (s - s.amax(-1, keepdim=True).detach()).exp()
    o = (p @ v) / p.sum(-1, keepdim=True)
    o = o.unflatten(3, (-1, C)).permute(0, 2, 4, 1, 3, 5).reshape(B, n * C, H, DH)[:, :T]
    return (o if real is None else o[real][None]).to(dt)


def _plain_linear_step(t, pool, at, dt):
    share = t["v"].shape[1] // t["q"].shape[1]
    q, k = (t[n].float().repeat_interleave(share, 1) for n in ("q", "k"))
    real = (at >= 0) & (at < pool.shape[0])
    rows = torch.where(real, at, 0).long()
    S = pool[rows] * t["g"].exp()[None, :, None, None] + k[..., None] * t["v"].float()[..., None, :]
    o = (S * q[..., None]).sum(-2) * SCALE
    pool[rows[real]] = S[real]
    return (o * real[:, None, None]).to(dt)


def _plain_window_step(t, caches, pos, at, W, S, dt):
    real = (at >= 0) & (at < caches[0].shape[0])
    slot = torch.where(real, at, 0).long()
    ring = caches[0].shape[1] - S
    row = torch.where(pos < S, pos, S + (pos - S).clamp_min(0) % ring)
    for c, n in zip(caches, ("k", "v")):
        c[slot[real], row[real]] = t[n][real]
    near = pos[:, None] - torch.arange(W, device=pos.device)                                       # the window, newest first
    rows = torch.cat([torch.arange(S, device=pos.device).expand(len(pos), S), S + (near - S) % ring], 1)
    seen = torch.cat([torch.arange(S, device=pos.device) <= pos[:, None], near >= S], 1)
    k, v = (c[slot[:, None], rows].float().transpose(1, 2) for c in caches)                        # [N, Hkv, S + W, d]
    N, H, _ = t["q"].shape
    q = t["q"].float().view(N, k.shape[1], -1, DH)
    s = (q @ k.transpose(-1, -2) * SCALE).masked_fill(~seen[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    o = (p @ v) / p.sum(-1, keepdim=True)
    return torch.where(real[:, None, None], o.view(N, H, DH), 0.0).to(dt)


def run(state):
    case, dt = state["case"], _DTYPES[state["case"]["dtype"]]
    t = state["in"]
    if case["op"] == "linear":
        if own:
            from gsa_gdn_benchmarkstudy_amd import linear_attention

            o, S = linear_attention(t["q"], t["k"], t["v"], t["g"], initial_state=t.get("state"), output_final_state=case["state"],
                                    cu_seqlens=state["cu"])
        else:
            o, S = _plain_linear(t, state["lens"], dt)
        out = {"o": o}
        if case["state"]:
            out["final"] = S
        if case["train"]:
            outs, grads = ([o, S], [state["do"], state["ds"]]) if case["state"] else ([o], [state["do"]])
            out |= {"d" + n: d for n, d in zip(t, torch.autograd.grad(outs, list(t.values()), grads))}
        return {n: a.detach() for n, a in out.items()}
    if case["op"] == "window":
        if own:
            from gsa_gdn_benchmarkstudy_amd import window_attention

            o = window_attention(t["q"], t["k"], t["v"], case["W"], sinks=case["S"], cu_seqlens=state["cu"])
        else:
            o = _plain_window(t, state["lens"], case["W"], case["S"], dt)
        out = {"o": o.detach()}
        if case["train"]:
            out |= {"d" + n: d for n, d in zip(t, torch.autograd.grad(o, list(t.values()), state["do"]))}
        return out
    if case["op"] == "linear_step":
        if own:
            from gsa_gdn_benchmarkstudy_amd import linear_attention_step

            o = linear_attention_step(t["q"], t["k"], t["v"], t["g"], state["pool"], state_indices=state["at"])
        else:
            o = _plain_linear_step(t, state["pool"], state["at"], dt)
        return {"o": o, "pool": state["pool"]}
    kc, vc = state["caches"]
    if own:
        from gsa_gdn_benchmarkstudy_amd import window_attention_step

        o = window_attention_step(t["q"], t["k"], t["v"], kc, vc, state["pos"], case["W"], sinks=case["S"], cache_indices=state["at"])
    else:
        o = _plain_window_step(t, state["caches"], state["pos"], state["at"], case["W"], case["S"], dt)
    return {"o": o, "k_cache": kc, "v_cache": vc}


# ---------------------------------------------------------------------------
# The work of a case
# ---------------------------------------------------------------------------

def _pairs(lens, W, S):
    """Visible pairs of a query and a key, over sequences of these lengths."""
    total = 0
    for T in lens:
        w = min(W, T)
        total += w * (w + 1) // 2 + (T - w) * w
        s = min(S, T - w)                        # first tokens: token j is out of the window from query j + W on
        total += s * (T - w) - s * (s - 1) // 2 if s > 0 else 0
    return total


def work(case):
    size = {"bf16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "linear":
        n, Hk, Hv = case["B"] * case["T"], case["Hk"], case["Hv"]
        states = (case["seqs"] or case["B"]) * Hv * DH * DH * 4 * 2 if case["state"] else 0
        ends = n * (2 * Hk + 2 * Hv) * DH * size + 4 * Hv + states                # q, k, v, o; g; the states
        flops = 4 * DH * DH * n * Hv
        if case["train"]:
            ends += n * (2 * Hk + 2 * Hv) * DH * size + 4 * Hv + states           # dq, dk, dv, do; dg; the states'
            flops += 10 * DH * DH * n * Hv
        return {"bytes": ends, "flops": flops}
    if case["op"] == "window":
        n, H, Hkv = case["B"] * case["T"], case["H"], case["Hkv"]
        # a packed batch's lengths are the seed's: as if they were equal
        lens = [case["T"]] * case["B"] if not case["seqs"] else [case["T"] // case["seqs"]] * case["seqs"]
        flops = 4 * DH * H * _pairs(lens, case["W"], case["S"])
        ends = n * (2 * H + 2 * Hkv) * DH * size
        return {"bytes": 2 * ends if case["train"] else ends, "flops": flops * 7 // 2 if case["train"] else flops}
    real = case["N"] - (len(range(5, case["N"], 8)) if case["N"] >= 8 else 0)
    if case["op"] == "linear_step":
        per = case["Hv"] * DH * DH
        return {"bytes": 2 * 4 * real * per + case["N"] * (2 * case["Hk"] + 2 * case["Hv"]) * DH * size + 4 * case["Hv"],
                "flops": 4 * real * per}
    # a quarter of the sequences is shorter than the window, by half in the mean
    keys = real * (0.75 * (case["S"] + case["W"]) + 0.25 * 0.5 * (case["S"] + case["W"])) if case["N"] > 1 else case["S"] + case["W"]
    return {"bytes": int(2 * keys * case["Hkv"] * DH * size + case["N"] * (2 * case["H"] + 4 * case["Hkv"]) * DH * size),
            "flops": int(4 * DH * case["H"] * keys)}


# ---------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_linear(x, S0, do, dS):
    """One sequence: q, k, v [T, H, 128], g [H], S0 [H, 128, 128] in 64 bits.  The recurrence written
    out: o_i = scale sum_j e^(g (i - j)) (q_i . k_j) v_j + scale e^(g (i + 1)) S0^T q_i, rows of queries at a time."""
    q, k, v = (x[n].transpose(0, 1) for n in ("q", "k", "v"))           # [H, T, d]
    g, T = x["g"], q.shape[1]
    at = torch.arange(T, device=q.device, dtype=torch.float64)
    up = (g[:, None] * (at + 1)).exp()[..., None]                       # what is left of S0 at each token
    down = (g[:, None] * (T - 1 - at)).exp()[..., None]                 # what is left of each token in the end
    o = SCALE * up * (q @ S0)
    final = (g * T).exp()[:, None, None] * S0 + (k * down).transpose(1, 2) @ v
    d = None
    if do is not None:
        do = do.transpose(0, 1)
        d = {"q": SCALE * up * (do @ S0.transpose(1, 2)), "k": down * (v @ dS.transpose(1, 2)), "v": down * (k @ dS),
             "state": (g * T).exp()[:, None, None] * dS + SCALE * (q * up).transpose(1, 2) @ do}
        d["g"] = T * (g * T).exp() * (S0 * dS).sum((1, 2)) + ((at * 0 + T - 1 - at)[:, None] * k * d["k"]).sum((1, 2)) \
            + ((at + 1)[:, None] * q * d["q"]).sum((1, 2))
    step = max(64, 2 ** 26 // (T * q.shape[0]))
    for i in range(0, T, step):
        sl = slice(i, min(i + step, T))
        gap = at[sl, None] - at[:sl.stop]
        D = torch.where(gap >= 0, (g[:, None, None] * gap.clamp_min(0)).exp(), 0.0) * SCALE
        qk = q[:, sl] @ k[:, :sl.stop].transpose(1, 2)
        o[:, sl] += (qk * D) @ v[:, :sl.stop]
        if do is not None:
            dv = do[:, sl] @ v[:, :sl.stop].transpose(1, 2)
            d["q"][:, sl] += (dv * D) @ k[:, :sl.stop]
            d["k"][:, :sl.stop] += (dv * D).transpose(1, 2) @ q[:, sl]
            d["v"][:, :sl.stop] += (qk * D).transpose(1, 2) @ do[:, sl]
            d["g"] += (qk * dv * D * gap).sum((1, 2))
    if d is not None:
        d = {n: a.transpose(0, 1) if n in "qkv" else a for n, a in d.items()}
    return o.transpose(0, 1), final, d


def _exact_window(x, W, S, do):
    """One sequence: q [T, H, 128], k, v [T, Hkv, 128] in 64 bits, rows of queries at a time against all keys."""
    q, k, v = (x[n].transpose(0, 1) for n in ("q", "k", "v"))
    Hkv, T = k.shape[:2]
    share = q.shape[0] // Hkv
    at = torch.arange(T, device=q.device)
    o = torch.empty_like(q)
    d = {n: torch.zeros_like(t) for n, t in zip("qkv", (q, k, v))} if do is not None else None
    do = do.transpose(0, 1) if do is not None else None
    step = max(64, 2 ** 28 // (T * q.shape[0]))
    for i in range(0, T, step):
        sl = slice(i, min(i + step, T))
        gap = at[sl, None] - at
        seen = (gap >= 0) & ((gap < W) | (at < S))
        qs = q[:, sl].unflatten(0, (Hkv, share))
        p = torch.softmax((qs @ k[:, None].transpose(2, 3) * SCALE).masked_fill(~seen, -math.inf), -1)
        o[:, sl] = (p @ v[:, None]).flatten(0, 1)
        if do is not None:
            dos = do[:, sl].unflatten(0, (Hkv, share))
            dp = dos @ v[:, None].transpose(2, 3)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * SCALE
            d["q"][:, sl] = (ds @ k[:, None]).flatten(0, 1)
            d["k"] += (ds.transpose(2, 3) @ qs).sum(1)
            d["v"] += (p.transpose(2, 3) @ dos).sum(1)
    if d is not None:
        d = {n: a.transpose(0, 1) for n, a in d.items()}
    return o.transpose(0, 1), d


def _exact_sequences(s, case):
    """Each sequence by itself; its results in their places."""
    t = {n: a.detach().double() for n, a in s["in"].items()}
    ends = [0]
    for L in s["lens"] or []:
        ends.append(ends[-1] + L)
    spans = [(0, a, b) for a, b in zip(ends, ends[1:])] if s["lens"] else [(b, 0, case["T"]) for b in range(case["B"])]
    do = s["do"].double() if case["train"] else None
    linear = case["op"] == "linear"
    out = {"o": torch.zeros(*t["q"].shape[:2], (t["v"] if linear else t["q"]).shape[2], DH, dtype=torch.float64, device="cuda")}
    if case["train"]:
        out |= {"d" + n: torch.zeros_like(a) for n, a in t.items()}
    if linear and case["state"]:
        out["final"] = torch.zeros_like(t["state"])
    share = case["Hv"] // case["Hk"] if linear else 1
    zero = torch.zeros(t["v"].shape[2], DH, DH, dtype=torch.float64, device="cuda")
    for i, (b, lo, hi) in enumerate(spans):
        x = {n: t[n][b, lo:hi] for n in ("q", "k", "v")}
        g = do[b, lo:hi] if do is not None else None
        if not linear:
            out["o"][b, lo:hi], d = _exact_window(x, case["W"], case["S"], g)
            for n in "qkv" if d else "":
                out["d" + n][b, lo:hi] = d[n]
            continue
        x = {"q": x["q"].repeat_interleave(share, 1), "k": x["k"].repeat_interleave(share, 1), "v": x["v"], "g": t["g"]}
        S0 = t["state"][i] if case["state"] else zero
        dS = s["ds"][i].double() if case["state"] and case["train"] else zero
        out["o"][b, lo:hi], final, d = _exact_linear(x, S0, g, dS)
        if case["state"]:
            out["final"][i] = final
        if d:
            for n in "qk":
                out["d" + n][b, lo:hi] = d[n].unflatten(1, (case["Hk"], share)).sum(2)
            out["dv"][b, lo:hi] = d["v"]
            out["dg"] += d["g"]
            if case["state"]:
                out["dstate"][i] = d["state"]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("linear", "window"):
            return _exact_sequences(s, case)
        x = {n: a.double() for n, a in s["in"].items()}
        if case["op"] == "linear_step":
            share = case["Hv"] // case["Hk"]
            pool, o = s["pool"].double(), torch.zeros_like(x["v"])
            for i, at in enumerate(s["at"].tolist()):
                if at < 0:
                    continue
                q, k = (x[n][i].repeat_interleave(share, 0) for n in ("q", "k"))
                pool[at] = pool[at] * x["g"].exp()[:, None, None] + k[..., None] * x["v"][i][:, None]
                o[i] = SCALE * (pool[at].transpose(-1, -2) @ q[..., None]).squeeze(-1)
            return {"o": o, "pool": pool}
        kc, vc = (c.double() for c in s["caches"])
        o, S, W = torch.zeros_like(x["q"]), case["S"], case["W"]
        ring = kc.shape[1] - S
        for i, (at, p) in enumerate(zip(s["at"].tolist(), s["pos"].tolist())):
            if at < 0:
                continue
            row = p if p < S else S + (p - S) % ring
            kc[at, row], vc[at, row] = x["k"][i], x["v"][i]
            # every position that the token sees, in order, and where the cache holds it
            seen = torch.tensor([j for j in range(p + 1) if j < S or j > p - W] if p < 2 * W + S else
                                [*range(S), *range(p - W + 1, p + 1)], device="cuda")
            rows = torch.where(seen < S, seen, S + (seen - S) % ring)
            k, v = (c[at, rows].transpose(0, 1) for c in (kc, vc))      # [Hkv, keys, d]
            q = x["q"][i].unflatten(0, (case["Hkv"], -1))
            o[i] = (torch.softmax(q @ k.transpose(1, 2) * SCALE, -1) @ v).flatten(0, 1)
        return {"o": o, "k_cache": kc, "v_cache": vc}
