"""Measured cases of the delta memory core's operators: the gated delta rule (whole
sequences with their gradients, prompts, single tokens), group norm with an activation
on channels-last tensors, and the clipped policy loss with a KL term that trains sampled
answers from their logits.

``run`` makes one pass through an operator, in its plain form (elementary torch
operations in 32 bits) or, with ``own`` set, through the framework's entry points;
``exact`` is the operator's definition in 64 bits.

Notation. Tokens are (b, t), value heads h < heads, key heads g < groups (heads / groups
value heads share one), a state S [values, keys] per (b, h). ``reset[b, t]`` says that
token t starts a new episode: nothing before it is seen. ``lengths[b]`` says how many
tokens of the row are real; the others change nothing, give zeros, and may hold anything
(the inputs here hold NaN there).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
NORM_EPS = 1e-6               # under the root of a key's and a query's length
CHUNK = 64                    # tokens that the plain form takes together


# ---- cases ------------------------------------------------------------------------
def listed():
    return [
        # one decision of a small env group: latency counts
        dict(name="delta step 64x8x64x64", op="delta_step", rows=64, pool=64, groups=8, heads=8, keys=64, values=64,
             dtype="bf16", reset=0.02),
        # one decision of the benchmark's 2048 envs
        dict(name="delta step 2048x8x64x64", op="delta_step", rows=2048, pool=2048, groups=8, heads=8, keys=64, values=64,
             dtype="bf16", reset=0.02),
        # a long recorded run read as a prompt, odd length, wide heads, state carried in
        dict(name="delta prompt 1x8191x8x128x128", op="delta", batch=1, length=8191, groups=8, heads=8, keys=128, values=128,
             dtype="bf16", reset=0.0, ragged=False),
        # ragged episodes in 32 bits, value heads that share keys, odd head sizes, an empty row
        dict(name="delta train 5x77x4x24x40 f32", op="delta_train", batch=5, length=77, groups=2, heads=4, keys=24, values=40,
             dtype="f32", reset=0.05, ragged=True),
        # the update of a rollout: 256 envs x 128 decisions, episodes ending inside the rows
        dict(name="delta train 256x128x8x64x64", op="delta_train", batch=256, length=128, groups=8, heads=8, keys=64, values=64,
             dtype="bf16", reset=0.02, ragged=False),
        # whole long runs, few rows
        dict(name="delta train 2x4096x16x64x64", op="delta_train", batch=2, length=4096, groups=16, heads=16, keys=64,
             values=64, dtype="bf16", reset=0.0005, ragged=False),
        # the heads of a rollout's core, each token normalised by itself
        dict(name="norm train 32768x1x512 g8", op="norm_train", batch=32768, positions=1, channels=512, groups=8,
             activation="silu", dtype="bf16"),
        # the trunk's images: 16 x 32 positions of 64 channels
        dict(name="norm train 2048x512x64 g8", op="norm_train", batch=2048, positions=512, channels=64, groups=8,
             activation="silu", dtype="bf16"),
        # one large image in 32 bits, odd sizes: an image's statistics span many SMs
        dict(name="norm 1x12321x120 g6 f32", op="norm", batch=1, positions=12321, channels=120, groups=6, activation="silu",
             dtype="f32"),
        # the answers of 2048 envs, one small head
        dict(name="policy 2048x15 f32", op="policy", rows=2048, vocab=15, dtype="f32", clip=0.2, kl=0.02, ent=0.01,
             temperature=1.0),
        # an update over many answers, vocabulary of an odd size
        dict(name="policy 4096x32003", op="policy", rows=4096, vocab=32003, dtype="bf16", clip=0.2, kl=0.05, ent=0.0,
             temperature=0.8),
        # few answers over the largest vocabulary: a row spans several SMs
        dict(name="policy 48x131072", op="policy", rows=48, vocab=131072, dtype="bf16", clip=0.1, kl=0.01, ent=0.001,
             temperature=1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: sizes spread over their logarithm, cut where a case would cost
    more than the largest listed one."""
    op = rng.choice(["delta_step", "delta", "delta_train", "delta_train", "norm", "norm_train", "policy", "policy"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "policy":
        vocab = _log_int(rng, 2, 131072)
        rows = _log_int(rng, 1, max(1, min(16384, (1 << 26) // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, clip=rng.choice([0.1, 0.2, 0.3]), kl=rng.choice([0.0, 0.02, 0.1]),
                    ent=rng.choice([0.0, 0.01]), temperature=rng.choice([1.0, 1.0, 0.7]))
    if op in ("norm", "norm_train"):
        groups = rng.choice([1, 2, 4, 8, 32])
        positions = rng.choice([1, _log_int(rng, 2, 16384)])
        channels = groups * _log_int(rng, 1 if positions >= 16 else 16, 64)     # what is normalised has 16 values or more
        batch = _log_int(rng, 1, max(1, min(65536, (1 << 25) // (positions * channels))))
        return dict(op=op, batch=batch, positions=positions, channels=channels, groups=groups,
                    activation=rng.choice(["none", "silu", "silu"]), dtype=dtype)
    groups = rng.choice([1, 2, 4, 8])
    heads = groups * rng.choice([1, 1, 1, 2, 3])
    keys, values = (rng.choice([16, 32, 64, 64, 128, rng.randint(4, 128)]) for _ in range(2))
    case = dict(op=op, groups=groups, heads=heads, keys=keys, values=values, dtype=dtype)
    if op == "delta_step":
        rows = _log_int(rng, 1, max(1, min(2048, (1 << 26) // (heads * keys * values))))
        return dict(case, rows=rows, pool=rows + _log_int(rng, 1, 64), reset=rng.choice([0.0, 0.05]))
    most = min(1 << 18, (1 << (30 if op == "delta" else 29)) // (keys * values)) // heads          # tokens
    length = _log_int(rng, 1, min(most, 8192 if op == "delta" else 4096))
    batch = _log_int(rng, 1, min(256, most // length))
    return dict(case, batch=batch, length=length, reset=rng.choice([0.0, 0.001, 0.05]), ragged=rng.random() < 0.4)


def work(case):
    e, op = SIZE[case["dtype"]], case["op"]
    if op == "policy":
        n, r = case["rows"] * case["vocab"], case["rows"]
        return {"bytes": 2 * n * e + r * 40, "flops": 10 * n}
    if op in ("norm", "norm_train"):
        n, c = case["batch"] * case["positions"] * case["channels"], case["channels"]
        fwd = {"bytes": 2 * n * e + 8 * c, "flops": 10 * n}
        return fwd if op == "norm" else {"bytes": 4 * n * e + 16 * c, "flops": 30 * n}
    g, h, k, v = case["groups"], case["heads"], case["keys"], case["values"]
    if op == "delta_step":
        r = case["rows"]
        return {"bytes": r * (e * (2 * g * k + 2 * h * v + 2 * h) + 8 * h * k * v), "flops": r * h * 7 * k * v}
    tokens = case["batch"] * case["length"]
    ends = case["batch"] * h * k * v * 8
    fwd = tokens * e * (2 * g * k + 2 * h * v + 2 * h) + ends + tokens
    if op == "delta":
        return {"bytes": fwd, "flops": tokens * h * 7 * k * v}
    return {"bytes": fwd + tokens * e * (2 * g * k + 2 * h * v + 2 * h) + ends, "flops": tokens * h * 23 * k * v}


# ---- inputs -----------------------------------------------------------------------
def _masks(case, gen, dev):
    b, t = case["batch"], case["length"]
    reset = torch.rand(b, t, generator=gen, device=dev) < case["reset"] if case["reset"] > 0 else None
    lengths = None
    if case["ragged"]:
        lengths = torch.randint(0, t + 1, (b,), generator=gen, device=dev, dtype=torch.int32)
        lengths[0] = t
        if b > 1:
            lengths[1] = 0
    return reset, lengths


def _spoil(x, lengths):
    """NaN in the tokens that are not real."""
    if lengths is not None:
        dead = torch.arange(x.shape[1], device=x.device)[None, :] >= lengths[:, None]
        x[dead] = float("nan")
    return x


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    s, op = dict(case), case["op"]
    if op == "policy":
        r, v = case["rows"], case["vocab"]
        z = 2.0 * randn(r, v)
        if v > 64:
            z[torch.rand(r, v, generator=gen, device=dev) < 0.02] = float("-inf")      # forbidden answers
        s["answers"] = torch.argmax(z + torch.empty_like(z).exponential_(generator=gen).log_().neg_(), 1).to(torch.int32)
        s["logits"] = z.to(dt)
        lp = torch.log_softmax(s["logits"].float() / case["temperature"], 1).gather(1, s["answers"].long()[:, None])[:, 0]
        moved = 0.2 * randn(r)                              # the policy has moved since it answered
        # no ratio within 0.001 of where it is clipped: 32 and 64 bits then clip the same rows
        near = ((torch.exp(moved) - 1).abs() - case["clip"]).abs() < 1e-3
        s["old_logp"] = lp - torch.where(near, 0.9 * moved, moved)
        s["ref_logp"] = lp + 0.3 * randn(r)
        s["advantages"] = 0.2 + randn(r)                    # this part of an update is better than the whole
        s["weights"] = torch.full((r,), 1.0 / r, device=dev)
        off = torch.rand(r, generator=gen, device=dev) < 0.05                          # decisions that count nothing
        s["answers"][off] = -1
        return s
    if op in ("norm", "norm_train"):
        c = case["channels"]
        shape = (case["batch"], case["positions"], c)
        s["x"] = (randn(*shape) * (0.5 + torch.rand(c, generator=gen, device=dev)) + 0.5 * randn(c)).to(dt)
        s["weight"], s["bias"] = 1.0 + 0.2 * randn(c), 0.2 * randn(c)
        if op == "norm_train":
            s["dy"] = randn(*shape).to(dt)
        return s
    g, h, k, v = case["groups"], case["heads"], case["keys"], case["values"]
    lead = (case["rows"],) if op == "delta_step" else (case["batch"], case["length"])
    s["len"] = None
    if op == "delta_step":
        r, p = case["rows"], case["pool"]
        s["reset_at"] = torch.rand(r, generator=gen, device=dev) < case["reset"] if case["reset"] > 0 else None
        s["slots"] = None
        if p > r:
            s["slots"] = torch.randperm(p, generator=gen, device=dev)[:r].to(torch.int32)
            s["slots"][r // 2] = -1                                                    # a row without an env
        s["state"] = 0.2 * randn(p, h, v, k)
    else:
        s["reset_at"], s["len"] = _masks(case, gen, dev)
        s["state"] = 0.2 * randn(case["batch"], h, v, k)
    # the core's convolution gives queries, keys and values side by side, behind a SiLU
    qkv = randn(*lead, 2 * g * k + h * v)
    qkv = _spoil((qkv * torch.sigmoid(qkv)).to(dt), s["len"])
    s["q"] = qkv[..., :g * k].unflatten(-1, (g, k))
    s["k"] = qkv[..., g * k:2 * g * k].unflatten(-1, (g, k))
    s["v"] = qkv[..., 2 * g * k:].unflatten(-1, (h, v))
    gates = _spoil(randn(*lead, 2 * h).to(dt), s["len"])                               # one projection gives both
    s["dt"], s["b"] = gates[..., :h], gates[..., h:]
    s["A"] = -(1.0 + 15.0 * torch.rand(h, generator=gen, device=dev))
    step = torch.exp(torch.rand(h, generator=gen, device=dev) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    s["dt_bias"] = torch.log(torch.expm1(step))
    if op == "delta_train":
        s["dout"] = _spoil(randn(*lead, h, v).to(dt), s["len"])
        s["dfinal"] = 0.2 * randn(case["batch"], h, v, k)
    return s


# ---- the plain forms --------------------------------------------------------------
def _softplus(v):
    return torch.where(v > 20.0, v, torch.log1p(torch.exp(v.clamp(max=20.0))))


def _unit(x):
    """(x / its length, 1 / its length) along the last axis."""
    r = torch.rsqrt((x * x).sum(-1, keepdim=True) + NORM_EPS)
    return x * r, r


def _heads_first(x, rep, pad):
    """[B, T, G, N] -> [B, H, chunks, CHUNK, N], zeros behind the row."""
    x = torch.cat([x, x.new_zeros(x.shape[0], pad, *x.shape[2:])], 1)
    x = x.repeat_interleave(rep, 2).transpose(1, 2)
    return x.unflatten(2, (-1, CHUNK))


def _tokens_first(x, t):
    """The way back of _heads_first."""
    return x.flatten(2, 3)[:, :, :t].transpose(1, 2)


def _delta_parts(s):
    """Everything of the chunks that does not depend on the state."""
    q, k, v = s["q"], s["k"], s["v"]
    b, t, g, _ = q.shape
    h = v.shape[2]
    dev = q.device
    real = torch.ones(b, t, dtype=torch.bool, device=dev) if s["len"] is None else \
        torch.arange(t, device=dev)[None, :] < s["len"][:, None]
    pad = -t % CHUNK
    on3, on4 = real[..., None], real[..., None, None]
    q, k, v = (torch.where(on4, x.float(), 0.0) for x in (q, k, v))
    qn, rq = _unit(q)
    kn, rk = _unit(k)
    pre = torch.where(on3, s["dt"].float(), 0.0) + s["dt_bias"]
    delta = torch.where(on3, _softplus(pre), 0.0)
    beta = torch.where(on3, torch.sigmoid(torch.where(on3, s["b"].float(), 0.0)), 0.0)
    p = dict(real=real, pre=pre, delta=delta, qn=qn, kn=kn, rq=rq, rk=rk, beta=beta, pad=pad)
    Q, K = (_heads_first(x, h // g, pad) for x in (qn, kn))
    V = _heads_first(v, 1, pad)
    beta, glog = (_heads_first(x[..., None], 1, pad)[..., 0] for x in (beta, delta * s["A"]))
    cut = torch.zeros(b, t, dtype=torch.bool, device=dev) if s["reset_at"] is None else s["reset_at"] & real
    seg = torch.cat([cut, cut.new_zeros(b, pad)], 1).view(b, 1, -1, CHUNK).long().cumsum(-1)
    # sums of logarithms in 64 bits: their differences are what decays
    G = glog.double().cumsum(-1)
    D = torch.exp((G[..., :, None] - G[..., None, :]).clamp(max=0.0)).float()
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=dev).tril()
    D = torch.where(lower & (seg[..., :, None] == seg[..., None, :]), D, 0.0)
    head = torch.where(seg == 0, torch.exp(G).float(), 0.0)               # of the state before the chunk
    tail = torch.where(seg == seg[..., -1:], torch.exp((G[..., -1:] - G).clamp(max=0.0)).float(), 0.0)
    M = (D * (K @ K.transpose(-1, -2))).tril(-1)
    P = s["scale"] * D * (Q @ K.transpose(-1, -2))
    # (I + M beta)^-1 row by row, of all chunks at once
    MB = M * beta[..., None, :]
    inv = torch.eye(CHUNK, device=dev).expand_as(MB).clone()
    for i in range(1, CHUNK):
        inv[..., i, :i] = -(MB[..., i, None, :i] @ inv[..., :i, :i])[..., 0, :]
    p.update(Q=Q, K=K, V=V, B=beta, D=D, head=head, tail=tail, M=M, P=P, inv=inv, glog=glog, end=head[..., -1])
    return p


def _delta_forward(s, p):
    """(out, final, states before the chunks, W) of the parts."""
    S = s["state"]
    Ss, Ws, Os = [], [], []
    for c in range(p["Q"].shape[2]):
        Ss.append(S)
        K, head = p["K"][:, :, c], p["head"][:, :, c, :, None]
        St = S.transpose(-1, -2)
        W = p["inv"][:, :, c] @ (p["V"][:, :, c] - head * (K @ St))
        U = p["B"][:, :, c, :, None] * W
        Os.append(s["scale"] * head * (p["Q"][:, :, c] @ St) + p["P"][:, :, c] @ U)
        S = p["end"][:, :, c, None, None] * S + (p["tail"][:, :, c, :, None] * U).transpose(-1, -2) @ K
        Ws.append(W)
    return torch.stack(Os, 2), S, Ss, Ws


def _delta_grad_plain(s, p, Ss, Ws):
    b, t, g, _ = s["q"].shape
    h = s["v"].shape[2]
    on4 = p["real"][..., None, None]
    dO = _heads_first(torch.where(on4, s["dout"].float(), 0.0), 1, p["pad"])
    dS = s["dfinal"]
    n = dO.shape[2]
    dQ, dK, dV, dB, dG = ([None] * n for _ in range(5))
    for c in range(n - 1, -1, -1):
        Q, K, D, M, P, inv = (p[x][:, :, c] for x in ("Q", "K", "D", "M", "P", "inv"))
        head, tail, beta = (p[x][:, :, c, :, None] for x in ("head", "tail", "B"))
        end, S, W, do = p["end"][:, :, c], Ss[c], Ws[c], dO[:, :, c]
        U = beta * W
        dU = P.transpose(-1, -2) @ do + tail * (K @ dS.transpose(-1, -2))
        Z = inv.transpose(-1, -2) @ (beta * dU)
        dM = -(Z @ U.transpose(-1, -2)).tril(-1)
        dP = (do @ U.transpose(-1, -2)).tril()
        dB[c] = (W * (dU - M.transpose(-1, -2) @ Z)).sum(-1)
        read = s["scale"] * head * (do @ S)
        keep = -head * (Z @ S)
        send = tail * (U @ dS)
        PD, MD = s["scale"] * dP * D, dM * D
        dQ[c] = read + PD @ K
        dK[c] = keep + send + PD.transpose(-1, -2) @ Q + MD @ K + MD.transpose(-1, -2) @ K
        # what a decay between two tokens gets cancels in the sums of all others: in 64 bits
        E = (dP * P + dM * M).double()
        f = (send * K).sum(-1).double()
        at = E.sum(-1) - E.sum(-2) + (read * Q).sum(-1) + (keep * K).sum(-1) - f
        at[..., -1] += f.sum(-1) + end * (dS * S).sum((-1, -2))
        dG[c] = at.flip(-1).cumsum(-1).flip(-1).float()
        dV[c] = Z
        dS = end[..., None, None] * dS + s["scale"] * (head * do).transpose(-1, -2) @ Q - (head * Z).transpose(-1, -2) @ K
    dQ, dK, dV = (_tokens_first(torch.stack(x, 2), t) for x in (dQ, dK, dV))
    dB, dG = (_tokens_first(torch.stack(x, 2)[..., None], t)[..., 0] for x in (dB, dG))
    dQ, dK = (x.unflatten(2, (g, h // g)).sum(3) for x in (dQ, dK))
    dq = p["rq"] * (dQ - p["qn"] * (p["qn"] * dQ).sum(-1, keepdim=True))
    dk = p["rk"] * (dK - p["kn"] * (p["kn"] * dK).sum(-1, keepdim=True))
    on3 = p["real"][..., None]
    db = torch.where(on3, dB * p["beta"] * (1 - p["beta"]), 0.0)
    dpre = torch.where(on3, dG * s["A"] * torch.sigmoid(p["pre"]), 0.0)
    return dict(dq=torch.where(on4, dq, 0.0), dk=torch.where(on4, dk, 0.0), dv=torch.where(on4, dV, 0.0), ddt=dpre, db=db,
                dA=torch.where(on3, dG * p["delta"], 0.0).sum((0, 1)), ddt_bias=dpre.sum((0, 1)), dstate=dS)


def _rows_of(s):
    """(rows that have a slot, their slots)."""
    r = s["v"].shape[0]
    if s["slots"] is None:
        return torch.ones(r, dtype=torch.bool, device=s["v"].device), torch.arange(r, device=s["v"].device)
    return s["slots"] >= 0, s["slots"].long().clamp(min=0)


def _delta_step_plain(s):
    on, at = _rows_of(s)
    rep = s["v"].shape[1] // s["q"].shape[1]
    old = s["state"][at]
    S = old
    if s["reset_at"] is not None:
        S = torch.where(s["reset_at"][:, None, None, None], 0.0, S)
    q, k = (_unit(x.float())[0].repeat_interleave(rep, 1) for x in (s["q"], s["k"]))
    decay = torch.exp(s["A"] * _softplus(s["dt"].float() + s["dt_bias"]))
    S = decay[..., None, None] * S
    u = torch.sigmoid(s["b"].float())[..., None] * (s["v"].float() - (S * k[:, :, None]).sum(-1))
    S = S + u[..., None] * k[:, :, None]
    out = s["scale"] * (S * q[:, :, None]).sum(-1)
    pool = torch.cat([s["state"], s["state"][:1]], 0)
    pool[torch.where(on, at, s["state"].shape[0])] = torch.where(on[:, None, None, None], S, old)
    s["state"].copy_(pool[:-1])
    return torch.where(on[:, None, None], out, 0.0)


def _norm_plain(s):
    x = s["x"].float()
    n, p, c = x.shape
    g = s["groups"]
    xg = x.view(n, p, g, c // g)
    mean = xg.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt(((xg - mean) ** 2).mean((1, 3), keepdim=True) + 1e-5)
    xh = ((xg - mean) * rstd).view(n, p, c)
    pre = xh * s["weight"] + s["bias"]
    sg = torch.sigmoid(pre)
    y, slope = {"none": (pre, None), "relu": (pre.clamp(min=0.0), (pre > 0).float()),
                "silu": (pre * sg, sg * (1 + pre * (1 - sg)))}[s["activation"]]
    if s["op"] == "norm":
        return (y,)
    d = s["dy"].float() if slope is None else s["dy"].float() * slope
    dw, db = (d * xh).sum((0, 1)), d.sum((0, 1))
    dh = (d * s["weight"]).view(n, p, g, c // g)
    xh = xh.view(n, p, g, c // g)
    dx = rstd * (dh - dh.mean((1, 3), keepdim=True) - xh * (dh * xh).mean((1, 3), keepdim=True))
    return y, dx.view(n, p, c), dw, db


def _policy_plain(s):
    z = s["logits"].float() / s["temperature"]
    z = torch.where(torch.isnan(z), float("-inf"), z)
    at = s["answers"].long().clamp(min=0)[:, None]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True, dtype=torch.float64)     # long sums, and what a small KL is the difference of
    log_total = torch.log(total)
    prob = e / total.float()
    logp_all = z - top - log_total.float()
    ent = -torch.where(prob > 0, prob * logp_all, 0.0).sum(1)
    lp = ((z.gather(1, at) - top) - log_total)[:, 0]
    on = (s["answers"] >= 0) & (lp > float("-inf"))
    lp = torch.where(on, lp, 0.0)
    ratio = torch.exp(lp - s["old_logp"])
    adv = s["advantages"]
    free, held = ratio * adv, ratio.clamp(1 - s["clip"], 1 + s["clip"]) * adv
    d = s["ref_logp"] - lp
    kl = torch.exp(d) - d - 1
    w = torch.where(on, s["weights"], 0.0)
    loss = (w * (-torch.minimum(free, held) + s["kl"] * kl - s["ent"] * ent)).sum()
    slope = w * (torch.where(free <= held, -free, 0.0) + s["kl"] * (1 - torch.exp(d)))
    slope = slope.float()
    grad = -slope[:, None] * prob + (w * s["ent"])[:, None] * torch.where(prob > 0, prob * (logp_all + ent[:, None]), 0.0)
    grad.scatter_add_(1, at, slope[:, None])
    return (loss.float(), lp.float(), torch.where(on, kl, 0.0).float(), torch.where(on, ent, 0.0), grad / s["temperature"])


def _run_plain(s):
    op, dt = s["op"], DTYPES[s["dtype"]]
    if op == "policy":
        loss, lp, kl, ent, grad = _policy_plain(s)
        return dict(loss=loss, logp=lp, kl=kl, entropy=ent, dlogits=grad.to(dt))
    if op in ("norm", "norm_train"):
        r = _norm_plain(s)
        return dict(zip(("out", "dx", "dweight", "dbias"), tuple(x.to(dt) for x in r[:2]) + r[2:]))
    s = dict(s, scale=s["keys"] ** -0.5)
    if op == "delta_step":
        return dict(out=_delta_step_plain(s).to(dt), state=s["state"])
    p = _delta_parts(s)
    O, final, Ss, Ws = _delta_forward(s, p)
    out = dict(out=torch.where(p["real"][..., None, None], _tokens_first(O, s["q"].shape[1]), 0.0).to(dt), final=final)
    if op == "delta_train":
        for k, v in _delta_grad_plain(s, p, Ss, Ws).items():
            out[k] = v.to(dt) if k in ("dq", "dk", "dv", "ddt", "db") else v
    return out


# ---- the framework's entry points -------------------------------------------------
def _run_own(s):
    op = s["op"]
    if op == "policy":
        from surfb200.ops import rl as R
        r = R.policy_loss(s["logits"], s["answers"], s["old_logp"], s["advantages"], ref_logp=s["ref_logp"],
                          weights=s["weights"], clip=s["clip"], kl_coef=s["kl"], ent_coef=s["ent"], temperature=s["temperature"])
        return dict(loss=r.loss, logp=r.logp, kl=r.kl, entropy=r.entropy, dlogits=r.dlogits)
    if op in ("norm", "norm_train"):
        from surfb200.ops import norm as N
        r = N.group_norm(s["x"], s["groups"], s["weight"], s["bias"], activation=s["activation"], train=op == "norm_train")
        out = dict(out=r.out)
        if op == "norm_train":
            d = N.group_norm_grad(s["dy"], s["x"], s["groups"], s["weight"], s["bias"], stats=r.stats, activation=s["activation"])
            out.update(dx=d.dx, dweight=d.dweight, dbias=d.dbias)
        return out
    from surfb200.ops import delta as DR
    args = (s["q"], s["k"], s["v"], s["dt"], s["b"], s["A"])
    if op == "delta_step":
        out = DR.gated_delta_step(*args, s["state"], dt_bias=s["dt_bias"], reset=s["reset_at"], slots=s["slots"])
        return dict(out=out, state=s["state"])
    kw = dict(dt_bias=s["dt_bias"], state=s["state"], reset=s["reset_at"], lengths=s["len"])
    r = DR.gated_delta(*args, train=op == "delta_train", **kw)
    out = dict(out=r.out, final=r.final)
    if op == "delta_train":
        d = DR.gated_delta_grad(s["dout"], *args, saved=r.saved, dfinal=s["dfinal"], **kw)
        out.update(dq=d.dq, dk=d.dk, dv=d.dv, ddt=d.ddt, db=d.db, dA=d.dA, ddt_bias=d.ddt_bias, dstate=d.dstate)
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ---------------------------------------------------
def _unit_of(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + NORM_EPS)


def _unit_back(d, x):
    """The gradient of x for the gradient d of _unit_of(x)."""
    n2 = (x * x).sum(-1, keepdim=True) + NORM_EPS
    return d / torch.sqrt(n2) - x * (d * x).sum(-1, keepdim=True) / (n2 * torch.sqrt(n2))


def _exact_delta(s, train):
    """The recurrence and its adjoint, one token after the other."""
    f = {x: s[x].double() for x in ("q", "k", "v", "dt", "b", "A", "dt_bias", "state")}
    bsz, t, g, K = f["q"].shape
    h = f["v"].shape[2]
    scale = K ** -0.5
    dev = s["q"].device
    n = torch.full((bsz,), t, device=dev) if s["len"] is None else s["len"].long()
    wide = lambda x: x.repeat_interleave(h // g, 1)  # noqa: E731

    def token(i):
        real = (i < n)[:, None]
        m3 = real[..., None]
        q, k, v = (torch.where(m3, f[x][:, i], 0.0) for x in ("q", "k", "v"))
        pre = torch.where(real, f["dt"][:, i], 0.0) + f["dt_bias"]
        delta = torch.logaddexp(pre, torch.zeros_like(pre))
        beta = 1 / (1 + torch.exp(-torch.where(real, f["b"][:, i], 0.0)))
        cut = torch.zeros_like(real) if s["reset_at"] is None else s["reset_at"][:, i:i + 1] & real
        return real, cut, q, k, v, wide(_unit_of(q)), wide(_unit_of(k)), pre, delta, beta

    S, kept, outs = f["state"], [], []
    for i in range(t):
        real, cut, _, _, v, qn, kn, _, delta, beta = token(i)
        m = real[..., None, None]
        past = torch.where(cut[..., None, None], 0.0, S)
        if train:
            kept.append(past)
        low = torch.exp(f["A"] * delta)[..., None, None] * past
        u = beta[..., None] * (v - torch.einsum("bhvk,bhk->bhv", low, kn))
        S = torch.where(m, low + u[..., None] * kn[:, :, None], S)
        outs.append(torch.where(m[..., 0], scale * torch.einsum("bhvk,bhk->bhv", S, qn), 0.0))
    out = dict(out=torch.stack(outs, 1), final=S)
    if not train:
        return out
    r = {x: [None] * t for x in ("dq", "dk", "dv", "ddt", "db")}
    dA, dbias = torch.zeros_like(f["A"]), torch.zeros_like(f["A"])
    dS, dout = s["dfinal"].double(), s["dout"].double()
    for i in range(t - 1, -1, -1):
        real, cut, q, k, v, qn, kn, pre, delta, beta = token(i)
        m = real[..., None, None]
        decay = torch.exp(f["A"] * delta)[..., None, None]
        low = decay * kept[i]
        w = v - torch.einsum("bhvk,bhk->bhv", low, kn)
        u = beta[..., None] * w
        new = low + u[..., None] * kn[:, :, None]
        do = torch.where(m[..., 0], dout[:, i], 0.0)
        dqn = scale * torch.einsum("bhvk,bhv->bhk", new, do)
        dn = dS + scale * do[..., None] * qn[:, :, None]
        du = torch.einsum("bhvk,bhk->bhv", dn, kn)
        dkn = torch.einsum("bhvk,bhv->bhk", dn, u)
        dv = beta[..., None] * du
        dkn = dkn - torch.einsum("bhvk,bhv->bhk", low, dv)
        dlow = dn - dv[..., None] * kn[:, :, None]
        dlog = (dlow * low).sum((-1, -2))
        zero = lambda x, at=real: torch.where(at.view(-1, *[1] * (x.dim() - 1)), x, 0.0)  # noqa: E731
        fold = lambda x: x.view(bsz, g, h // g, K).sum(2)  # noqa: E731
        r["dq"][i], r["dk"][i] = zero(_unit_back(fold(dqn), q)), zero(_unit_back(fold(dkn), k))
        r["dv"][i] = zero(dv)
        r["db"][i] = zero((du * w).sum(-1) * beta * (1 - beta))
        r["ddt"][i] = zero(dlog * f["A"] / (1 + torch.exp(-pre)))
        dA += zero(dlog * delta).sum(0)
        dbias += r["ddt"][i].sum(0)
        dS = torch.where(m, torch.where(cut[..., None, None], 0.0, dlow * decay), dS)
    out.update({x: torch.stack(v, 1) for x, v in r.items()}, dA=dA, ddt_bias=dbias, dstate=dS)
    return out


def _exact_step(s):
    r = s["v"].shape[0]
    dev = s["v"].device
    on = torch.ones(r, dtype=torch.bool, device=dev) if s["slots"] is None else s["slots"] >= 0
    at = (torch.arange(r, device=dev) if s["slots"] is None else s["slots"].long())[on]
    pool = s["state"].double().clone()
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device=dev)
    q, k, v, dt, b = (s[x][on].double() for x in ("q", "k", "v", "dt", "b"))
    rep = v.shape[1] // q.shape[1]
    q, k = (_unit_of(x).repeat_interleave(rep, 1) for x in (q, k))
    S = pool[at]
    if s["reset_at"] is not None:
        S = S * (~s["reset_at"][on]).double()[:, None, None, None]
    pre = dt + s["dt_bias"].double()
    S = torch.exp(s["A"].double() * torch.logaddexp(pre, torch.zeros_like(pre)))[..., None, None] * S
    u = (v - torch.einsum("rhvk,rhk->rhv", S, k)) / (1 + torch.exp(-b))[..., None]
    S = S + torch.einsum("rhv,rhk->rhvk", u, k)
    out[on] = torch.einsum("rhvk,rhk->rhv", S, q) * s["keys"] ** -0.5
    pool[at] = S
    return dict(out=out, state=pool)


def _exact_norm(s):
    x = s["x"].double()
    n, p, c = x.shape
    g = s["groups"]
    per = lambda v: v.reshape(n, p, g, c // g).transpose(1, 2).reshape(n, g, -1)  # noqa: E731
    back = lambda v: v.reshape(n, g, p, c // g).transpose(1, 2).reshape(n, p, c)  # noqa: E731
    var, mean = torch.var_mean(per(x), -1, correction=0, keepdim=True)
    sd = torch.sqrt(var + 1e-5)
    xh = (per(x) - mean) / sd
    w = s["weight"].double()
    pre = back(xh) * w + s["bias"].double()
    act = s["activation"]
    if act == "none":
        y, slope = pre, torch.ones_like(pre)
    elif act == "relu":
        y, slope = torch.where(pre > 0, pre, 0.0), (pre > 0).double()
    else:
        sg = 1 / (1 + torch.exp(-pre))
        y, slope = pre * sg, sg + pre * sg * (1 - sg)
    if s["op"] == "norm":
        return dict(out=y)
    d = s["dy"].double() * slope
    a = per(d * w)
    dx = (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True)) / sd
    return dict(out=y, dx=back(dx), dweight=(d * back(xh)).sum((0, 1)), dbias=d.sum((0, 1)))


def _exact_policy(s):
    z = s["logits"].double() / s["temperature"]
    live = ~torch.isnan(z) & (z > float("-inf"))
    z = torch.where(live, z, float("-inf"))
    on = (s["answers"] >= 0) & live.gather(1, s["answers"].long().clamp(min=0)[:, None])[:, 0]
    z = torch.where(on[:, None], z, 0.0)                    # rows that count nothing: any finite numbers
    live = live | ~on[:, None]
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(logp)
    ent = -torch.where(live, p * torch.where(live, logp, 0.0), 0.0).sum(1)
    one = torch.zeros_like(z).scatter_(1, s["answers"].long().clamp(min=0)[:, None], 1.0)
    lp = torch.where(one > 0, logp, 0.0).sum(1)
    old, ref, adv = (s[x].double() for x in ("old_logp", "ref_logp", "advantages"))
    ratio = torch.exp(lp - old)
    lo, hi = 1 - s["clip"], 1 + s["clip"]
    free, held = ratio * adv, torch.clamp(ratio, lo, hi) * adv
    kl = torch.exp(ref - lp) - (ref - lp) - 1
    w = torch.where(on, s["weights"].double(), 0.0)
    loss = (w * (s["kl"] * kl - torch.minimum(free, held) - s["ent"] * ent)).sum()
    moves = ~(((ratio > hi) & (adv > 0)) | ((ratio < lo) & (adv < 0)))
    c = w * (s["kl"] * (1 - torch.exp(ref - lp)) - torch.where(moves, free, 0.0))
    grad = c[:, None] * (one - p) + (w * s["ent"])[:, None] * torch.where(live, p * (torch.where(live, logp, 0.0) + ent[:, None]), 0.0)
    zero = lambda v: torch.where(on, v, 0.0)  # noqa: E731
    return dict(loss=loss, logp=zero(lp), kl=zero(kl), entropy=zero(ent), dlogits=grad / s["temperature"])


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "policy":
        return _exact_policy(s)
    if op in ("norm", "norm_train"):
        return _exact_norm(s)
    if op == "delta_step":
        return _exact_step(s)
    train = op == "delta_train"
    if train and 8 * case["batch"] * case["length"] * case["heads"] * case["keys"] * case["values"] > 3e10:
        return None                                          # the states of every token would not fit
    return _exact_delta(s, train)
