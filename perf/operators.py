"""Measured cases of the sequence operators: the short causal convolution and the
selective state space scan of a policy's memory core (whole sequences with their
gradients, prompts, single tokens) and the sampling of its answers.

``run`` makes one pass through an operator, in its plain form (elementary torch
operations in 32 bits) or, with ``own`` set, through the framework's entry points;
``exact`` is the operator's definition in 64 bits.

Notation. Tokens are (b, t) with b < batch and t < length, channels d, states n.
``reset[b, t]`` says that token t starts a new episode: nothing before it is seen.
``lengths[b]`` says how many tokens of the row are real; the others change nothing,
give zeros, and may hold anything (the inputs here hold NaN there).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
FIX = float(1 << 40)          # sampling weights are whole multiples of 2^-40


# ---- cases ------------------------------------------------------------------------
def listed():
    return [
        # one rollout decision of a small env group: latency counts
        dict(name="conv step 64x1024", op="conv_step", rows=64, pool=64, dim=1024, width=4, dtype="bf16", reset=0.01),
        # a long recorded run read as a prompt, odd length, state carried in
        dict(name="conv prompt 1x16385x1024", op="conv", batch=1, length=16385, dim=1024, width=4, dtype="bf16",
             reset=0.001, ragged=False),
        # the update of a rollout: 256 envs x 128 decisions, episodes ending inside the rows
        dict(name="conv train 256x128x1024", op="conv_train", batch=256, length=128, dim=1024, width=4, dtype="bf16",
             reset=0.02, ragged=False),
        # one decision of a small group, inactive slots among it
        dict(name="scan step 32x512x16", op="scan_step", rows=32, pool=48, dim=512, state=16, groups=1, dtype="bf16",
             reset=0.05),
        # one decision of the benchmark's 2048 envs
        dict(name="scan step 2048x1024x16", op="scan_step", rows=2048, pool=2048, dim=1024, state=16, groups=1,
             dtype="bf16", reset=0.02),
        # ragged episodes in 32 bits, shared heads, an empty row: an odd small update
        dict(name="scan train 5x77x194x8 f32", op="scan_train", batch=5, length=77, dim=194, state=8, groups=2,
             dtype="f32", reset=0.05, ragged=True),
        # the update of a rollout: 256 envs x 128 decisions
        dict(name="scan train 256x128x512x16", op="scan_train", batch=256, length=128, dim=512, state=16, groups=1,
             dtype="bf16", reset=0.02, ragged=False),
        # whole long runs, few rows: the length has to be split
        dict(name="scan train 2x4096x1024x16", op="scan_train", batch=2, length=4096, dim=1024, state=16, groups=1,
             dtype="bf16", reset=0.0005, ragged=False),
        # one long prompt
        dict(name="scan prompt 1x8191x1024x16", op="scan", batch=1, length=8191, dim=1024, state=16, groups=1,
             dtype="bf16", reset=0.0, ragged=False),
        # the action heads of 2048 envs, each head an answer of its own
        dict(name="sample heads 2048x6", op="sample", rows=2048, vocab=32, heads=True, dtype="f32", temperature=0.8,
             top_k=0, top_p=0.9, min_p=0.02),
        # one answer over a large vocabulary
        dict(name="sample 1x32768", op="sample", rows=1, vocab=32768, heads=False, dtype="f32", temperature=0.7,
             top_k=50, top_p=0.95, min_p=0.0),
        # a serving batch over the largest vocabulary
        dict(name="sample 256x131072", op="sample", rows=256, vocab=131072, heads=False, dtype="bf16",
             temperature=1.0, top_k=0, top_p=0.95, min_p=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: sizes spread over their logarithm, cut where a case would cost
    more than the largest listed one."""
    op = rng.choice(["conv_step", "conv", "conv_train", "scan_step", "scan", "scan_train", "scan_train", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "sample":
        if rng.random() < 0.3:
            return dict(op=op, rows=_log_int(rng, 1, 8192), vocab=32, heads=True, dtype=dtype,
                        temperature=round(rng.uniform(0.3, 1.5), 3), top_k=rng.choice([0, 2, 3]),
                        top_p=rng.choice([1.0, 0.9, 0.5]), min_p=rng.choice([0.0, 0.05]))
        vocab = _log_int(rng, 33, 131072)
        rows = _log_int(rng, 1, max(1, min(1024, (256 * 131072) // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, heads=False, dtype=dtype, temperature=round(rng.uniform(0.3, 1.5), 3),
                    top_k=rng.choice([0, 0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 0.95, 0.9, 0.5]),
                    min_p=rng.choice([0.0, 0.0, 0.05]))
    if op in ("conv_step", "scan_step"):
        rows, dim = _log_int(rng, 1, 2048), _log_int(rng, 16, 1024)
        case = dict(op=op, rows=rows, pool=rows + _log_int(rng, 1, 64), dim=dim, dtype=dtype, reset=rng.choice([0.0, 0.05]))
        if op == "conv_step":
            return dict(case, width=rng.choice([2, 3, 4, 4]))
        groups = rng.choice([1, 1, 2, 4])
        return dict(case, dim=max(1, dim // groups) * groups, state=rng.choice([4, 8, 16, 16, 24]), groups=groups)
    if op in ("conv", "conv_train"):
        length, dim = _log_int(rng, 1, 16384), _log_int(rng, 16, 1024)
        batch = _log_int(rng, 1, max(1, min(512, (1 << 24) // (length * dim))))
        return dict(op=op, batch=batch, length=length, dim=dim, width=rng.choice([2, 3, 4, 4]), dtype=dtype,
                    reset=rng.choice([0.0, 0.001, 0.05]), ragged=rng.random() < 0.4)
    state, groups = rng.choice([4, 8, 16, 16, 16, 24, 64]), rng.choice([1, 1, 1, 2, 4])
    length, dim = _log_int(rng, 1, 8192), _log_int(rng, 16, 1024)
    dim = max(1, dim // groups) * groups
    length = min(length, (1 << 27) // (dim * state))
    batch = _log_int(rng, 1, max(1, min(256, (1 << 27) // (length * dim * state))))
    return dict(op=op, batch=batch, length=length, dim=dim, state=state, groups=groups, dtype=dtype,
                reset=rng.choice([0.0, 0.001, 0.05]), ragged=rng.random() < 0.4)


HEADS = (15, 7, 3, 3, 2, 2)       # categories of the framework's six action heads


def work(case):
    e = SIZE[case["dtype"]]
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + case["rows"] * (len(HEADS) if case["heads"] else 1) * 12, "flops": 8 * n}
    if op == "conv_step":
        n, w = case["rows"] * case["dim"], case["width"]
        return {"bytes": n * e * (2 + 2 * (w - 1)) + case["dim"] * (w + 1) * 4, "flops": n * (2 * w + 4)}
    if op == "scan_step":
        n, s = case["rows"] * case["dim"], case["state"]
        return {"bytes": n * (4 * e + 8 * s) + case["rows"] * case["groups"] * s * 2 * e + case["dim"] * (s + 2) * 4,
                "flops": n * (7 * s + 12)}
    tokens = case["batch"] * case["length"]
    n = tokens * case["dim"]
    if op in ("conv", "conv_train"):
        w = case["width"]
        ends = case["batch"] * (w - 1) * case["dim"] * e * 2
        if op == "conv":
            return {"bytes": n * 2 * e + ends + tokens, "flops": n * (2 * w + 4)}
        return {"bytes": n * 4 * e + 2 * ends + tokens, "flops": n * (2 * w + 4) + n * (6 * w + 10)}
    s = case["state"]
    ends = case["batch"] * case["dim"] * s * 4 * 2
    shared = tokens * case["groups"] * s * e
    if op == "scan":
        return {"bytes": n * 4 * e + 2 * shared + ends + tokens, "flops": n * (7 * s + 12)}
    return {"bytes": n * 8 * e + 4 * shared + 2 * ends + tokens, "flops": n * (7 * s + 12) + n * (20 * s + 30)}


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


def _scan_weights(case, gen, dev):
    d, n = case["dim"], case["state"]
    a = -(torch.arange(1, n + 1, device=dev, dtype=torch.float32)[None, :] *
          torch.exp(0.2 * torch.randn(d, n, generator=gen, device=dev)))
    step = torch.exp(torch.rand(d, generator=gen, device=dev) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    return dict(A=a.contiguous(), D=torch.randn(d, generator=gen, device=dev), dt_bias=torch.log(torch.expm1(step)))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    s = dict(case)
    op = case["op"]
    if op == "sample":
        r, v = case["rows"], case["vocab"]
        if case["heads"]:
            # the columns of a policy's output row, wider than the logits
            s["logits"] = (1.5 * randn(r, 64)).to(dt)[:, :v]
            s["u"] = torch.rand(r, len(HEADS), generator=gen, device=dev)
        else:
            z = 2.5 * randn(r, v)
            at = torch.randint(0, v, (r, min(24, v)), generator=gen, device=dev)
            z.scatter_add_(1, at, 3.0 + 3.0 * torch.rand(at.shape, generator=gen, device=dev))
            z[torch.rand(r, v, generator=gen, device=dev) < 0.02] = float("-inf")      # forbidden answers
            s["logits"] = z.to(dt)
            s["u"] = torch.rand(r, 1, generator=gen, device=dev)
        return s
    d = case["dim"]
    if op in ("conv_step", "scan_step"):
        r, p = case["rows"], case["pool"]
        s["reset_rows"] = torch.rand(r, generator=gen, device=dev) < case["reset"] if case["reset"] > 0 else None
        s["slots"] = None
        if p > r:
            s["slots"] = torch.randperm(p, generator=gen, device=dev)[:r].to(torch.int32)
            s["slots"][r // 2] = -1                                                    # a row without an env
        xz = randn(r, 2 * d).to(dt)                         # one projection gives both
        s["x"], s["z"] = xz[:, :d], xz[:, d:]
        if op == "conv_step":
            w = case["width"]
            s["weight"], s["bias"] = randn(d, w) / math.sqrt(w), 0.1 * randn(d)
            s["state_rows"] = randn(p, w - 1, d).to(dt)
            return s
        g, n = case["groups"], case["state"]
        s.update(_scan_weights(case, gen, dev))
        s["dt"] = (0.5 * randn(r, d)).to(dt)
        bc = randn(r, 2 * g * n).to(dt)
        s["B"], s["C"] = bc[:, :g * n].unflatten(1, (g, n)), bc[:, g * n:].unflatten(1, (g, n))
        s["state_rows"] = randn(p, d, n)
        return s
    b, t = case["batch"], case["length"]
    s["reset_at"], s["len"] = _masks(case, gen, dev)
    xz = _spoil(randn(b, t, 2 * d).to(dt), s["len"])        # one projection gives both
    s["x"], s["z"] = xz[..., :d], xz[..., d:]
    if op in ("conv", "conv_train"):
        w = case["width"]
        s["weight"], s["bias"] = randn(d, w) / math.sqrt(w), 0.1 * randn(d)
        s["start"] = randn(b, w - 1, d).to(dt)
        if op == "conv_train":
            s["dy"] = _spoil(randn(b, t, d).to(dt), s["len"])
            s["dfinal"] = randn(b, w - 1, d).to(dt)
        return s
    g, n = case["groups"], case["state"]
    s.update(_scan_weights(case, gen, dev))
    s["dt"] = _spoil((0.5 * randn(b, t, d)).to(dt), s["len"])
    bc = _spoil(randn(b, t, 2 * g * n).to(dt), s["len"])    # one projection gives both
    s["B"], s["C"] = bc[..., :g * n].unflatten(2, (g, n)), bc[..., g * n:].unflatten(2, (g, n))
    s["start"] = randn(b, d, n)
    if op == "scan_train":
        s["dout"] = _spoil(randn(b, t, d).to(dt), s["len"])
        s["dfinal"] = randn(b, d, n)
    return s


# ---- the plain forms --------------------------------------------------------------
def _live(lengths, b, t, dev):
    """[B, T] truth values: the token is real."""
    if lengths is None:
        return torch.ones(b, t, dtype=torch.bool, device=dev)
    return torch.arange(t, device=dev)[None, :] < lengths[:, None]


def _conv_taps(s):
    """The inputs of every token's taps [B, T, D, W], whether each is seen [B, T, 1, W],
    and what the next token would find behind it."""
    x, w = s["x"], s["weight"].shape[1]
    b, t, d = x.shape
    live = _live(s["len"], b, t, x.device)
    xf = torch.where(live[..., None], x.float(), 0.0)
    ext = torch.cat([s["start"].float(), xf], 1)
    ep = torch.zeros(b, t, dtype=torch.int64, device=x.device) if s["reset_at"] is None else \
        (s["reset_at"] & live).long().cumsum(1)
    ext_ep = torch.cat([torch.zeros(b, w - 1, dtype=torch.int64, device=x.device), ep], 1)
    taps = ext.unfold(1, w, 1)
    seen = (ext_ep.unfold(1, w, 1) == ep[..., None]) & live[..., None]
    n = torch.full((b,), t, device=x.device) if s["len"] is None else s["len"].long()
    at = n[:, None] + torch.arange(w - 1, device=x.device)[None, :]
    last = torch.where(n > 0, ext_ep.gather(1, (n + w - 2).clamp(min=0)[:, None])[:, 0], 0)
    keep = ext_ep.gather(1, at) == last[:, None]
    return live, ext, taps, seen[:, :, None, :], at, keep


def _conv_plain(s):
    live, ext, taps, seen, at, keep = _conv_taps(s)
    pre = torch.where(seen, taps * s["weight"], 0.0).sum(-1) + s["bias"]
    y = torch.where(live[..., None], pre * torch.sigmoid(pre), 0.0)
    final = torch.where(keep[..., None], ext.gather(1, at[..., None].expand(-1, -1, ext.shape[2])), 0.0)
    return y, final, pre


def _conv_grad_plain(s, pre):
    live, ext, taps, seen, at, keep = _conv_taps(s)
    w = s["weight"]
    t = pre.shape[1]
    sg = torch.sigmoid(pre)
    dpre = torch.where(live[..., None], s["dy"].float() * (sg * (1 + pre * (1 - sg))), 0.0)
    dw = torch.where(seen, taps * dpre[..., None], 0.0).sum((0, 1))
    dext = torch.zeros_like(ext)
    for k in range(w.shape[1]):
        dext[:, k:k + t] += torch.where(seen[..., k], dpre * w[:, k], 0.0)
    dext.scatter_add_(1, at[..., None].expand(-1, -1, ext.shape[2]), torch.where(keep[..., None], s["dfinal"].float(), 0.0))
    head = w.shape[1] - 1
    return dext[:, head:], dw, dpre.sum((0, 1)), dext[:, :head]


def _linear_scan(a, b):
    """h[t] = a[t] h[t - 1] + b[t] along dimension 1, h[-1] = 0, by doubling."""
    off = 1
    while off < a.shape[1]:
        b = torch.cat([b[:, :off], b[:, off:] + a[:, off:] * b[:, :-off]], 1)
        a = torch.cat([a[:, :off], a[:, off:] * a[:, :-off]], 1)
        off *= 2
    return b


def _softplus(v):
    return torch.where(v > 20.0, v, torch.log1p(torch.exp(v.clamp(max=20.0))))


def _scan_parts(s):
    x = s["x"]
    b, t, d = x.shape
    live = _live(s["len"], b, t, x.device)
    on = live[..., None]
    g = s["B"].shape[2]
    p = dict(live=on, x=torch.where(on, x.float(), 0.0), z=torch.where(on, s["z"].float(), 0.0),
             v=torch.where(on, s["dt"].float(), 0.0) + s["dt_bias"],
             B=torch.where(on[..., None], s["B"].float(), 0.0).repeat_interleave(d // g, 2),
             C=torch.where(on[..., None], s["C"].float(), 0.0).repeat_interleave(d // g, 2))
    p["delta"] = torch.where(on, _softplus(p["v"]), 0.0)
    p["a"] = torch.exp(p["delta"][..., None] * s["A"])
    if s["reset_at"] is not None:
        p["a"] = torch.where((s["reset_at"] & live)[..., None, None], 0.0, p["a"])
    u = (p["delta"] * p["x"])[..., None] * p["B"]
    u[:, 0] += p["a"][:, 0] * s["start"]
    p["h"] = _linear_scan(p["a"], u)
    p["y"] = (p["h"] * p["C"]).sum(-1) + s["D"] * p["x"]
    p["sz"] = torch.sigmoid(p["z"])
    return p


def _scan_grad_plain(s, p):
    b, t, d = p["x"].shape
    g, n = s["B"].shape[2:]
    dout = torch.where(p["live"], s["dout"].float(), 0.0)
    gate = p["z"] * p["sz"]
    dz = dout * p["y"] * (p["sz"] * (1 + p["z"] * (1 - p["sz"])))
    gy = dout * gate
    gh = gy[..., None] * p["C"]
    gh[:, -1] += s["dfinal"]
    later = torch.cat([p["a"][:, 1:], torch.zeros_like(p["a"][:, :1])], 1)
    dh = _linear_scan(later.flip(1), gh.flip(1)).flip(1)
    before = torch.cat([s["start"][:, None], p["h"][:, :-1]], 1)
    q = dh * p["a"] * before
    ub = (dh * p["B"]).sum(-1)
    ddelta = (q * s["A"]).sum(-1) + ub * p["x"]
    dv = torch.where(p["live"], ddelta * torch.sigmoid(p["v"]), 0.0)
    dx = ub * p["delta"] + gy * s["D"]
    dB = (dh * (p["delta"] * p["x"])[..., None]).view(b, t, g, d // g, n).sum(3)
    dC = (gy[..., None] * p["h"]).view(b, t, g, d // g, n).sum(3)
    return dict(dx=dx, ddt=dv, dz=dz, dB=torch.where(p["live"][..., None], dB, 0.0), dC=dC,
                dA=(q * p["delta"][..., None]).sum((0, 1)), dD=(gy * p["x"]).sum((0, 1)), ddt_bias=dv.sum((0, 1)),
                dstate=p["a"][:, 0] * dh[:, 0])


def _rows_of(s):
    """(rows that have a slot, their slots)."""
    if s["slots"] is None:
        on = torch.ones(s["x"].shape[0], dtype=torch.bool, device=s["x"].device)
        return on, torch.arange(s["x"].shape[0], device=s["x"].device)
    return s["slots"] >= 0, s["slots"].long().clamp(min=0)


def _put_rows(state, on, at, old, new):
    """state[at[r]] = new[r] for the rows that have a slot."""
    wide = on.view(-1, *[1] * (new.dim() - 1))
    extra = torch.cat([state, state[:1]], 0)
    extra[torch.where(on, at, state.shape[0])] = torch.where(wide, new, old).to(state.dtype)
    state.copy_(extra[:-1])


def _conv_step_plain(s):
    on, at = _rows_of(s)
    old = s["state_rows"][at]
    seen = old.float()
    if s["reset_rows"] is not None:
        seen = torch.where(s["reset_rows"][:, None, None], 0.0, seen)
    taps = torch.cat([seen, s["x"].float()[:, None]], 1)
    pre = (taps * s["weight"].t()).sum(1) + s["bias"]
    _put_rows(s["state_rows"], on, at, old, taps[:, 1:].to(s["x"].dtype))
    return torch.where(on[:, None], pre * torch.sigmoid(pre), 0.0)


def _scan_step_plain(s):
    on, at = _rows_of(s)
    old = s["state_rows"][at]
    h = old
    if s["reset_rows"] is not None:
        h = torch.where(s["reset_rows"][:, None, None], 0.0, h)
    x, z = s["x"].float(), s["z"].float()
    r, d = x.shape
    g = s["B"].shape[1]
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    B, C = (s[k].float().repeat_interleave(d // g, 1) for k in ("B", "C"))
    new = torch.exp(delta[..., None] * s["A"]) * h + (delta * x)[..., None] * B
    y = ((new * C).sum(-1) + s["D"] * x) * (z * torch.sigmoid(z))
    _put_rows(s["state_rows"], on, at, old, new)
    return torch.where(on[:, None], y, 0.0)


def _sample_rows_plain(logits, u, s):
    """(answers [R], log-probabilities [R]) of rows of logits and one number each."""
    z = logits.float()
    z = torch.where(torch.isnan(z), float("-inf"), z)
    top = z.amax(1, keepdim=True)
    inv = 1.0 / torch.tensor(s["temperature"], dtype=torch.float32, device=z.device)
    e = torch.where(z == top, 1.0, torch.exp((z - top) * inv))
    weight = torch.where(z > float("-inf"), e * FIX, 0.0).long()
    weight = torch.where(e >= s["min_p"], weight, 0)
    order = torch.sort(z, dim=1, descending=True, stable=True).indices
    ranked = weight.gather(1, order)
    if s["top_k"] > 0:
        ranked[:, s["top_k"]:] = 0
    upto = ranked.cumsum(1)
    if s["top_p"] < 1.0:
        p = torch.tensor(s["top_p"], dtype=torch.float32).double().item()
        most = torch.ceil(p * upto[:, -1:].double()).long().clamp(min=1)
        ranked = torch.where(upto - ranked < most, ranked, 0)
    weight = torch.zeros_like(weight).scatter_(1, order, ranked)
    upto = weight.cumsum(1)
    total = upto[:, -1:]
    at = torch.minimum((u[:, None].double() * total.double()).long(), total - 1)
    token = (upto <= at).sum(1, keepdim=True).clamp(max=z.shape[1] - 1)
    logp = torch.log(weight.gather(1, token).double() / total.double()).float()
    return torch.where(total > 0, token, -1)[:, 0].int(), torch.where(total > 0, logp, float("-inf"))[:, 0]


def _sample_plain(s):
    if not s["heads"]:
        return tuple(v[:, None] for v in _sample_rows_plain(s["logits"], s["u"][:, 0], s))
    parts = [_sample_rows_plain(z, s["u"][:, k], s) for k, z in enumerate(s["logits"].split(HEADS, 1))]
    return torch.stack([p[0] for p in parts], 1), torch.stack([p[1] for p in parts], 1)


def _run_plain(s):
    op, dt = s["op"], DTYPES[s["dtype"]]
    if op == "sample":
        return _sample_plain(s)
    if op == "conv_step":
        return _conv_step_plain(s).to(dt), s["state_rows"]
    if op == "scan_step":
        return _scan_step_plain(s).to(dt), s["state_rows"]
    if op in ("conv", "conv_train"):
        y, final, pre = _conv_plain(s)
        out = (y.to(dt), final.to(dt))
        if op == "conv_train":
            dx, dw, db, dstate = _conv_grad_plain(s, pre)
            out += (dx.to(dt), dw, db, dstate.to(dt))
        return out
    p = _scan_parts(s)
    out = {"out": (p["y"] * (p["z"] * p["sz"])).to(dt), "final": p["h"][:, -1]}
    if op == "scan_train":
        for k, v in _scan_grad_plain(s, p).items():
            out[k] = v.to(dt) if k in ("dx", "ddt", "dz", "dB", "dC") else v
    return out


# ---- the framework's entry points -------------------------------------------------
def _run_own(s):
    op = s["op"]
    if op == "sample":
        from surfb200.ops import tokens as TK
        return TK.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                min_p=s["min_p"], heads=HEADS if s["heads"] else None)
    from surfb200.ops import ssm as S
    if op == "conv_step":
        y = S.causal_conv_step(s["x"], s["weight"], s["bias"], s["state_rows"], reset=s["reset_rows"], slots=s["slots"])
        return y, s["state_rows"]
    if op == "scan_step":
        y = S.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state_rows"], D=s["D"], z=s["z"],
                                  dt_bias=s["dt_bias"], reset=s["reset_rows"], slots=s["slots"])
        return y, s["state_rows"]
    masks = dict(reset=s["reset_at"], lengths=s["len"])
    if op in ("conv", "conv_train"):
        y, final = S.causal_conv(s["x"], s["weight"], s["bias"], state=s["start"], **masks)
        if op == "conv":
            return y, final
        g = S.causal_conv_grad(s["dy"], s["x"], s["weight"], s["bias"], state=s["start"], dfinal=s["dfinal"], **masks)
        return y, final, g.dx, g.dweight, g.dbias, g.dstate
    args = (s["x"], s["dt"], s["A"], s["B"], s["C"])
    kw = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["start"], **masks)
    r = S.selective_scan(*args, train=op == "scan_train", **kw)
    out = {"out": r.out, "final": r.final}
    if op == "scan_train":
        g = S.selective_scan_grad(s["dout"], *args, saved=r.saved, dfinal=s["dfinal"], **kw)
        out.update(dx=g.dx, ddt=g.ddt, dz=g.dz, dB=g.dB, dC=g.dC, dA=g.dA, dD=g.dD, ddt_bias=g.ddt_bias, dstate=g.dstate)
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ---------------------------------------------------
def _exact_conv(s, train):
    """Token by token, tap by tap, as the definition says it."""
    x, st = s["x"].double(), s["start"].double()
    w, bias = s["weight"].double(), s["bias"].double()
    b, t, d = x.shape
    width = w.shape[1]
    n = torch.full((b,), t, device=x.device) if s["len"] is None else s["len"].long()
    reset = torch.zeros(b, t, dtype=torch.bool, device=x.device) if s["reset_at"] is None else s["reset_at"]
    hist = [st[:, j] for j in range(width - 1)]             # oldest first
    y, marks = [], []
    for i in range(t):
        real = (i < n)[:, None]
        cut = reset[:, i:i + 1] & real
        past = [torch.where(cut, 0.0, h) for h in hist]
        taps = past + [torch.where(real, x[:, i], 0.0)]
        pre = bias + sum(w[:, k] * taps[k] for k in range(width))
        y.append(torch.where(real, pre / (1 + torch.exp(-pre)), 0.0))
        marks.append((real, cut, taps, pre))
        hist = [torch.where(real, taps[k + 1], hist[k]) for k in range(width - 1)]
    zeros = torch.zeros(b, 0, d, dtype=torch.float64, device=x.device)
    out = [torch.stack(y, 1) if t else zeros, torch.stack(hist, 1)]
    if not train:
        return tuple(out)
    dy = s["dy"].double()
    dh = [s["dfinal"].double()[:, j] for j in range(width - 1)]
    dx, dw, db = [None] * t, torch.zeros_like(w), torch.zeros_like(bias)
    for i in range(t - 1, -1, -1):
        real, cut, taps, pre = marks[i]
        sg = 1 / (1 + torch.exp(-pre))
        dp = torch.where(real, dy[:, i] * (sg + pre * sg * (1 - sg)), 0.0)
        db += dp.sum(0)
        dw += torch.stack([(dp * taps[k]).sum(0) for k in range(width)], 1)
        dt = [dp * w[:, k] + (dh[k - 1] if k > 0 else 0.0) for k in range(width)]
        dx[i] = torch.where(real, dt[-1], 0.0)
        dh = [torch.where(real, torch.where(cut, 0.0, dt[k]), dh[k]) for k in range(width - 1)]
    out += [torch.stack(dx, 1), dw, db, torch.stack(dh, 1)]
    return tuple(out)


def _exact_scan(s, train):
    """The recurrence and its adjoint, one token after the other."""
    f = {k: s[k].double() for k in ("x", "z", "dt", "A", "B", "C", "D", "dt_bias", "start")}
    b, t, d = f["x"].shape
    g = f["B"].shape[2]
    dev = s["x"].device
    n = torch.full((b,), t, device=dev) if s["len"] is None else s["len"].long()
    h = f["start"]
    outs, keep, ys = [], [], []
    wide = lambda m: m.repeat_interleave(d // g, 1)  # noqa: E731
    for i in range(t):
        real = (i < n)[:, None]
        cut = torch.zeros_like(real) if s["reset_at"] is None else s["reset_at"][:, i:i + 1] & real
        v = f["dt"][:, i] + f["dt_bias"]
        delta = torch.logaddexp(v, torch.zeros_like(v))
        past = torch.where(cut[..., None], 0.0, h)
        if train:
            keep.append(past)
        new = torch.exp(delta[..., None] * f["A"]) * past + (delta * f["x"][:, i])[..., None] * wide(f["B"][:, i])
        h = torch.where(real[..., None], new, h)
        y = (h * wide(f["C"][:, i])).sum(-1) + f["D"] * f["x"][:, i]
        ys.append(y)
        z = f["z"][:, i]
        outs.append(torch.where(real, y * z / (1 + torch.exp(-z)), 0.0))
    out = {"out": torch.stack(outs, 1), "final": h}
    if not train:
        return out
    dh = s["dfinal"].double()
    dout = s["dout"].double()
    r = {k: [None] * t for k in ("dx", "ddt", "dz", "dB", "dC")}
    dA, dD, dbias = torch.zeros_like(f["A"]), torch.zeros_like(f["D"]), torch.zeros_like(f["D"])
    for i in range(t - 1, -1, -1):
        real = (i < n)[:, None]
        on = real[..., None]
        cut = torch.zeros_like(real) if s["reset_at"] is None else s["reset_at"][:, i:i + 1] & real
        zero = lambda m, c=real: torch.where(c, m, 0.0)  # noqa: E731
        x, z, v = zero(f["x"][:, i]), zero(f["z"][:, i]), zero(f["dt"][:, i] + f["dt_bias"])
        Bt, Ct = wide(zero(f["B"][:, i], on)), wide(zero(f["C"][:, i], on))
        delta = torch.logaddexp(v, torch.zeros_like(v))
        dec = torch.exp(delta[..., None] * f["A"])
        past = keep[i]
        now = dec * past + (delta * x)[..., None] * Bt
        sz = 1 / (1 + torch.exp(-z))
        do = zero(dout[:, i])
        r["dz"][i] = do * zero(ys[i]) * (sz + z * sz * (1 - sz))
        gy = do * z * sz
        dn = torch.where(on, dh + gy[..., None] * Ct, 0.0)
        r["dC"][i] = (gy[..., None] * torch.where(on, now, 0.0)).view(b, g, d // g, -1).sum(2)
        r["dB"][i] = (dn * (delta * x)[..., None]).view(b, g, d // g, -1).sum(2)
        ub, q = (dn * Bt).sum(-1), dn * dec * past
        r["dx"][i] = ub * delta + gy * f["D"]
        r["ddt"][i] = ((q * f["A"]).sum(-1) + ub * x) / (1 + torch.exp(-v))
        dA += (q * delta[..., None]).sum(0)
        dD += (gy * x).sum(0)
        dbias += r["ddt"][i].sum(0)
        dh = torch.where(on, torch.where(cut[..., None], 0.0, dn * dec), dh)
    out.update({k: torch.stack(v, 1) for k, v in r.items()}, dA=dA, dD=dD, ddt_bias=dbias, dstate=dh)
    return out


def _exact_step(s):
    on = torch.ones(s["x"].shape[0], dtype=torch.bool, device=s["x"].device) if s["slots"] is None else s["slots"] >= 0
    at = torch.arange(s["x"].shape[0], device=s["x"].device) if s["slots"] is None else s["slots"].long()
    pool = s["state_rows"].double().clone()
    x = s["x"].double()[on]
    old = pool[at[on]]
    if s["reset_rows"] is not None:
        old = old * (~s["reset_rows"][on]).double()[:, None, None]
    if s["op"] == "conv_step":
        taps = torch.cat([old, x[:, None]], 1)
        pre = torch.einsum("rkd,dk->rd", taps, s["weight"].double()) + s["bias"].double()
        y, new = pre / (1 + torch.exp(-pre)), taps[:, 1:]
    else:
        z, v = s["z"].double()[on], s["dt"].double()[on] + s["dt_bias"].double()
        delta = torch.logaddexp(v, torch.zeros_like(v))
        rep = x.shape[1] // s["B"].shape[1]
        B, C = (s[k].double()[on].repeat_interleave(rep, 1) for k in ("B", "C"))
        new = torch.exp(delta[..., None] * s["A"].double()) * old + (delta * x)[..., None] * B
        y = (torch.einsum("rdn,rdn->rd", new, C) + s["D"].double() * x) * z / (1 + torch.exp(-z))
    pool[at[on]] = new
    out = torch.zeros(s["x"].shape, dtype=torch.float64, device=x.device)
    out[on] = y
    return out, pool


def _exact_sample(s):
    sizes = HEADS if s["heads"] else (s["vocab"],)
    tokens, logps = [], []
    for k, z in enumerate(s["logits"].double().split(sizes, 1)):
        r, v = z.shape
        inv = 1.0 / torch.tensor(s["temperature"], dtype=torch.float32, device=z.device).double()
        order = torch.argsort(z, dim=1, descending=True, stable=True)
        zs = z.gather(1, order)
        p = torch.exp((zs - zs[:, :1]) * inv)
        p[p < torch.tensor(s["min_p"], dtype=torch.float32).double().item()] = 0
        if s["top_k"]:
            p[:, s["top_k"]:] = 0
        if s["top_p"] < 1:
            share = torch.tensor(s["top_p"], dtype=torch.float32).double().item()
            p[(p.cumsum(1) - p) >= share * p.sum(1, keepdim=True)] = 0
        q = torch.zeros_like(p).scatter(1, order, p)
        c = q.cumsum(1)
        i = (c <= s["u"][:, k:k + 1].double() * c[:, -1:]).sum(1, keepdim=True).clamp(max=v - 1)
        tokens.append(i.int())
        logps.append(torch.log(q.gather(1, i) / c[:, -1:]))
    return torch.cat(tokens, 1), torch.cat(logps, 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        return _exact_sample(s)
    if op in ("conv_step", "scan_step"):
        return _exact_step(s)
    if op in ("conv", "conv_train"):
        return _exact_conv(s, op == "conv_train")
    return _exact_scan(s, op == "scan_train")
