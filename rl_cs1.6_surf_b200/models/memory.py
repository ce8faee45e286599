"""A memory core: a policy network whose state lives as long as an episode.

Frame stacking shows a policy a handful of earlier decisions; this core carries a
state through all of them. One block, features -> answers:

    xz = W_in f                    two streams of `dim` channels
    c  = causal_conv(x)            short convolution + SiLU
    (r, B, C) = W_x c              step rank, input and output maps of the state
    o  = selective_scan(c, W_dt r, A, B, C, gate z)
    logits = W_out o + b

with ``ops.gemm`` for the projections and ``ops.ssm`` for the rest. Three ways to run
it: ``forward_sequence`` / ``backward`` over rows of decisions [envs, T] with episode
resets inside the rows (training, states carried from row to row), ``step`` for one
decision of every env (rollout: one slot of the state pools per env) and ``act``, a
step whose answers are drawn by ``ops.tokens.sample_tokens``. ``forward_reference`` is
the float32 autograd statement (CPU path and the oracle of the kernels' path).

Parameters live in one flat fp32 buffer with a flat gradient and a bf16 shadow, as in
``models.policy``: ``ops.rl.Adam`` works on a ``MemoryNet`` unchanged.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from ..ops import ssm


@dataclass
class MemoryConfig:
    features: int = 16          # input columns (a multiple of 8)
    dim: int = 256              # channels of the core (a multiple of 8)
    state: int = 16             # states of a channel
    width: int = 4              # taps of the convolution
    rank: int = 16              # of the step projection (a multiple of 8)
    answers: int = 8            # categories of the answer
    out_pad: int = 64           # columns of the output (>= answers)


class MemoryState:
    """Convolution windows [S, W-1, D] and scan states [S, D, N] of S envs."""

    def __init__(self, net: "MemoryNet", envs: int):
        c = net.cfg
        dt = torch.bfloat16 if net.device.type == "cuda" else torch.float32
        self.conv = torch.zeros(envs, c.width - 1, c.dim, dtype=dt, device=net.device)
        self.scan = torch.zeros(envs, c.dim, c.state, device=net.device)


class MemoryNet:
    """Flat-parameter memory core; see the module docstring."""

    def __init__(self, cfg: MemoryConfig, device="cpu", seed: int = 0):
        self.cfg, self.device = cfg, torch.device(device)
        c = cfg
        if c.features % 8 or c.dim % 8 or c.rank % 8 or c.state % 4 or c.answers > c.out_pad:
            raise ValueError("features, dim and rank must be multiples of 8, state of 4, answers at most out_pad")
        self.specs = [("in.w", (2 * c.dim, c.features)), ("x.w", (c.rank + 2 * c.state, c.dim)), ("dt.w", (c.dim, c.rank)),
                      ("out.w", (c.out_pad, c.dim)), ("conv.w", (c.dim, c.width)), ("conv.b", (c.dim,)), ("dt.b", (c.dim,)),
                      ("a_log", (c.dim, c.state)), ("skip", (c.dim,)), ("out.b", (c.out_pad,))]
        self.offsets, off = {}, 0
        for name, shape in self.specs:
            self.offsets[name] = (off, shape)
            off += (int(np.prod(shape)) + 63) // 64 * 64           # 256-byte aligned views
        self.numel = off
        self.flat = torch.zeros(off, device=self.device)
        self.grad = torch.zeros(off, device=self.device)
        self.flat16 = torch.zeros(off, dtype=torch.bfloat16, device=self.device) if self.device.type == "cuda" else None
        self._init(seed)

    def view(self, name: str, buf: Optional[torch.Tensor] = None) -> torch.Tensor:
        off, shape = self.offsets[name]
        b = self.flat if buf is None else buf
        return b[off:off + int(np.prod(shape))].view(*shape)

    def p(self, name):
        return self.view(name)

    def g(self, name):
        return self.view(name, self.grad)

    def w16(self, name):
        return self.view(name, self.flat16)

    def _init(self, seed: int) -> None:
        """Uniform +-1/sqrt(fan in) weights; decays exp(-delta n), n = 1 .. N, with steps
        spread over 0.001 .. 0.1, so that a channel remembers 10 to 1000 decisions."""
        c, gen = self.cfg, torch.Generator().manual_seed(seed)
        for name in ("in.w", "x.w", "dt.w", "out.w", "conv.w"):
            shape = self.offsets[name][1]
            w = (torch.rand(shape, generator=gen) * 2 - 1) / math.sqrt(shape[1])
            if name == "out.w":
                w[c.answers:] = 0.0
            self.p(name).copy_(w)
        step = torch.exp(torch.rand(c.dim, generator=gen) * math.log(100.0) + math.log(0.001))
        self.p("dt.b").copy_(torch.log(torch.expm1(step)))
        self.p("a_log").copy_(torch.log(torch.arange(1, c.state + 1).float()).expand(c.dim, -1))
        self.p("skip").fill_(1.0)
        self.sync_bf16()

    def sync_bf16(self) -> None:
        if self.flat16 is not None:
            self.flat16.copy_(self.flat)

    # ---- float32 autograd path --------------------------------------------------------
    def autograd_params(self) -> dict:
        return {name: self.p(name).detach().requires_grad_(True) for name, _ in self.specs}

    def collect_grads(self, params: dict) -> None:
        for name, t in params.items():
            if t.grad is not None:
                self.g(name).add_(t.grad)

    def forward_reference(self, x: torch.Tensor, state: MemoryState, reset: Optional[torch.Tensor],
                          params: Optional[dict] = None):
        """(logits [B, T, out_pad], conv, scan): x [B, T, features]; the states behind the rows."""
        c = self.cfg
        P = params if params is not None else {n: self.p(n) for n, _ in self.specs}
        B, T, _ = x.shape
        xz = x.float() @ P["in.w"].t()
        xc, conv = ssm.causal_conv_reference(xz[..., :c.dim], P["conv.w"], P["conv.b"], state=state.conv.float(), reset=reset)
        proj = xc @ P["x.w"].t()
        r, Bm, Cm = proj.split([c.rank, c.state, c.state], -1)
        out, scan = ssm.selective_scan_reference(xc, r @ P["dt.w"].t(), -torch.exp(P["a_log"]), Bm[:, :, None], Cm[:, :, None],
                                                 D=P["skip"], z=xz[..., c.dim:], dt_bias=P["dt.b"], state=state.scan, reset=reset)
        return out @ P["out.w"].t() + P["out.b"], conv, scan


# ---- kernels' path ----------------------------------------------------------------------
class SequenceCache:
    """What ``backward`` reads of a ``forward_sequence``."""
    __slots__ = ("x", "xz", "xc", "proj", "dt", "out", "saved", "conv0", "scan0", "reset", "A")


def forward_sequence(net: MemoryNet, x: torch.Tensor, state: MemoryState, reset: Optional[torch.Tensor], train: bool = True):
    """(logits [B, T, out_pad] fp32, cache): x [B, T, features] bf16, a decision of env b in
    row b; ``state`` is carried on to the rows' ends (row b is slot b)."""
    from ..ops import gemm as G
    c, k = net.cfg, SequenceCache()
    B, T, _ = x.shape
    k.x, k.reset, k.conv0, k.scan0 = x.reshape(B * T, c.features), reset, state.conv, state.scan
    k.xz = G.gemm(k.x, net.w16("in.w")).view(B, T, 2 * c.dim)
    k.xc, state.conv = ssm.causal_conv(k.xz[..., :c.dim], net.p("conv.w"), net.p("conv.b"), state=k.conv0, reset=reset)
    k.proj = G.gemm(k.xc.view(B * T, c.dim), net.w16("x.w"))
    k.dt = G.gemm(k.proj[:, :c.rank], net.w16("dt.w")).view(B, T, c.dim)
    k.A = -torch.exp(net.p("a_log"))
    r = ssm.selective_scan(k.xc, k.dt, k.A, *_maps(net, k.proj, B, T), D=net.p("skip"), z=k.xz[..., c.dim:],
                           dt_bias=net.p("dt.b"), state=k.scan0, reset=reset, train=train)
    k.out, k.saved, state.scan = r.out, r.saved, r.final
    logits = G.gemm(k.out.view(B * T, c.dim), net.w16("out.w"), out_dtype=torch.float32, bias=net.p("out.b"))
    return logits.view(B, T, c.out_pad), k


def _maps(net, proj, B, T):
    c = net.cfg
    p = proj.view(B, T, 1, c.rank + 2 * c.state)
    return p[..., c.rank:c.rank + c.state], p[..., c.rank + c.state:]


def backward(net: MemoryNet, k: SequenceCache, dlogits: torch.Tensor) -> None:
    """Accumulate the parameters' gradients into net.grad from ``dlogits`` [B, T, out_pad]
    (bf16). The rows' starting states are constants (truncated at the row)."""
    from ..ops import gemm as G
    from .policy import _wgrad
    c = net.cfg
    B, T, _ = dlogits.shape
    n = B * T
    dl = dlogits.reshape(n, c.out_pad)
    _wgrad(G, dl, k.out.view(n, c.dim), net.g("out.w"), n)
    G.colsum(dl, net.g("out.b"))
    dout = G.gemm(dl, net.w16("out.w"), b_mn=True).view(B, T, c.dim)
    s = ssm.selective_scan_grad(dout, k.xc, k.dt, k.A, *_maps(net, k.proj, B, T), saved=k.saved, D=net.p("skip"),
                                z=k.xz[..., c.dim:], dt_bias=net.p("dt.b"), state=k.scan0, reset=k.reset)
    net.g("a_log").add_(s.dA * k.A)
    net.g("skip").add_(s.dD)
    net.g("dt.b").add_(s.ddt_bias)
    ddt = s.ddt.view(n, c.dim)
    dproj = torch.empty_like(k.proj)
    G.gemm(ddt, net.w16("dt.w"), b_mn=True, out=dproj[:, :c.rank])
    dproj[:, c.rank:c.rank + c.state] = s.dB.view(n, c.state)
    dproj[:, c.rank + c.state:] = s.dC.view(n, c.state)
    _wgrad(G, ddt, k.proj[:, :c.rank], net.g("dt.w"), n)
    _wgrad(G, dproj, k.xc.view(n, c.dim), net.g("x.w"), n)
    # the two paths into xc, each rounded to bf16 as its kernel stores it, and their sum once more:
    # 2^-9 each, as of the activations that they belong to
    dxc = s.dx.add_(G.gemm(dproj, net.w16("x.w"), b_mn=True).view(B, T, c.dim))
    g = ssm.causal_conv_grad(dxc, k.xz[..., :c.dim], net.p("conv.w"), net.p("conv.b"), state=k.conv0, reset=k.reset)
    net.g("conv.w").add_(g.dweight)
    net.g("conv.b").add_(g.dbias)
    dxz = torch.cat([g.dx, s.dz], -1).view(n, 2 * c.dim)
    _wgrad(G, dxz, k.x, net.g("in.w"), n)


def step(net: MemoryNet, x: torch.Tensor, state: MemoryState, reset: Optional[torch.Tensor] = None,
         slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits [R, out_pad] (fp32) of one decision of R envs; their slots of ``state`` move on. A
    slot out of range is reported through ``ops.gemm.check_error_flag``, which the caller looks
    at when it synchronises; its row's core output is zero."""
    from ..ops import gemm as G
    c = net.cfg
    R = x.shape[0]
    xz = G.gemm(x, net.w16("in.w"))
    xc = ssm.causal_conv_step(xz[:, :c.dim], net.p("conv.w"), net.p("conv.b"), state.conv, reset=reset, slots=slots)
    proj = G.gemm(xc, net.w16("x.w"))
    dt = G.gemm(proj[:, :c.rank], net.w16("dt.w"))
    Bm, Cm = (m[:, 0] for m in _maps(net, proj, R, 1))
    out = ssm.selective_scan_step(xc, dt, -torch.exp(net.p("a_log")), Bm, Cm, state.scan, D=net.p("skip"), z=xz[:, c.dim:],
                                  dt_bias=net.p("dt.b"), reset=reset, slots=slots)
    return G.gemm(out, net.w16("out.w"), out_dtype=torch.float32, bias=net.p("out.b"))


def act(net: MemoryNet, x: torch.Tensor, state: MemoryState, u: torch.Tensor, reset: Optional[torch.Tensor] = None,
        slots: Optional[torch.Tensor] = None, **rule):
    """(answers int32 [R], log-probabilities [R]) of one decision, drawn with the numbers
    ``u`` [R, 1] under ``rule`` (temperature, top_k, top_p, min_p of ``sample_tokens``); errors
    as of ``step``."""
    from ..ops.tokens import sample_tokens
    logits = step(net, x, state, reset, slots)
    token, logp = sample_tokens(logits[:, :net.cfg.answers], u, **rule)
    return token[:, 0], logp[:, 0]


# ---- the recall task --------------------------------------------------------------------
class RecallTask:
    """Rows of decisions in which memory is all that helps: an episode's first decision shows
    one of ``answers`` symbols, its last asks for it; in between there is noise. Episodes of
    4 to ``longest`` decisions follow one another through the rows."""

    def __init__(self, envs: int, answers: int = 8, longest: int = 48, features: int = 16, seed: int = 0):
        if features < answers + 2:
            raise ValueError("the features hold the symbol, the question and noise")
        self.n, self.answers, self.longest, self.features = envs, answers, longest, features
        self.rng = np.random.default_rng(seed)
        self.left = np.zeros(envs, np.int64)
        self.cue = np.zeros(envs, np.int64)

    def decision(self):
        """(features [N, F] float32, reset [N] bool, asked-for answer [N] int64, -1 where none)."""
        fresh = self.left == 0
        self.left[fresh] = self.rng.integers(4, self.longest + 1, fresh.sum())
        self.cue[fresh] = self.rng.integers(0, self.answers, fresh.sum())
        x = np.zeros((self.n, self.features), np.float32)
        x[:, self.answers + 1:] = self.rng.standard_normal((self.n, self.features - self.answers - 1))
        x[np.flatnonzero(fresh), self.cue[fresh]] = 1.0
        self.left -= 1
        asked = self.left == 0
        x[asked, self.answers] = 1.0
        return x, fresh, np.where(asked, self.cue, -1)

    def rows(self, length: int):
        xs, rs, ts = zip(*(self.decision() for _ in range(length)))
        return np.stack(xs, 1), np.stack(rs, 1), np.stack(ts, 1)


def train_recall(iterations: int = 400, envs: int = 128, length: int = 64, cfg: Optional[MemoryConfig] = None, device="cuda",
                 lr: float = 1e-2, seed: int = 0, longest: int = 48, act_steps: int = 96, temperature: float = 0.5, top_p: float = 0.9,
                 log=None) -> dict:
    """Train a memory core on the recall task and let it answer, decision by decision, with
    sampled answers: {"loss": first and last, "accuracy": of the sampled answers}. An error that
    a kernel reported (a wait that ran out, an index out of range) is raised every 25 iterations
    and at the end."""
    from ..ops.gemm import check_error_flag
    from ..ops.rl import Adam
    dev = torch.device(device)
    net = MemoryNet(cfg or MemoryConfig(), dev, seed)
    c = net.cfg
    opt = Adam(net, lr=lr, max_norm=1.0)
    task = RecallTask(envs, c.answers, longest, c.features, seed)
    state = MemoryState(net, envs)
    gpu = dev.type == "cuda"
    losses = []
    for it in range(iterations):
        x, r, t = (torch.as_tensor(v, device=dev) for v in task.rows(length))
        asked = t >= 0
        count = asked.sum().clamp(min=1)
        if gpu:
            logits, cache = forward_sequence(net, x.bfloat16(), state, r)
        else:
            params = net.autograd_params()
            logits, conv, scan = net.forward_reference(x, state, r, params)
            state.conv, state.scan = conv.detach(), scan.detach()
        lsm = torch.log_softmax(logits[..., :c.answers].float(), -1)
        target = t.clamp(min=0)[..., None]
        loss = -(lsm.gather(-1, target)[..., 0] * asked).sum() / count
        if gpu:
            d = torch.zeros_like(logits)
            d[..., :c.answers] = lsm.exp()
            d.scatter_add_(-1, target, torch.full_like(lsm[..., :1], -1.0))
            backward(net, cache, (d * (asked[..., None] / count)).bfloat16())
        else:
            loss.backward()
            net.collect_grads(params)
        opt.step()
        losses.append(loss.detach())
        if gpu and (it + 1) % 25 == 0:
            check_error_flag(dev)
        if log is not None and (it + 1) % 25 == 0:
            log(f"iteration {it + 1}: loss {float(loss):.4f}")
    right = asked_n = 0
    state, task = MemoryState(net, envs), RecallTask(envs, c.answers, longest, c.features, seed + 1)
    gen = torch.Generator().manual_seed(seed)
    for _ in range(act_steps):
        x, r, t = (torch.as_tensor(v, device=dev) for v in task.decision())
        u = torch.rand(envs, 1, generator=gen)
        if gpu:
            answer, _ = act(net, x.bfloat16(), state, u.to(dev), reset=r, temperature=temperature, top_p=top_p)
        else:
            from ..ops.tokens import sample_tokens_reference
            with torch.no_grad():
                logits, state.conv, state.scan = net.forward_reference(x[:, None], state, r[:, None])
            answer = sample_tokens_reference(logits[:, 0, :c.answers], u, temperature=temperature, top_p=top_p)[0][:, 0]
        right += int(((answer == t) & (t >= 0)).sum())
        asked_n += int((t >= 0).sum())
    if gpu:
        check_error_flag(dev)
    return {"loss": [float(losses[0]), float(losses[-1])], "accuracy": right / max(1, asked_n), "questions": asked_n}
