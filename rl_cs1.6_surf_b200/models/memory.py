"""A memory core: a policy network whose state lives as long as an episode.

Frame stacking shows a policy a handful of earlier decisions; this core carries a
state through all of them. One block, features -> answers:

    xz = W_in f                    two streams of `dim` channels
    c  = causal_conv(x)            short convolution + SiLU
    (r, B, C) = W_x c              step rank, input and output maps of the state
    o  = selective_scan(c, W_dt r, A, B, C, gate z)
    logits = W_out o + b

with ``ops.gemm`` for the projections and ``ops.ssm`` for the rest. With ``core="delta"`` the
memory is a matrix per head that is written by correction (``ops.delta``):

    c  = causal_conv(W_in f)       queries, keys and values of the heads, side by side
    (dt, b) = W_g f                decay and writing strength of each head
    o  = gated_delta(c, dt, b, A)
    logits = W_out group_norm(o, heads, SiLU) + b

Three ways to run it: ``forward_sequence`` / ``backward`` over rows of decisions [envs, T] with episode
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

from ..ops import delta, norm, ssm


@dataclass
class MemoryConfig:
    features: int = 16          # input columns (a multiple of 8)
    dim: int = 256              # channels of the core (a multiple of 8)
    state: int = 16             # states of a channel
    width: int = 4              # taps of the convolution
    rank: int = 16              # of the step projection (a multiple of 8)
    answers: int = 8            # categories of the answer
    out_pad: int = 64           # columns of the output (>= answers)
    core: str = "scan"          # or "delta"
    heads: int = 4              # of the delta core (a multiple of 4); dim / heads values each
    keys: int = 32              # of a head of the delta core (a multiple of 8)

    @property
    def conv_dim(self) -> int:
        """Channels of the convolution: the core's, or the heads' queries, keys and values."""
        return self.dim if self.core == "scan" else 2 * self.heads * self.keys + self.dim

    def heads_of(self, c: torch.Tensor):
        """(queries, keys, values) of the delta core's convolution, by heads."""
        h, hk = self.heads, self.heads * self.keys
        return (c[..., :hk].unflatten(-1, (h, self.keys)), c[..., hk:2 * hk].unflatten(-1, (h, self.keys)),
                c[..., 2 * hk:].unflatten(-1, (h, self.dim // h)))


class MemoryState:
    """Convolution windows [S, W-1, channels] and the core's states (scan [S, D, N], delta rule
    [S, H, values, keys]) of S envs."""

    def __init__(self, net: "MemoryNet", envs: int):
        c = net.cfg
        dt = torch.bfloat16 if net.device.type == "cuda" else torch.float32
        self.conv = torch.zeros(envs, c.width - 1, c.conv_dim, dtype=dt, device=net.device)
        core = (c.dim, c.state) if c.core == "scan" else (c.heads, c.dim // c.heads, c.keys)
        self.scan = torch.zeros(envs, *core, device=net.device)


class MemoryNet:
    """Flat-parameter memory core; see the module docstring."""

    def __init__(self, cfg: MemoryConfig, device="cpu", seed: int = 0):
        self.cfg, self.device = cfg, torch.device(device)
        c = cfg
        if c.features % 8 or c.dim % 8 or c.rank % 8 or c.state % 4 or c.answers > c.out_pad:
            raise ValueError("features, dim and rank must be multiples of 8, state of 4, answers at most out_pad")
        if c.core not in ("scan", "delta"):
            raise ValueError(f"core must be scan or delta, not {c.core!r}")
        if c.core == "delta" and (c.heads < 4 or c.heads % 4 or c.dim % c.heads or not 0 < c.dim // c.heads <= delta.MAX_HEAD or
                                  c.keys % 8 or not 0 < c.keys <= delta.MAX_HEAD):
            raise ValueError(f"heads must be a positive multiple of 4 that divides dim, with 1 to {delta.MAX_HEAD} values and "
                             f"8 to {delta.MAX_HEAD} keys, a multiple of 8")
        self.specs = [("in.w", (c.conv_dim, c.features)), ("gate.w", (2 * c.heads, c.features)), ("out.w", (c.out_pad, c.dim)),
                      ("conv.w", (c.conv_dim, c.width)), ("conv.b", (c.conv_dim,)), ("dt.b", (c.heads,)), ("a_log", (c.heads,)),
                      ("norm.w", (c.dim,)), ("norm.b", (c.dim,)), ("out.b", (c.out_pad,))] if c.core == "delta" else \
                     [("in.w", (2 * c.dim, c.features)), ("x.w", (c.rank + 2 * c.state, c.dim)), ("dt.w", (c.dim, c.rank)),
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
        for name in ("in.w", "x.w", "dt.w", "out.w", "conv.w") if c.core == "scan" else ("in.w", "gate.w", "out.w", "conv.w"):
            shape = self.offsets[name][1]
            w = (torch.rand(shape, generator=gen) * 2 - 1) / math.sqrt(shape[1])
            if name == "out.w":
                w[c.answers:] = 0.0
            self.p(name).copy_(w)
        step = torch.exp(torch.rand(self.p("dt.b").shape, generator=gen) * math.log(100.0) + math.log(0.001))
        self.p("dt.b").copy_(torch.log(torch.expm1(step)))
        if c.core == "delta":
            self.p("norm.w").fill_(1.0)             # and decays exp(-step), a_log = 0
            self.sync_bf16()
            return
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
        if c.core == "delta":
            qkv, conv = ssm.causal_conv_reference(x.float() @ P["in.w"].t(), P["conv.w"], P["conv.b"], state=state.conv.float(),
                                                  reset=reset)
            gates = x.float() @ P["gate.w"].t()
            o, scan = delta.gated_delta_reference(*c.heads_of(qkv), gates[..., :c.heads], gates[..., c.heads:], -torch.exp(P["a_log"]),
                                                  dt_bias=P["dt.b"], state=state.scan, reset=reset)
            o = norm.group_norm_reference(o.reshape(B * T, c.dim), c.heads, P["norm.w"], P["norm.b"], activation="silu")
            return o.view(B, T, c.dim) @ P["out.w"].t() + P["out.b"], conv, scan
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
    __slots__ = ("x", "xz", "xc", "proj", "dt", "out", "saved", "conv0", "scan0", "reset", "A", "core", "stats")


def forward_sequence(net: MemoryNet, x: torch.Tensor, state: MemoryState, reset: Optional[torch.Tensor], train: bool = True):
    """(logits [B, T, out_pad] fp32, cache): x [B, T, features] bf16, a decision of env b in
    row b; ``state`` is carried on to the rows' ends (row b is slot b)."""
    from ..ops import gemm as G
    c, k = net.cfg, SequenceCache()
    B, T, _ = x.shape
    k.x, k.reset, k.conv0, k.scan0 = x.reshape(B * T, c.features), reset, state.conv, state.scan
    if c.core == "delta":
        return _forward_delta(net, k, state, B, T, train), k
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


def _forward_delta(net: MemoryNet, k: SequenceCache, state: MemoryState, B: int, T: int, train: bool) -> torch.Tensor:
    from ..ops import gemm as G
    c = net.cfg
    k.xz = G.gemm(k.x, net.w16("in.w")).view(B, T, c.conv_dim)
    k.xc, state.conv = ssm.causal_conv(k.xz, net.p("conv.w"), net.p("conv.b"), state=k.conv0, reset=k.reset)
    k.dt = G.gemm(k.x, net.w16("gate.w")).view(B, T, 2 * c.heads)
    k.A = -torch.exp(net.p("a_log"))
    r = delta.gated_delta(*c.heads_of(k.xc), k.dt[..., :c.heads], k.dt[..., c.heads:], k.A, dt_bias=net.p("dt.b"), state=k.scan0,
                          reset=k.reset, train=train)
    k.core, k.saved, state.scan = r.out.view(B * T, c.dim), r.saved, r.final
    n = norm.group_norm(k.core, c.heads, net.p("norm.w"), net.p("norm.b"), activation="silu", train=train)
    k.out, k.stats = n.out, n.stats
    return G.gemm(k.out, net.w16("out.w"), out_dtype=torch.float32, bias=net.p("out.b")).view(B, T, c.out_pad)


def _backward_delta(net: MemoryNet, k: SequenceCache, dout: torch.Tensor, B: int, T: int) -> torch.Tensor:
    """The gradient of the convolution's output, for the gradient ``dout`` [B T, dim] of the normalised heads."""
    from .policy import _wgrad
    from ..ops import gemm as G
    c = net.cfg
    n = norm.group_norm_grad(dout, k.core, c.heads, net.p("norm.w"), net.p("norm.b"), stats=k.stats, activation="silu")
    net.g("norm.w").add_(n.dweight)
    net.g("norm.b").add_(n.dbias)
    d = delta.gated_delta_grad(n.dx.view(B, T, c.heads, c.dim // c.heads), *c.heads_of(k.xc), k.dt[..., :c.heads], k.dt[..., c.heads:], k.A,
                               saved=k.saved, dt_bias=net.p("dt.b"), state=k.scan0, reset=k.reset)
    net.g("a_log").add_(d.dA * k.A)
    net.g("dt.b").add_(d.ddt_bias)
    _wgrad(G, torch.cat([d.ddt, d.db], -1).view(B * T, 2 * c.heads), k.x, net.g("gate.w"), B * T)
    return torch.cat([v.flatten(2) for v in (d.dq, d.dk, d.dv)], -1)


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
    if c.core == "delta":
        g = ssm.causal_conv_grad(_backward_delta(net, k, dout.view(n, c.dim), B, T), k.xz, net.p("conv.w"), net.p("conv.b"), state=k.conv0,
                                 reset=k.reset)
        net.g("conv.w").add_(g.dweight)
        net.g("conv.b").add_(g.dbias)
        _wgrad(G, g.dx.view(n, c.conv_dim), k.x, net.g("in.w"), n)
        return
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
    if c.core == "delta":
        xc = ssm.causal_conv_step(xz, net.p("conv.w"), net.p("conv.b"), state.conv, reset=reset, slots=slots)
        gates = G.gemm(x, net.w16("gate.w"))
        out = delta.gated_delta_step(*c.heads_of(xc), gates[:, :c.heads], gates[:, c.heads:], -torch.exp(net.p("a_log")), state.scan,
                                     dt_bias=net.p("dt.b"), reset=reset, slots=slots)
        out = norm.group_norm(out.view(R, c.dim), c.heads, net.p("norm.w"), net.p("norm.b"), activation="silu").out
        return G.gemm(out, net.w16("out.w"), out_dtype=torch.float32, bias=net.p("out.b"))
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


def _answers_gradient(logits, targets, cfg):
    """(cross-entropy of the asked-for answers, its gradient by all of the output's columns)."""
    asked = targets >= 0
    count = asked.sum().clamp(min=1)
    lsm = torch.log_softmax(logits[..., :cfg.answers].float(), -1)
    target = targets.clamp(min=0)[..., None]
    loss = -(lsm.gather(-1, target)[..., 0] * asked).sum() / count
    d = torch.zeros_like(logits)
    d[..., :cfg.answers] = lsm.detach().exp()
    d.scatter_add_(-1, target, torch.full_like(target, -1.0, dtype=d.dtype))
    return loss, d * (asked[..., None] / count)


class _Answered:
    """Answers that the policy gave to a batch of rows, and what they were worth: a drawn answer to every
    question, 1 for a right one, against the batch's mean."""

    def __init__(self, logits, targets, cfg, u, sample):
        z = logits.detach().reshape(-1, logits.shape[-1])[:, :cfg.answers]
        t = targets.reshape(-1)
        token, logp = sample(z, u)
        asked = t >= 0
        self.count = asked.sum().clamp(min=1)
        right = ((token[:, 0] == t) & asked).float()
        self.answers = torch.where(asked, token[:, 0], -1).to(torch.int32)
        self.logp = logp[:, 0].contiguous()
        self.advantages = right - right.sum() / self.count
        self.weights = (asked / self.count).float()
        self.right = right.sum() / self.count

    def options(self):
        """Of ``ops.rl.policy_loss``: the KL term holds the policy to the one that answered."""
        return dict(ref_logp=self.logp, weights=self.weights, clip=0.2, kl_coef=0.02, ent_coef=0.005)


def train_recall(iterations: int = 400, envs: int = 128, length: int = 64, cfg: Optional[MemoryConfig] = None, device="cuda",
                 lr: Optional[float] = None, seed: int = 0, longest: int = 48, act_steps: int = 96, temperature: float = 0.5, top_p: float = 0.9,
                 objective: str = "answers", epochs: int = 2, log=None) -> dict:
    """Train a memory core on the recall task and let it answer, decision by decision, with
    sampled answers: {"loss": first and last, "accuracy": of the sampled answers}. The objective is the
    asked-for answers' cross-entropy ("answers") or what the core's own sampled answers earn ("policy": 1 for a right one,
    ``epochs`` updates of ``ops.rl.policy_loss`` for each batch of rows); ``lr`` None: 1e-2, and 2e-3 for the
    policy, whose KL term grows with e^(its step). An error that
    a kernel reported (a wait that ran out, an index out of range) is raised every 25 iterations
    and at the end."""
    from ..ops import rl as R
    from ..ops.gemm import check_error_flag
    from ..ops.tokens import sample_tokens, sample_tokens_reference
    if objective not in ("answers", "policy"):
        raise ValueError(f"objective must be answers or policy, not {objective!r}")
    if epochs < 1:
        raise ValueError(f"epochs must be positive, not {epochs}")
    dev = torch.device(device)
    net = MemoryNet(cfg or MemoryConfig(), dev, seed)
    c = net.cfg
    opt = R.Adam(net, lr=lr if lr is not None else 1e-2 if objective == "answers" else 2e-3, max_norm=1.0)
    task = RecallTask(envs, c.answers, longest, c.features, seed)
    state = MemoryState(net, envs)
    gpu = dev.type == "cuda"
    draws = torch.Generator().manual_seed(seed)
    sample = sample_tokens if gpu else sample_tokens_reference
    losses = []
    for it in range(iterations):
        x, r, t = (torch.as_tensor(v, device=dev) for v in task.rows(length))
        began, answered = (state.conv, state.scan), None
        for epoch in range(epochs if objective == "policy" else 1):
            state.conv, state.scan = began
            if gpu:
                logits, cache = forward_sequence(net, x.bfloat16(), state, r)
            else:
                params = net.autograd_params()
                logits, conv, scan = net.forward_reference(x, state, r, params)
                state.conv, state.scan = conv.detach(), scan.detach()
            if objective == "answers":
                loss, d = _answers_gradient(logits, t, c)
            else:
                if answered is None:
                    answered = _Answered(logits, t, c, torch.rand(t.numel(), 1, generator=draws).to(dev), sample)
                z = logits.reshape(-1, c.out_pad)[:, :c.answers]
                if gpu:
                    d = torch.zeros_like(logits)
                    loss = R.policy_loss(z, answered.answers, answered.logp, answered.advantages, out=d.view(-1, c.out_pad)[:, :c.answers],
                                         **answered.options()).loss
                else:
                    loss = R.policy_loss_reference(z, answered.answers, answered.logp, answered.advantages, **answered.options())
            if gpu:
                backward(net, cache, d.bfloat16())
            else:
                loss.backward()
                net.collect_grads(params)
            opt.step()
        losses.append(loss.detach())
        if gpu and (it + 1) % 25 == 0:
            check_error_flag(dev)
        if log is not None and (it + 1) % 25 == 0:
            share = "" if answered is None else f", {float(answered.right):.3f} of the answers right"
            log(f"iteration {it + 1}: loss {float(loss):.4f}{share}")
    right = asked_n = 0
    state, task = MemoryState(net, envs), RecallTask(envs, c.answers, longest, c.features, seed + 1)
    gen = torch.Generator().manual_seed(seed)
    for _ in range(act_steps):
        x, r, t = (torch.as_tensor(v, device=dev) for v in task.decision())
        u = torch.rand(envs, 1, generator=gen)
        if gpu:
            answer, _ = act(net, x.bfloat16(), state, u.to(dev), reset=r, temperature=temperature, top_p=top_p)
        else:
            with torch.no_grad():
                logits, state.conv, state.scan = net.forward_reference(x[:, None], state, r[:, None])
            answer = sample_tokens_reference(logits[:, 0, :c.answers], u, temperature=temperature, top_p=top_p)[0][:, 0]
        right += int(((answer == t) & (t >= 0)).sum())
        asked_n += int((t >= 0).sum())
    if gpu:
        check_error_flag(dev)
    return {"loss": [float(losses[0]), float(losses[-1])], "accuracy": right / max(1, asked_n), "questions": asked_n}
