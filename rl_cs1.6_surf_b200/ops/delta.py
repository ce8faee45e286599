"""The gated delta rule (csrc/kernels/delta.cu, delta_grad.cu) and its PyTorch oracle.

A memory S [values, keys] per sequence and value head that is written by correction:

    S <- e^g S,  S <- S + beta (v - S k) k^T,  o = scale S q

with g = A softplus(dt + dt_bias) and beta = sigmoid(b). ``gated_delta`` runs whole
sequences [B, T, ...], ``gated_delta_grad`` is its gradient, ``gated_delta_step`` runs single
tokens of many envs (one state per slot of a pool, moved on in place).

q and k [.., G, K], v [.., H, V], dt and b [.., H]: G groups of H / G value heads share keys and
queries; K and V are 1 to 128. Tokens are bfloat16 or float32, the weights A (<= 0) and
dt_bias [H] and the states [.., H, V, K] float32. With ``normalize`` keys and queries are
divided by their lengths, sqrt(|k|^2 + 1e-6); ``scale`` None: 1 / sqrt(K).

``reset`` and ``lengths``, strides and gradients are as of ``ops.ssm``: a reset empties the
state before its token (infinities and NaN end with their episode too), tokens past a row's
length give zeros, change nothing and are never read; nothing here records a graph for autograd.
NaN in a token, gate or weight is NaN in all that is made of it, and may reach up to 15 tokens
before it in its episode too: rows are taken 16 tokens at a time, later ones with a factor of 0.
"""
from __future__ import annotations

import struct
from collections import namedtuple
from ctypes import c_char_p
from typing import Optional

import torch

from . import _lib
from ._lib import launch
from .gemm import error_flag
from .ssm import _bits, _dense, _dtype_code, _flags, _like, _p, _real, _tokens

DLIB = "libsurf_delta.so"
_V, _I = _lib._V, _lib._I
_lib.register(DLIB, {
    "surf_delta": (_I, [c_char_p, _I, _V]),
    "surf_delta_grad": (_I, [c_char_p, _I, _V]),
    "surf_delta_step": (_I, [c_char_p, _I, _V]),
})

MAX_HEAD, TILE, NORM_EPS = 128, 16, 1e-6
_VALUES = 64                                    # of a block of the gradient

Delta = namedtuple("Delta", "out final saved")
DeltaGrads = namedtuple("DeltaGrads", "dq dk dv ddt db dA ddt_bias dstate")

_ARGS = struct.Struct("46qf9i")
_STEP = struct.Struct("22qf7i")


def _heads(what, q, v):
    """(groups, heads, keys, values) of q [.., G, K] and v [.., H, V]."""
    g, k = q.shape[-2:]
    h, n = v.shape[-2:]
    if g < 1 or h < 1 or h % g:
        raise ValueError(f"{what}: the key heads must divide the value heads, {g} and {h}")
    if not 1 <= k <= MAX_HEAD or not 1 <= n <= MAX_HEAD:
        raise ValueError(f"{what}: heads of 1 to {MAX_HEAD} keys and values, not {k} and {n}")
    return g, h, k, n


def _check(what, q, k, v, dt, b, A, dt_bias, state, reset, lengths):
    _lib.require_cuda(q, what)
    if q.dim() != 4 or v.dim() != 4:
        raise ValueError(f"{what}: q must be [batch, tokens, groups, keys], v [batch, tokens, heads, values]")
    code = _dtype_code(q, what)
    g, h, nk, nv = _heads(what, q, v)
    bsz, t = q.shape[:2]
    at, dtype, f32 = q.get_device(), q.dtype, torch.float32
    _tokens(what, "q", q, (bsz, t, g, nk), dtype, at)
    _tokens(what, "k", k, (bsz, t, g, nk), dtype, at)
    _tokens(what, "v", v, (bsz, t, h, nv), dtype, at)
    _tokens(what, "dt", dt, (bsz, t, h), dtype, at)
    _tokens(what, "b", b, (bsz, t, h), dtype, at)
    _dense(what, "A", A, (h,), f32, at)
    _dense(what, "dt_bias", dt_bias, (h,), f32, at)
    _dense(what, "state", state, (bsz, h, nv, nk), f32, at)
    _flags(what, reset, (bsz, t), at)
    _dense(what, "lengths", lengths, (bsz,), torch.int32, at)
    if bsz * h > 2 ** 31 - 1:
        raise ValueError(f"{what}: at most 2^31 - 1 heads of sequences")
    return code, 4 - 2 * code, at, bsz, t, g, h, nk, nv


def _scale(what: str, scale: Optional[float], keys: int) -> float:
    scale = keys ** -0.5 if scale is None else float(scale)
    if not _lib.within_float32(scale):
        raise ValueError(f"{what}: scale must be finite in float32")
    return scale


def _piece(bits: int) -> int:
    return 16 if bits & 15 == 0 else 0


def _strides(*tensors) -> list:
    return [s for t in tensors for s in (t.stride()[:-1] if t is not None else (0, 0, 0))]


def gated_delta(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, dt: torch.Tensor, b: torch.Tensor, A: torch.Tensor, *,
                dt_bias: Optional[torch.Tensor] = None, scale: Optional[float] = None, normalize: bool = True,
                state: Optional[torch.Tensor] = None, reset: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, train: bool = False, out: Optional[torch.Tensor] = None) -> Delta:
    """The rule over whole rows: ``out`` [B, T, H, V] and ``final`` [B, H, V, K]. ``train`` keeps in
    ``saved`` what ``gated_delta_grad`` starts from, the states before and the corrections of every 16
    tokens: 4 H V (K + 16) bytes. ``out`` must
    not share memory with an input."""
    what = "gated_delta"
    code, e, at, bsz, t, g, h, nk, nv = _check(what, q, k, v, dt, b, A, dt_bias, state, reset, lengths)
    if out is None:
        out = _like(v)
    else:
        _tokens(what, "out", out, v.shape, v.dtype, at)
        _lib.require_apart(what, "out", out, dict(q=q, k=k, v=v, dt=dt, b=b, A=A, dt_bias=dt_bias, state=state, reset=reset,
                                                  lengths=lengths))
    final = A.new_empty((bsz, h, nv, nk))
    saved = A.new_empty((bsz, -(-t // TILE), h, nv, nk + TILE)) if train else None
    if bsz == 0:
        return Delta(out, final, saved)
    args = _ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), dt.data_ptr(), b.data_ptr(), A.data_ptr(), _p(dt_bias), _p(state),
                      _p(reset), _p(lengths), out.data_ptr(), final.data_ptr(), _p(saved), *(0,) * 14,
                      *_strides(q, k, v), *dt.stride()[:2], *b.stride()[:2], *_strides(out), 0, 0, 0,
                      _scale(what, scale, nk), bsz, t, g, h, nk, nv, normalize,
                      _piece(_bits(e, q, k) | nk * e), _piece(_bits(e, v, out) | nv * e))
    launch(_lib.lib(DLIB).surf_delta, "surf_delta", at, args, code)
    return Delta(out, final, saved)


def gated_delta_grad(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, dt: torch.Tensor, b: torch.Tensor,
                     A: torch.Tensor, *, saved: torch.Tensor, dt_bias: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None, normalize: bool = True, state: Optional[torch.Tensor] = None,
                     reset: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                     dfinal: Optional[torch.Tensor] = None) -> DeltaGrads:
    """Gradients of ``gated_delta`` for the gradient ``dout`` of out and ``dfinal`` of final (None:
    zero). The tokens' gradients come in the tokens' type (summed in 32 bits first where value heads
    share a key head), the weights' and the state's in float32; None for an input that was None."""
    what = "gated_delta_grad"
    code, e, at, bsz, t, g, h, nk, nv = _check(what, q, k, v, dt, b, A, dt_bias, state, reset, lengths)
    f32 = torch.float32
    _tokens(what, "dout", dout, v.shape, v.dtype, at)
    _dense(what, "dfinal", dfinal, (bsz, h, nv, nk), f32, at)
    if saved is None:
        raise ValueError(f"{what}: needs the states that gated_delta(train=True) saved")
    _dense(what, "saved", saved, (bsz, -(-t // TILE), h, nv, nk + TILE), f32, at)
    if saved.data_ptr() & 15:
        raise ValueError(f"{what}: saved must start on a 16-byte boundary")
    dq, dk, dv, ddt, db = (_like(x) for x in (q, k, v, dt, b))
    dA, dbias, dstate = torch.empty_like(A), None if dt_bias is None else torch.empty_like(dt_bias), \
        None if state is None else torch.empty_like(state)
    if bsz == 0:
        return DeltaGrads(dq, dk, dv, ddt, db, dA.zero_(), None if dbias is None else dbias.zero_(), dstate)
    splits = -(-nv // _VALUES)
    n = bsz * t * h * splits * nk if g != h * splits else 0         # parts that a second kernel sums
    m = bsz * t * h * splits * 2 if splits > 1 else 0
    ws = A.new_empty(2 * n + m + 2 * bsz * h * splits)
    base = ws.data_ptr()
    args = _ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), dt.data_ptr(), b.data_ptr(), A.data_ptr(), _p(dt_bias), _p(state),
                      _p(reset), _p(lengths), 0, 0, saved.data_ptr(), dout.data_ptr(), _p(dfinal), dq.data_ptr(), dk.data_ptr(),
                      dv.data_ptr(), ddt.data_ptr(), db.data_ptr(), _p(dstate), base if n else 0,
                      base + 4 * n if n else 0, base + 8 * n if m else 0, base + 8 * n + 4 * m, dA.data_ptr(), _p(dbias),
                      *_strides(q, k, v), *dt.stride()[:2], *b.stride()[:2], 0, 0, 0, *_strides(dout),
                      _scale(what, scale, nk), bsz, t, g, h, nk, nv, normalize,
                      _piece(_bits(e, q, k) | nk * e), _piece(_bits(e, dout) | nv * e))
    launch(_lib.lib(DLIB).surf_delta_grad, "surf_delta_grad", at, args, code)
    del ws                                     # the stream's next user comes after the launch
    _lib.add_launches(2 if n else 1)
    return DeltaGrads(dq, dk, dv, ddt, db, dA, dbias, dstate)


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, dt: torch.Tensor, b: torch.Tensor, A: torch.Tensor,
                     state: torch.Tensor, *, dt_bias: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     normalize: bool = True, reset: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token for each of R envs: q, k [R, G, K], v [R, H, V], dt, b [R, H] -> out [R, H, V].
    ``state`` [S, H, V, K] is the pool of states, ``slots`` [R] (int32) each row's place in it
    (None: row r is slot r; below 0: no env, its output is zero), moved on in place. No two rows
    may name one slot. A slot past the pool gives zeros and is reported through
    ``ops.gemm.check_error_flag``. ``out`` must not share memory with an input."""
    what = "gated_delta_step"
    _lib.require_cuda(q, what)
    if q.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{what}: q must be [rows, groups, keys], v [rows, heads, values]")
    code = _dtype_code(q, what)
    g, h, nk, nv = _heads(what, q, v)
    r, at, dtype, f32 = q.shape[0], q.get_device(), q.dtype, torch.float32
    _tokens(what, "q", q, (r, g, nk), dtype, at)
    _tokens(what, "k", k, (r, g, nk), dtype, at)
    _tokens(what, "v", v, (r, h, nv), dtype, at)
    _tokens(what, "dt", dt, (r, h), dtype, at)
    _tokens(what, "b", b, (r, h), dtype, at)
    _dense(what, "A", A, (h,), f32, at)
    _dense(what, "dt_bias", dt_bias, (h,), f32, at)
    _dense(what, "state", state, (state.shape[0], h, nv, nk), f32, at)
    _flags(what, reset, (r,), at)
    _dense(what, "slots", slots, (r,), torch.int32, at)
    if slots is None and state.shape[0] < r:
        raise ValueError(f"{what}: {r} rows, but {state.shape[0]} slots")
    if state.data_ptr() & 15:
        raise ValueError(f"{what}: the state pool must start on a 16-byte boundary")
    if out is None:
        out = _like(v)
    else:
        _tokens(what, "out", out, v.shape, dtype, at)
        _lib.require_apart(what, "out", out, dict(q=q, k=k, v=v, dt=dt, b=b, A=A, dt_bias=dt_bias, state=state, reset=reset,
                                                  slots=slots))
    if r == 0:
        return out
    args = _STEP.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), dt.data_ptr(), b.data_ptr(), A.data_ptr(), _p(dt_bias),
                      state.data_ptr(), _p(reset), _p(slots), out.data_ptr(), error_flag(q.device).data_ptr(), *q.stride()[:2],
                      *k.stride()[:2], *v.stride()[:2], dt.stride(0), b.stride(0), *out.stride()[:2],
                      _scale(what, scale, nk), r, g, h, nk, nv, normalize, state.shape[0])
    launch(_lib.lib(DLIB).surf_delta_step, "surf_delta_step", at, args, code)
    return out


# ---- oracle -------------------------------------------------------------------------
def gated_delta_reference(q, k, v, dt, b, A, *, dt_bias=None, scale=None, normalize=True, state=None, reset=None, lengths=None):
    """``gated_delta`` token by token, in the type of its inputs (differentiable): (out, final)."""
    bsz, t, g, nk = q.shape
    h = v.shape[2]
    real = _real(lengths, bsz, t, q.device)
    S = q.new_zeros(bsz, h, v.shape[3], nk) if state is None else state
    scale = nk ** -0.5 if scale is None else scale

    def unit(x):
        x = x.repeat_interleave(h // g, 1)
        return x / torch.sqrt((x * x).sum(-1, keepdim=True) + NORM_EPS) if normalize else x

    outs = []
    for i in range(t):
        on = real[:, i, None]
        here = lambda x: torch.where(on.view(bsz, *[1] * (x.dim() - 1)), x, torch.zeros_like(x))  # noqa: E731
        qi, ki, vi = unit(here(q[:, i])), unit(here(k[:, i])), here(v[:, i])
        pre = here(dt[:, i]) + (dt_bias if dt_bias is not None else 0.0)
        past = S
        if reset is not None:
            cut = (reset[:, i].bool() & real[:, i])[:, None, None, None]
            past = torch.where(cut, torch.zeros_like(S), S)
        low = torch.exp(A * torch.nn.functional.softplus(pre))[..., None, None] * past
        u = torch.sigmoid(here(b[:, i]))[..., None] * (vi - (low * ki[:, :, None]).sum(-1))
        new = low + u[..., None] * ki[:, :, None]
        S = torch.where(on[..., None, None], new, S)
        outs.append(here(scale * (new * qi[:, :, None]).sum(-1)))
    return (torch.stack(outs, 1) if outs else v.new_zeros(v.shape)), S
