"""Sequence operators of a policy's memory core (csrc/kernels/seq_conv.cu,
seq_scan.cu, seq_scan_grad.cu) and their PyTorch oracles.

* ``causal_conv`` — short depthwise convolution over the tokens of a row, SiLU
  behind it;
* ``selective_scan`` — the selective state space recurrence
  h <- exp(delta A) h + delta x B, out = (C . h + D x) silu(z);

each over whole sequences [B, T, ...], with its gradient (``*_grad``), and for
single tokens of many envs (``*_step``: one state per slot of a pool, moved on in
place). The weights are float32; tokens and windows are bfloat16 or float32, the
scan's state always float32.

``reset`` [B, T] (bool or uint8) empties window and state before the marked tokens
(episode starts); ``lengths`` [B] (int32) says how many tokens of a row are there:
the others give zeros, change nothing and are never read. ``state`` is what the row
starts from (None: empty), ``final`` what the next call starts from.

None of them records a graph for autograd: gradients come from the ``*_grad`` functions
alone, and an input that requires one gets none.

Inputs may be strided views (slices of a projection) as long as the last axis is
dense; 16-byte aligned rows are copied asynchronously, others element by element.
"""
from __future__ import annotations

import struct
from collections import namedtuple
from ctypes import c_char_p
from typing import Optional

import torch

from . import _lib
from ._lib import KernelError, launch
from .gemm import error_flag

SLIB = "libsurf_seq.so"
_V, _I, _L = _lib._V, _lib._I, _lib._L
_lib.register(SLIB, {
    "surf_seq_conv": (_I, [c_char_p, _I, _I, _I, _I, _V]),
    "surf_seq_conv_grad": (_I, [c_char_p, _I, _I, _I, _I, _V, _V, _V]),
    "surf_seq_conv_step": (_I, [_V, _L, _V, _V, _V, _V, _V, _I, _V, _L, _I, _I, _I, _I, _I, _I, _V, _V]),
    "surf_seq_scan": (_I, [c_char_p, _I, _V]),
    "surf_seq_scan_grad": (_I, [c_char_p, _I, _V]),
    "surf_seq_scan_grad_blocks": (_I, [_I, _I]),
    "surf_seq_scan_threads": (_I, [_I, _I, _I]),
    "surf_seq_scan_step": (_I, [c_char_p, _I, _V]),
})
_lib._KERNELS_PER_CALL["surf_seq_conv_grad"] = 2

MAX_WIDTH, MAX_STATE, SAVE_EVERY = 4, 64, 8

ConvGrads = namedtuple("ConvGrads", "dx dweight dbias dstate")
Scan = namedtuple("Scan", "out final saved")
ScanGrads = namedtuple("ScanGrads", "dx ddt dz dB dC dA dD ddt_bias dstate")

_CONV = struct.Struct("18q6i")
_SCAN = struct.Struct("48q10i")
_STEP = struct.Struct("21q8i")


def _p(t) -> int:
    return t.data_ptr() if t is not None else 0


def _dtype_code(t: torch.Tensor, what: str) -> int:
    if t.dtype == torch.bfloat16:
        return 1
    if t.dtype == torch.float32:
        return 0
    raise TypeError(f"{what}: tokens must be bfloat16 or float32, not {t.dtype}")


def _tokens(what: str, name: str, t: Optional[torch.Tensor], shape: tuple, dtype, index: int) -> None:
    """An input with the tokens' type: shape, type, device and a dense last axis."""
    if t is None or (t.dtype is dtype and t.shape == shape and t.get_device() == index and t.stride(-1) == 1):
        return
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{what}: {name} is {t.dtype}, the tokens are {dtype}")
    if t.get_device() != index:
        raise ValueError(f"{what}: {name} is on {t.device}, the tokens on cuda:{index}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{what}: {name} needs a dense last axis")


def _dense(what: str, name: str, t: Optional[torch.Tensor], shape: tuple, dtype, index: int) -> None:
    """A contiguous input (weights, states, masks)."""
    if t is None or (t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous()):
        return
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{what}: {name} must be {dtype}, not {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{what}: {name} is on {t.device}, the tokens on cuda:{index}")
    raise ValueError(f"{what}: {name} must be contiguous")


def _even(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """``t`` on a 16-byte boundary, where the kernels read their 32-bit operands four at a
    time: itself, unless it is a view that starts elsewhere."""
    return t if t is None or t.data_ptr() & 15 == 0 else t.clone()


def _flags(what: str, t: Optional[torch.Tensor], shape: tuple, index: int) -> None:
    if t is None:
        return
    if t.dtype is not torch.bool and t.dtype is not torch.uint8:
        raise TypeError(f"{what}: reset must be bool or uint8, not {t.dtype}")
    _dense(what, "reset", t, shape, t.dtype, index)


def _bits(size: int, *tensors) -> int:
    """What the bases and the strides of the tensors' rows, in bytes, have in their low bits."""
    bits = 0
    for t in tensors:
        if t is not None:
            bits |= t.data_ptr()
            for s in t.stride()[:-1]:
                bits |= s * size
    return bits


def _piece(bits: int) -> int:
    """Bytes of the pieces that rows may be copied in (copy_rows): 16 or 4 where the row's
    length, every base and every stride, whose low bits these are, is a multiple of it, else 0."""
    return 16 if bits & 15 == 0 else 4 if bits & 3 == 0 else 0


def _like(t: torch.Tensor) -> torch.Tensor:
    """A new dense tensor of ``t``'s shape and type (half the host time of ``torch.empty``,
    of which a training step needs a dozen)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


# ---- causal convolution -----------------------------------------------------------
def _conv_check(what, x, weight, bias, state, reset, lengths):
    _lib.require_cuda(x, what)
    if x.dim() != 3:
        raise ValueError(f"{what}: x must be [batch, tokens, channels]")
    code = _dtype_code(x, what)
    b, t, d = x.shape
    at = x.get_device()
    if weight.dim() != 2 or not 2 <= weight.shape[1] <= MAX_WIDTH:
        raise ValueError(f"{what}: weight must be [channels, width] with a width of 2 to {MAX_WIDTH}")
    w = weight.shape[1]
    _tokens(what, "x", x, x.shape, x.dtype, at)
    _dense(what, "weight", weight, (d, w), torch.float32, at)
    _dense(what, "bias", bias, (d,), torch.float32, at)
    _dense(what, "state", state, (b, w - 1, d), x.dtype, at)
    _flags(what, reset, (b, t), at)
    _dense(what, "lengths", lengths, (b,), torch.int32, at)
    return code, 4 - 2 * code, at, b, t, d, w


def _stretches(b: int, t: int, groups: int):
    """(tokens of a stretch, stretches of a row, rows of blocks) of the convolution for
    ``groups`` threads across a row: the longest stretch (each reads width - 1 tokens of its
    neighbour again) that still gives every SM 256 threads, two blocks on an SM to take them.

    Forward and gradient, bf16, us at 128, 256 and 512 threads: 256 x 128 x 1024 35 + 62,
    31 + 62, 34 + 66; 1 x 16385 x 1024 21 + 43, 18 + 36, 19 + 39. Stretches of at most 64
    tokens take 58 + 124 at 256 x 512 x 512, of 128 56 + 118, of 256 64 + 113."""
    tt = 128
    while tt > 8 and b * -(-t // tt) * groups < 148 * 256:
        tt //= 2
    chunks = max(1, -(-t // tt))
    bx = min(32, 1 << (groups - 1).bit_length())
    return tt, chunks, max(1, min(-(-b * chunks * bx // 256), -(-296 // -(-groups // bx)), 65535))


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                state: Optional[torch.Tensor] = None, reset: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, silu: bool = True, out: Optional[torch.Tensor] = None):
    """(y [B, T, D], final [B, W-1, D]): y[t] = silu(bias + sum_k weight[:, k] x[t - (W-1) + k])
    over the tokens that t sees; ``state`` and ``final`` hold the W - 1 tokens before
    and behind the row, oldest first. ``out`` must not share memory with an input: a token is
    read by the stretches of the W - 1 behind it too."""
    what = "causal_conv"
    code, e, at, b, t, d, w = _conv_check(what, x, weight, bias, state, reset, lengths)
    weight = _even(weight)
    if out is None:
        out = _like(x)
    else:
        _tokens(what, "out", out, x.shape, x.dtype, at)
        _lib.require_apart(what, "out", out, dict(x=x, weight=weight, bias=bias, state=state, reset=reset, lengths=lengths))
    final = x.new_empty((b, w - 1, d))
    if b == 0 or d == 0:
        return out, final
    bits = _bits(e, x, out, state) | d * e
    size = 16 if bits & 15 == 0 else 4 if bits & 3 == 0 else 2
    tt, chunks, rows = _stretches(b, t, d * e // size)
    args = _CONV.pack(_p(x), 0, _p(state), 0, _p(weight), _p(bias), _p(reset), _p(lengths), out.data_ptr(),
                      final.data_ptr(), 0, x.stride(0), x.stride(1), 0, 0, out.stride(0), out.stride(1), t,
                      b, t, d, int(silu), tt, chunks)
    launch(_lib.lib(SLIB).surf_seq_conv, "surf_seq_conv", at, args, code, w, size, rows)
    return out, final


def causal_conv_grad(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                     state: Optional[torch.Tensor] = None, reset: Optional[torch.Tensor] = None,
                     lengths: Optional[torch.Tensor] = None, silu: bool = True,
                     dfinal: Optional[torch.Tensor] = None) -> ConvGrads:
    """Gradients of ``causal_conv`` for the gradient ``dy`` of y and ``dfinal`` of
    final (None: zero): dx and dstate in the tokens' type, dweight and dbias float32."""
    what = "causal_conv_grad"
    code, e, at, b, t, d, w = _conv_check(what, x, weight, bias, state, reset, lengths)
    _tokens(what, "dy", dy, x.shape, x.dtype, at)
    _dense(what, "dfinal", dfinal, (b, w - 1, d), x.dtype, at)
    weight = _even(weight)
    dx = _like(x)
    dstate = torch.empty_like(state) if state is not None else None
    if b == 0 or d == 0:
        return ConvGrads(dx, torch.zeros_like(weight), None if bias is None else torch.zeros_like(bias), dstate)
    dw = torch.empty_like(weight)
    db = torch.empty_like(bias) if bias is not None else None
    bits = _bits(e, x, dy, state, dfinal) | d * e
    size = 8 if bits & 7 == 0 else 4 if bits & 3 == 0 else 2
    tt, chunks, rows = _stretches(b, t, d * e // size)
    part = weight.new_empty((rows, w + 1, d))
    args = _CONV.pack(_p(x), dy.data_ptr(), _p(state), _p(dfinal), _p(weight), _p(bias), _p(reset), _p(lengths),
                      dx.data_ptr(), _p(dstate), part.data_ptr(), x.stride(0), x.stride(1), dy.stride(0), dy.stride(1),
                      t * d, d, t, b, t, d, int(silu), tt, chunks)
    launch(_lib.lib(SLIB).surf_seq_conv_grad, "surf_seq_conv_grad", at, args, code, w, size, rows, _p(dw), _p(db))
    return ConvGrads(dx, dw, db, dstate)


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], state: torch.Tensor, *,
                     reset: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None, silu: bool = True,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token x [R, D] for each of R envs: y [R, D]. ``state`` [S, W-1, D] is the pool
    of windows, ``slots`` [R] (int32) each row's place in it (None: row r is slot r; below
    0: no env, its output is zero), moved on in place. No two rows may name one slot. A slot past
    the pool gives zeros and is reported through ``ops.gemm.check_error_flag``. ``out`` may be x
    itself, and shares no memory with an input otherwise."""
    what = "causal_conv_step"
    _lib.require_cuda(x, what)
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be [rows, channels]")
    code = _dtype_code(x, what)
    r, d = x.shape
    dev, at, e = x.device, x.get_device(), x.element_size()
    if weight.dim() != 2 or not 2 <= weight.shape[1] <= MAX_WIDTH:
        raise ValueError(f"{what}: weight must be [channels, width] with a width of 2 to {MAX_WIDTH}")
    w = weight.shape[1]
    _tokens(what, "x", x, x.shape, x.dtype, at)
    _dense(what, "weight", weight, (d, w), torch.float32, at)
    _dense(what, "bias", bias, (d,), torch.float32, at)
    _dense(what, "state", state, (state.shape[0], w - 1, d), x.dtype, at)
    _flags(what, reset, (r,), at)
    _dense(what, "slots", slots, (r,), torch.int32, at)
    if slots is None and state.shape[0] < r:
        raise ValueError(f"{what}: {r} rows, but {state.shape[0]} slots")
    if out is None:
        out = _like(x)
    else:
        _tokens(what, "out", out, x.shape, x.dtype, at)
        _lib.require_apart(what, "out", out, dict(x=x, weight=weight, bias=bias, state=state, reset=reset, slots=slots), ("x",))
    if r == 0 or d == 0:
        return out
    vec = (_bits(e, x, out, state) | d * e) % (4 * e) == 0
    launch(_lib.lib(SLIB).surf_seq_conv_step, "surf_seq_conv_step", at, x.data_ptr(), x.stride(0), weight.data_ptr(),
           _p(bias), state.data_ptr(), _p(reset), _p(slots), state.shape[0], out.data_ptr(), out.stride(0), r, d, w,
           int(silu), code, int(vec), error_flag(dev).data_ptr())
    return out


# ---- selective scan ---------------------------------------------------------------
def _scan_check(what, x, dt, A, B, C, D, z, dt_bias, state, reset, lengths):
    _lib.require_cuda(x, what)
    if x.dim() != 3:
        raise ValueError(f"{what}: x must be [batch, tokens, channels]")
    code = _dtype_code(x, what)
    b, t, d = x.shape
    at = x.get_device()
    if A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATE:
        raise ValueError(f"{what}: A must be [channels, states] with 1 to {MAX_STATE} states")
    n = A.shape[1]
    if B.dim() != 4 or B.shape[2] < 1 or d % B.shape[2]:
        raise ValueError(f"{what}: B must be [batch, tokens, groups, states], its groups dividing the channels")
    g = B.shape[2]
    dtype, shape = x.dtype, x.shape
    _tokens(what, "x", x, shape, dtype, at)
    _tokens(what, "dt", dt, shape, dtype, at)
    _tokens(what, "z", z, shape, dtype, at)
    _tokens(what, "B", B, (b, t, g, n), dtype, at)
    _tokens(what, "C", C, (b, t, g, n), dtype, at)
    f32 = torch.float32
    _dense(what, "A", A, (d, n), f32, at)
    _dense(what, "D", D, (d,), f32, at)
    _dense(what, "dt_bias", dt_bias, (d,), f32, at)
    _dense(what, "state", state, (b, d, n), f32, at)
    _flags(what, reset, (b, t), at)
    _dense(what, "lengths", lengths, (b,), torch.int32, at)
    return code, 4 - 2 * code, at, b, t, d, n, g


def _chunks(b: int, t: int, d: int, n: int, g: int):
    """(tokens of a chunk, chunks): a row is cut where its channels leave room on the GPU for
    three times as many threads (512 an SM), since the pass that leaves the chunks' ends costs
    nearly half of the scan itself; a chunk has 16 tokens at least. A row below 128 stays whole
    for the sake of calls one by one, where the host has not launched the two kernels more before
    it is done: 5 x 77 x 194 f32 cut and whole 41 + 74 and 28 + 59 us a call. On the device alone,
    as in a graph, it is the other way (20 + 39 and 23 + 52 us). Other lengths on that side were
    not measured; 128 is where a row gives eight chunks.

    Forward and gradient, bf16, 16 states, us whole and cut: 64 x 1024 x 512 in 2 323 + 797 and
    467 + 1045; 48 rows in 3 323 + 795 and 312 + 716; 16 x 512 x 512 in 8 133 + 266 and 69 + 152;
    16 x 128 x 512 in 8 36 + 69 and 28 + 55. Chunks of 64, 32 and 16 tokens at 4 x 512 x 256:
    36 + 55, 24 + 36, 20 + 32. 256 and 1024 threads an SM at 2 x 4096 x 1024: 137 + 261 and
    112 + 257, against 110 + 249."""
    threads = b * _lib.lib(SLIB).surf_seq_scan_threads(d // g, g, n)
    want = min(148 * 512 // threads if threads else 1, -(-t // 16))
    if want >= 3 and t >= 128:
        chunk = -(-t // want)
        chunk = -(-chunk // 16) * 16
        if t > 2 * chunk:
            return chunk, -(-t // chunk)
    return max(16, -(-t // 16) * 16), 1


def _scan_inputs(x, dt, z, B, C):
    """(addresses, strides of rows, what the strides and addresses of x, dt and z, and of B
    and C, have in their low bits, in bytes) of the scan's tokens, in the kernel's order."""
    e = x.element_size()
    px, pdt, pz, pB, pC = x.data_ptr(), dt.data_ptr(), _p(z), B.data_ptr(), C.data_ptr()
    x0, x1, _ = x.stride()
    t0, t1, _ = dt.stride()
    z0, z1, _ = (0, 0, 0) if z is None else z.stride()
    B0, B1, B2, _ = B.stride()
    C0, C1, C2, _ = C.stride()
    return ((px, pdt, pz, pB, pC), (x0, x1, t0, t1, z0, z1, B0, B1, B2, C0, C1, C2),
            px | pdt | pz | (x0 | x1 | t0 | t1 | z0 | z1) * e, pB | pC | (B0 | B1 | B2 | C0 | C1 | C2) * e)


def _workspace(like, *floats):
    """One allocation for pieces of so many 32-bit numbers, by ``like``'s device: (it, the
    pieces' addresses)."""
    at, total = [], 0
    for n in floats:
        at.append(4 * total)
        total += (n + 3) // 4 * 4
    ws = like.new_empty(total)
    base = ws.data_ptr()
    return ws, [base + o for o in at]


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None, softplus: bool = True,
                   state: Optional[torch.Tensor] = None, reset: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None, train: bool = False,
                   out: Optional[torch.Tensor] = None) -> Scan:
    """The recurrence over x, dt, z [B, T, D], B, C [B, T, G, N] (each group of D / G
    channels shares a row of them), A [D, N]: ``out`` [B, T, D] and ``final`` [B, D, N].
    delta = softplus(dt + dt_bias), or the sum itself with ``softplus=False``. ``train``
    keeps in ``saved`` the states that ``selective_scan_grad`` starts from: 4 D N bytes
    for every 8 tokens. ``out`` may be x, dt or z itself, and shares no memory otherwise."""
    what = "selective_scan"
    code, e, at, b, t, d, n, g = _scan_check(what, x, dt, A, B, C, D, z, dt_bias, state, reset, lengths)
    A, state = _even(A), _even(state)
    if out is None:
        out = _like(x)
    else:
        _tokens(what, "out", out, x.shape, x.dtype, at)
        _lib.require_apart(what, "out", out, dict(x=x, dt=dt, z=z, A=A, B=B, C=C, D=D, dt_bias=dt_bias, state=state, reset=reset,
                                                  lengths=lengths), ("x", "dt", "z"))
    final = A.new_empty((b, d, n))
    saved = A.new_empty((b, -(-t // SAVE_EVERY), d, n)) if train else None
    if b == 0 or d == 0:
        return Scan(out, final, saved)
    chunk, chunks = _chunks(b, t, d, n, g)
    ws, (carry, sumd, cut) = _workspace(A, b * chunks * d * n, b * chunks * d, b * chunks) if chunks > 1 else (None, (0, 0, 0))
    where, strides, bits_d, bits_n = _scan_inputs(x, dt, z, B, C)
    o0, o1, _ = out.stride()
    to = out.data_ptr()
    args = _SCAN.pack(
        *where, 0, A.data_ptr(), _p(D), _p(dt_bias), _p(state), 0,
        _p(reset), _p(lengths), to, final.data_ptr(), _p(saved), carry, sumd, cut,
        0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
        *strides, 0, 0, o0, o1, t, b, t, d, n, g, softplus, chunk, chunks,
        _piece(bits_d | to | (o0 | o1 | d // g) * e), _piece(bits_n | n * e))
    launch(_lib.lib(SLIB).surf_seq_scan, "surf_seq_scan", at, args, code)
    del ws                                     # the stream's next user comes after the launch
    if chunks > 1:
        _lib.add_launches(2)
    return Scan(out, final, saved)


def selective_scan_grad(dout: torch.Tensor, x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                        C: torch.Tensor, *, saved: torch.Tensor, D: Optional[torch.Tensor] = None,
                        z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                        softplus: bool = True, state: Optional[torch.Tensor] = None,
                        reset: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                        dfinal: Optional[torch.Tensor] = None) -> ScanGrads:
    """Gradients of ``selective_scan`` for the gradient ``dout`` of out and ``dfinal`` of
    final (None: zero). The tokens' gradients come in the tokens' type (summed in 32 bits
    first where heads share them), the weights' and the state's in float32; None for an
    input that was None."""
    what = "selective_scan_grad"
    code, e, at, b, t, d, n, g = _scan_check(what, x, dt, A, B, C, D, z, dt_bias, state, reset, lengths)
    f32 = torch.float32
    _tokens(what, "dout", dout, x.shape, x.dtype, at)
    _dense(what, "dfinal", dfinal, (b, d, n), f32, at)
    if saved is None:
        raise ValueError(f"{what}: needs the states that selective_scan(train=True) saved")
    _dense(what, "saved", saved, (b, -(-t // SAVE_EVERY), d, n), f32, at)
    A, saved, dfinal = _even(A), _even(saved), _even(dfinal)

    dx, ddt, dz = _like(x), _like(dt), None if z is None else _like(z)
    dB, dC, dA = _like(B), _like(C), torch.empty_like(A)
    dD, dbias, dstate = (None if v is None else torch.empty_like(v) for v in (D, dt_bias, state))
    if b == 0 or d == 0:
        for v in (dA, dD, dbias):
            if v is not None:
                v.zero_()
        return ScanGrads(dx, ddt, dz, dB, dC, dA, dD, dbias, dstate)
    chunk, chunks = _chunks(b, t, d, n, g)
    L = _lib.lib(SLIB)
    split = b * chunks if chunks > 1 else 0
    ws, (part_bc, part_a, part_v, carry, sumd, cut) = _workspace(
        A, L.surf_seq_scan_grad_blocks(d // g, n) * b * t * g * 2 * n, b * chunks * d * n, b * chunks * d * 2,
        split * d * n, split * d, split)
    where, strides, bits_d, bits_n = _scan_inputs(x, dt, z, B, C)
    o0, o1, _ = dout.stride()
    of = dout.data_ptr()
    args = _SCAN.pack(
        *where, of, A.data_ptr(), _p(D), _p(dt_bias),
        _p(state), _p(dfinal), _p(reset), _p(lengths), 0, 0, saved.data_ptr(), carry, sumd, cut,
        dx.data_ptr(), ddt.data_ptr(), _p(dz), dB.data_ptr(), dC.data_ptr(), part_bc, part_a, part_v, dA.data_ptr(), _p(dD), _p(dbias), _p(dstate),
        *strides, o0, o1, 0, 0, t, b, t, d, n, g, softplus, chunk, chunks,
        _piece(bits_d | of | (o0 | o1 | d // g) * e), _piece(bits_n | n * e))
    launch(L.surf_seq_scan_grad, "surf_seq_scan_grad", at, args, code)
    del ws
    _lib.add_launches(3 if chunks > 1 else 1)
    return ScanGrads(dx, ddt, dz, dB, dC, dA, dD, dbias, dstate)


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        state: torch.Tensor, *, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None, softplus: bool = True,
                        reset: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token for each of R envs: x, dt, z [R, D], B, C [R, G, N] -> out [R, D].
    ``state`` [S, D, N] is the pool of states, ``slots`` [R] (int32) each row's place in
    it (None: row r is slot r; below 0: no env, its output is zero), moved on in place.
    No two rows may name one slot. A slot past the pool gives zeros and is reported through
    ``ops.gemm.check_error_flag``. ``out`` may be x, dt or z itself, and shares no memory with an
    input otherwise."""
    what = "selective_scan_step"
    if not x.is_cuda:
        _lib.require_cuda(x, what)
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be [rows, channels]")
    dtype, f32 = x.dtype, torch.float32
    code = _dtype_code(x, what)
    r, d = shape = x.shape
    at = x.get_device()
    if A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATE:
        raise ValueError(f"{what}: A must be [channels, states] with 1 to {MAX_STATE} states")
    n = A.shape[1]
    if B.dim() != 3 or B.shape[1] < 1 or d % B.shape[1]:
        raise ValueError(f"{what}: B must be [rows, groups, states], its groups dividing the channels")
    g = B.shape[1]
    pools = state.shape[0]
    _tokens(what, "x", x, shape, dtype, at)
    _tokens(what, "dt", dt, shape, dtype, at)
    _tokens(what, "z", z, shape, dtype, at)
    _tokens(what, "B", B, (r, g, n), dtype, at)
    _tokens(what, "C", C, (r, g, n), dtype, at)
    _dense(what, "A", A, (d, n), f32, at)
    _dense(what, "D", D, (d,), f32, at)
    _dense(what, "dt_bias", dt_bias, (d,), f32, at)
    _dense(what, "state", state, (pools, d, n), f32, at)
    _flags(what, reset, (r,), at)
    _dense(what, "slots", slots, (r,), torch.int32, at)
    if slots is None and pools < r:
        raise ValueError(f"{what}: {r} rows, but {pools} slots")
    if out is None:
        out = _like(x)
    else:
        _tokens(what, "out", out, shape, dtype, at)
        _lib.require_apart(what, "out", out, dict(x=x, dt=dt, z=z, A=A, B=B, C=C, D=D, dt_bias=dt_bias, state=state, reset=reset,
                                                  slots=slots), ("x", "dt", "z"))
    if r == 0 or d == 0:
        return out
    A = _even(A)
    if state.data_ptr() & 15:
        raise ValueError(f"{what}: the state pool must start on a 16-byte boundary")
    e = 4 - 2 * code
    pB, pC = B.data_ptr(), C.data_ptr()
    B0, B1, _ = B.stride()
    C0, C1, _ = C.stride()
    whole = (pB | pC | (B0 | B1 | C0 | C1 | n) * e) % (4 * e) == 0
    args = _STEP.pack(x.data_ptr(), dt.data_ptr(), _p(z), pB, pC, A.data_ptr(), _p(D), _p(dt_bias), state.data_ptr(),
                      _p(reset), _p(slots), out.data_ptr(), error_flag(x.device).data_ptr(), x.stride(0), dt.stride(0),
                      0 if z is None else z.stride(0), B0, B1, C0, C1, out.stride(0), r, d, n, g, softplus, pools, whole, 0)
    launch(_lib.lib(SLIB).surf_seq_scan_step, "surf_seq_scan_step", at, args, code)
    return out


# ---- oracles ------------------------------------------------------------------------
def _real(lengths, b, t, device):
    if lengths is None:
        return torch.ones(b, t, dtype=torch.bool, device=device)
    return torch.arange(t, device=device)[None, :] < lengths.to(device)[:, None]


def causal_conv_reference(x, weight, bias=None, *, state=None, reset=None, lengths=None, silu=True):
    """``causal_conv`` token by token, in the type of its inputs (differentiable)."""
    b, t, d = x.shape
    w = weight.shape[1]
    real = _real(lengths, b, t, x.device)
    past = [x.new_zeros(b, d) for _ in range(w - 1)] if state is None else [state[:, j] for j in range(w - 1)]
    ys = []
    for i in range(t):
        on = real[:, i:i + 1]
        seen = past
        if reset is not None:
            seen = [torch.where(reset[:, i:i + 1].bool(), torch.zeros_like(h), h) for h in past]
        taps = seen + [torch.where(on, x[:, i], torch.zeros_like(x[:, i]))]
        pre = sum(weight[:, k] * taps[k] for k in range(w))
        if bias is not None:
            pre = pre + bias
        y = pre * torch.sigmoid(pre) if silu else pre
        ys.append(torch.where(on, y, torch.zeros_like(y)))
        past = [torch.where(on, taps[k + 1], past[k]) for k in range(w - 1)]
    return (torch.stack(ys, 1) if ys else x.new_zeros(b, 0, d)), torch.stack(past, 1)


def selective_scan_reference(x, dt, A, B, C, *, D=None, z=None, dt_bias=None, softplus=True, state=None, reset=None,
                             lengths=None):
    """``selective_scan`` token by token, in the type of its inputs (differentiable):
    (out, final)."""
    b, t, d = x.shape
    rep = d // B.shape[2]
    real = _real(lengths, b, t, x.device)
    h = x.new_zeros(b, d, A.shape[1]) if state is None else state
    outs = []
    for i in range(t):
        on = real[:, i:i + 1]
        off = torch.zeros_like(x[:, i])
        xi, v = torch.where(on, x[:, i], off), torch.where(on, dt[:, i], off)
        Bi, Ci = (torch.where(on[..., None], m[:, i], torch.zeros_like(m[:, i])).repeat_interleave(rep, 1) for m in (B, C))
        if dt_bias is not None:
            v = v + dt_bias
        if softplus:
            v = torch.nn.functional.softplus(v)
        past = h if reset is None else torch.where(reset[:, i, None, None].bool(), torch.zeros_like(h), h)
        new = torch.exp(v[..., None] * A) * past + (v * xi)[..., None] * Bi
        h = torch.where(on[..., None], new, h)
        y = (h * Ci).sum(-1)
        if D is not None:
            y = y + D * xi
        if z is not None:
            zi = torch.where(on, z[:, i], off)
            y = y * zi * torch.sigmoid(zi)
        outs.append(torch.where(on, y, torch.zeros_like(y)))
    return (torch.stack(outs, 1) if outs else x.new_zeros(b, 0, d)), h


__all__ = ["causal_conv", "causal_conv_grad", "causal_conv_step", "selective_scan", "selective_scan_grad",
           "selective_scan_step", "causal_conv_reference", "selective_scan_reference", "ConvGrads", "Scan", "ScanGrads",
           "KernelError"]
