"""Group norm with an activation on channels-last tensors (csrc/kernels/group_norm.cu)
and its PyTorch oracle.

``group_norm`` normalises every sample's groups of channels over all positions, scales and
shifts each channel and applies an activation; ``group_norm_grad`` is its gradient. A sample
is x[n], its positions the axes between the first and the last: images [N, H, W, C], or rows
of tokens [N, C] whose heads are the groups. Values are bfloat16 or float32, weights and
statistics float32; sums are float32 in a fixed order, so that a rerun gives the same bits.

Neither records a graph for autograd: gradients come from ``group_norm_grad`` alone.
"""
from __future__ import annotations

import struct
from collections import namedtuple
from ctypes import c_char_p
from typing import Optional

import torch

from . import _lib
from ._lib import launch
from .ssm import _bits, _dense, _dtype_code, _like, _p, _tokens

DLIB = "libsurf_delta.so"
_V, _I = _lib._V, _lib._I
_lib.register(DLIB, {"surf_group_norm": (_I, [c_char_p, _I, _I, _I, _I, _I, _I, _I, _I, _V])})

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2}
LANES, BLOCK, PARTS = 0, 1, 2
_ARGS = struct.Struct("9q8q2if3iq")

Norm = namedtuple("Norm", "out stats")
NormGrads = namedtuple("NormGrads", "dx dweight dbias")


def _flat(what: str, name: str, x: torch.Tensor) -> tuple:
    """(samples, positions, stride of samples, stride of positions): the axes between the first
    and the last as one."""
    n, p, sp = x.shape[0], 1, 0
    for size, stride in zip(reversed(x.shape[1:-1]), reversed(x.stride()[1:-1])):
        if size == 1:
            continue
        if p == 1:
            sp = stride
        elif stride != p * sp and x.numel():
            raise ValueError(f"{what}: the positions of {name} must lie a constant stride apart")
        p *= size
    return n, p, x.stride(0), sp


def _check(what, x, groups, weight, bias, activation, eps):
    _lib.require_cuda(x, what)
    if x.dim() < 2:
        raise ValueError(f"{what}: x must be [samples, ..., channels]")
    code = _dtype_code(x, what)
    c, at = x.shape[-1], x.get_device()
    groups = int(groups)
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"{what}: the groups must divide the channels, {c} in {groups} do not")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation must be one of {', '.join(ACTIVATIONS)}, not {activation!r}")
    if not 2.0 ** -126 <= eps or not _lib.within_float32(eps):
        raise ValueError(f"{what}: eps must be positive and finite in float32")
    _tokens(what, "x", x, x.shape, x.dtype, at)
    _dense(what, "weight", weight, (c,), torch.float32, at)
    _dense(what, "bias", bias, (c,), torch.float32, at)
    return code, 4 - 2 * code, at, c, groups


def _piece(cg: int, e: int, bits: int) -> int:
    """Channels of a piece: the most that divide a group's and that every row's address allows, up
    to 16 bytes."""
    v = 16 // e
    while v > 1 and (cg % v or bits % (v * e)):
        v //= 2
    return v


def _pow2(n: int) -> int:
    return 1 << max(0, n - 1).bit_length()


def _plan(n: int, p: int, c: int, g: int, e: int, v: int, grad: bool):
    """(form, lanes of a group, pieces that a lane or thread holds, threads, blocks along the samples,
    groups of a slab, parts, positions of a part)."""
    cg = c // g
    per_group = cg // v
    items = p * per_group
    # a warp's registers: up to 4 pieces a lane, or 2 where positions are shorter than a 32-byte sector. Lanes and
    # block, forward and gradient in us: 8192x64x64 g8 61 + 120 and 84 + 139, 8192x8192 g8 103 + 158 and
    # 186 + 256; 2048x128x64 g8 31 + 105 and 28 + 40
    if items <= 64 or (items <= 128 and cg * e >= 32):
        lanes = min(32, _pow2(items))
        hold = _pow2(-(-items // lanes))
        blocks = min(-(-n // 8), max(1, 148 * 4 // -(-g // (32 // lanes))), 65535)
        return LANES, lanes, hold, 256, blocks, 1, 1, p
    # the narrowest slab of whole groups with rows of 32 bytes (a sector) that a block's registers
    # take, twice as wide where that still leaves three for every SM (2048x512x64 g8 97 -> 79 us forward).
    # Block and parts, where both can be: 1x512x64 4.3 + 8.5 and 6.6 + 10.3, 24x512x64 4.6 + 9.1 and 12.3 + 21.3
    threads, most = 256, 4 if grad else 8
    fits = [k for k in range(1, g + 1) if g % k == 0 and k * per_group <= threads and
            -(-p // (threads // (k * per_group))) <= most]
    slab = next((k for k in fits if k * cg * e >= 32), fits[-1] if fits else 0)
    slab = next((k for k in fits if k >= 2 * slab and n * (g // k) >= 148 * 3), slab)
    if slab:
        per = slab * per_group
        hold = -(-p // (threads // per))
        # no more threads than the pieces take
        threads = -(-min(threads // per, -(-p // hold)) * per // 32) * 32
        hold = max(2, _pow2(-(-p // (threads // per))))
        return BLOCK, 0, hold, threads, min(n, max(1, 148 * (2 if grad else 3) // (g // slab))), slab, 1, p
    threads = 256
    slab = max((k for k in range(1, g + 1) if g % k == 0 and k * per_group <= threads), default=1)
    slabs = -(-(c // v) // 32) if grad else g // slab
    parts = max(1, min(-(-148 * 3 // max(1, n * slabs)), -(-p // 16)))
    span = -(-p // parts)
    return PARTS, 0, 0, threads, 0, slab, -(-p // span), span


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5, activation: str = "none", train: bool = False, out: Optional[torch.Tensor] = None) -> Norm:
    """act((x - mean) / sqrt(var + eps) * weight + bias) of x [N, ..., C] over each sample's
    positions and each of ``groups`` groups of channels; ``weight`` and ``bias`` [C] (None: 1
    and 0), ``activation`` none, relu or silu. ``train`` keeps in ``stats`` [N, groups, 2] the
    means and 1 / sqrt(var + eps) that ``group_norm_grad`` starts from. ``out`` may be x itself, and shares no
    memory with an input otherwise."""
    what = "group_norm"
    code, e, at, c, g = _check(what, x, groups, weight, bias, activation, eps)
    if out is None:
        out = _like(x)
    else:
        _tokens(what, "out", out, x.shape, x.dtype, at)
        _lib.require_apart(what, "out", out, dict(x=x, weight=weight, bias=bias), ("x",))
    n, p, xn, xp = _flat(what, "x", x)
    _, _, yn, yp = _flat(what, "out", out)
    stats = torch.empty((n, g, 2), dtype=torch.float32, device=x.device) if train else None
    if n == 0 or p == 0:
        return Norm(out, stats)
    v = _piece(c // g, e, _bits(e, x, out))
    mode, lanes, hold, threads, blocks, slab, parts, span = _plan(n, p, c, g, e, v, False)
    part = torch.empty(n * g * parts * 3, dtype=torch.float32, device=x.device) if mode == PARTS else None
    args = _ARGS.pack(x.data_ptr(), 0, _p(weight), _p(bias), out.data_ptr(), _p(stats), _p(part), 0, 0,
                      xn, xp, 0, 0, yn, yp, n, p, c, g, eps, ACTIVATIONS[activation], slab, parts, span)
    launch(_lib.lib(DLIB).surf_group_norm, "surf_group_norm", at, args, code, 0, v, mode, lanes, hold, threads, blocks)
    if mode == PARTS:
        _lib.add_launches(1)
    return Norm(out, stats)


def group_norm_grad(dy: torch.Tensor, x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None,
                    bias: Optional[torch.Tensor] = None, *, stats: torch.Tensor, activation: str = "none") -> NormGrads:
    """Gradients of ``group_norm`` for the gradient ``dy`` of out: dx in x's type, dweight and
    dbias float32 (None for an input that was None)."""
    what = "group_norm_grad"
    code, e, at, c, g = _check(what, x, groups, weight, bias, activation, 1.0)
    _tokens(what, "dy", dy, x.shape, x.dtype, at)
    if stats is None:
        raise ValueError(f"{what}: needs the statistics that group_norm(train=True) kept")
    _dense(what, "stats", stats, (x.shape[0], g, 2), torch.float32, at)
    if stats.data_ptr() & 7:
        raise ValueError(f"{what}: stats must start on an 8-byte boundary")
    n, p, xn, xp = _flat(what, "x", x)
    _, _, dn, dp = _flat(what, "dy", dy)
    dx = _like(x)
    _, _, yn, yp = _flat(what, "dx", dx)
    dw = None if weight is None else torch.empty_like(weight)
    db = None if bias is None else torch.empty_like(bias)
    if n == 0 or p == 0:
        return NormGrads(dx, None if dw is None else dw.zero_(), None if db is None else db.zero_())
    v = _piece(c // g, e, _bits(e, x, dy, dx))
    mode, lanes, hold, threads, blocks, slab, parts, span = _plan(n, p, c, g, e, v, True)
    rows = n * parts if mode == PARTS else blocks
    part = torch.empty(rows * 2 * c + (n * g * 2 if mode == PARTS else 0), dtype=torch.float32, device=x.device)
    args = _ARGS.pack(x.data_ptr(), dy.data_ptr(), _p(weight), _p(bias), dx.data_ptr(), stats.data_ptr(), part.data_ptr(),
                      _p(dw), _p(db), xn, xp, dn, dp, yn, yp, n, p, c, g, 0.0, ACTIVATIONS[activation], slab, parts, span)
    launch(_lib.lib(DLIB).surf_group_norm, "surf_group_norm", at, args, code, 1, v, mode, lanes, hold, threads, blocks)
    _lib.add_launches((2 if mode == PARTS else 0) + (dw is not None or db is not None))
    return NormGrads(dx, dw, db)


def group_norm_reference(x, groups, weight=None, bias=None, *, eps=1e-5, activation="none"):
    """``group_norm`` from its definition, in the type of its inputs (differentiable)."""
    n, c = x.shape[0], x.shape[-1]
    v = x.reshape(n, -1, groups, c // groups)
    v = v - v.mean((1, 3), keepdim=True)
    v = (v / torch.sqrt((v * v).mean((1, 3), keepdim=True) + eps)).reshape(x.shape)
    if weight is not None:
        v = v * weight
    if bias is not None:
        v = v + bias
    return {"none": lambda t: t, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t)}[activation](v)
