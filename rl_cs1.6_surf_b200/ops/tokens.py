"""Sampled answers from rows of logits (csrc/kernels/tokens.cu).

``sample_tokens`` applies temperature, min-p, top-k and top-p and draws one answer
per row (or per head of a row) with a given uniform number. The rule, shared by the
kernel and ``sample_tokens_reference``:

* with m the row's largest logit, e = exp((z - m) / temperature) in float32 and the
  weight is the whole number w = floor(e * 2^40): sums of weights are exact, so the
  answer does not depend on the order they are taken in;
* kept are the candidates with e >= min_p; of these the first ``top_k`` in the order
  (logit falling, index rising); of these the ones that have less than
  ceil(top_p * their total weight) before them;
* the answer is the first index whose running kept weight exceeds floor(u * W), W the
  kept total, and its log-probability is log(w / W).

NaN logits count as -inf. A row with nothing else answers -1, log-probability -inf.
Temperature 0 takes the largest logit (the first of equals).
"""
from __future__ import annotations

import struct
from ctypes import c_char_p
from itertools import accumulate
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import launch

SLIB = "libsurf_seq.so"
_V, _I = _lib._V, _lib._I
_lib.register(SLIB, {"surf_sample_tokens": (_I, [c_char_p, _I, _I, _V])})

MAX_HEADS, MAX_VOCAB = 16, 16 * 16384
_ARGS = struct.Struct("9q3f3i32i")
_SCALE = float(1 << 40)


def _per_row(name: str, v, rows: int, dtype, device):
    """(device pointer, number) of a rule's parameter: one number, or a tensor with one per row."""
    if not isinstance(v, torch.Tensor):
        return 0, v
    if v.shape != (rows,) or v.dtype != dtype or v.device != device or not v.is_contiguous():
        raise ValueError(f"sample_tokens: {name} must be one number or a contiguous {dtype} tensor [{rows}] on {device}")
    return v.data_ptr(), 0


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  heads: Optional[Sequence[int]] = None, out: Optional[torch.Tensor] = None,
                  logp: Optional[torch.Tensor] = None):
    """(tokens int32 [R, H], log-probabilities float32 [R, H]) of ``logits`` [R, V]
    (float32 or bfloat16, rows any stride apart) with uniform numbers ``u`` [R, H] in
    [0, 1). Without ``heads`` the row is one answer (H = 1); with them its columns are the
    heads' categories side by side, each an answer of its own. ``temperature``, ``top_p``,
    ``min_p`` (float32) and ``top_k`` (int32; 0: no limit) are numbers or tensors [R]. ``out`` and
    ``logp`` must not share memory with an input: other blocks of a row's cluster still read its
    number when the answer is written."""
    _lib.require_cuda(logits, "sample_tokens")
    if logits.dim() != 2:
        raise ValueError("sample_tokens: logits must be [rows, candidates]")
    if logits.dtype == torch.bfloat16:
        code = 1
    elif logits.dtype == torch.float32:
        code = 0
    else:
        raise TypeError(f"sample_tokens: logits must be bfloat16 or float32, not {logits.dtype}")
    rows, width = logits.shape
    dev = logits.device
    if width > 1 and logits.stride(1) != 1:
        raise ValueError("sample_tokens: logits need a dense last axis")
    sizes = (width,) if heads is None else tuple(heads)
    n = len(sizes)
    if not 1 <= n <= MAX_HEADS or min(sizes) < 1 or sum(sizes) > width:
        raise ValueError(f"sample_tokens: heads must be 1 to {MAX_HEADS} positive sizes within {width} columns")
    widest = max(sizes)
    if widest > MAX_VOCAB:
        raise ValueError(f"sample_tokens: at most {MAX_VOCAB} candidates, not {widest}")
    if u.shape != (rows, n) or u.dtype != torch.float32 or u.device != dev or not u.is_contiguous():
        raise ValueError(f"sample_tokens: u must be a contiguous float32 tensor [{rows}, {n}] on {dev}")
    f32 = torch.float32
    tp, t0 = _per_row("temperature", temperature, rows, f32, dev)
    kp, k0 = _per_row("top_k", top_k, rows, torch.int32, dev)
    pp, p0 = _per_row("top_p", top_p, rows, f32, dev)
    mp, m0 = _per_row("min_p", min_p, rows, f32, dev)
    if not t0 >= 0 or k0 < 0 or not 0 <= p0 <= 1 or not 0 <= m0 <= 1:
        raise ValueError("sample_tokens: temperature and top_k must not be negative, top_p and min_p lie in [0, 1]")
    for name, t, dt in (("out", out, torch.int32), ("logp", logp, f32)):
        if t is not None and (t.shape != (rows, n) or t.dtype != dt or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"sample_tokens: {name} must be a contiguous {dt} tensor [{rows}, {n}] on {dev}")
    if out is not None or logp is not None:
        inputs = dict(logits=logits, u=u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        if out is not None:
            _lib.require_apart("sample_tokens", "out", out, dict(inputs, logp=logp))
        if logp is not None:
            _lib.require_apart("sample_tokens", "logp", logp, inputs)
    if out is None:
        out = torch.empty_like(u, dtype=torch.int32)
    if logp is None:
        logp = torch.empty_like(u)
    if rows == 0:
        return out, logp
    pad = (0,) * (MAX_HEADS - n)
    offsets = (0, *accumulate(sizes[:-1]))
    args = _ARGS.pack(logits.data_ptr(), u.data_ptr(), tp, pp, mp, kp, out.data_ptr(), logp.data_ptr(), logits.stride(0),
                      t0, p0, m0, min(int(k0), 2 ** 31 - 1), rows, n, *offsets, *pad, *sizes, *pad)
    launch(_lib.lib(SLIB).surf_sample_tokens, "surf_sample_tokens", logits.get_device(), args, code, widest)
    return out, logp


def sample_tokens_reference(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                            heads: Optional[Sequence[int]] = None):
    """The same rule by sorting, row by row (CPU path and the kernel's oracle)."""
    rows, width = logits.shape
    sizes = (width,) if heads is None else tuple(heads)
    tokens = torch.full((rows, len(sizes)), -1, dtype=torch.int32)
    logp = torch.full((rows, len(sizes)), float("-inf"))

    def of(v, r):
        return v[r].item() if isinstance(v, torch.Tensor) else v

    off = 0
    for h, size in enumerate(sizes):
        for r in range(rows):
            t, k, p, q = (of(v, r) for v in (temperature, top_k, top_p, min_p))
            z = logits[r, off:off + size].float().cpu()
            z = torch.where(z.isnan(), torch.tensor(float("-inf")), z)
            m = z.max()
            if m == float("-inf"):
                continue
            inv, k = (1.0 / torch.tensor(t, dtype=torch.float32), k) if t > 0 else (torch.tensor(1.0), 1)
            e = torch.where(z == m, torch.tensor(1.0), torch.exp((z - m) * inv))
            w = torch.where((z > float("-inf")) & (e >= min(q, 1.0)), e * _SCALE, torch.tensor(0.0)).long()
            order = torch.sort(z, descending=True, stable=True).indices
            ranked = w[order]
            if k > 0:
                ranked[k:] = 0
            if p < 1.0:
                total = ranked.sum()
                lim = max(1, int(torch.ceil(torch.tensor(p, dtype=torch.float32).double() * total.double())))
                ranked[(ranked.cumsum(0) - ranked) >= lim] = 0
            kept = torch.zeros_like(w)
            kept[order] = ranked
            upto = kept.cumsum(0)
            at = min(int(float(u[r, h]) * float(upto[-1])), int(upto[-1]) - 1)
            i = int((upto <= at).sum())
            tokens[r, h] = i
            logp[r, h] = torch.log(kept[i].double() / upto[-1].double()).float()
        off += size
    return tokens, logp
