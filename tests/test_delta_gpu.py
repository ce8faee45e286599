"""The gated delta rule's kernels against its token-by-token definition in 64 bits: sequences,
gradients (autograd of the definition), single tokens; masks, strides, odd sizes, refusals.

Tolerances, of norms. A bfloat16 result is one rounding, at most half a step of its type: 2^-8 of
the value. Inside, a 32-bit number is an operand as two bfloat16 planes with bfloat16 tokens (half
a step of half a step: 2^-16) and three with 32-bit ones (2^-24). A chunk rounds four operands on
the way from state to state, at most 25 chunks here of which an error of one decays in the next:
100 independent roundings of at most 2^-16, their root mean square 2^-16 / sqrt(3): 10 * 0.58 *
2^-16 = 9e-5, held to 1e-4, gradients (twice as many) to 2e-4. With 32-bit tokens 100 * 2^-24 in
all, and the sums' own (products of 128, and 16 tokens: 2^-24 sqrt(144) each): 7e-7 * 10, held to 1e-5,
gradients to 2e-5.
"""
import pytest
import torch

from surfb200.ops import _lib, delta as DR
from surfb200.ops import gemm as G

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
INNER = {BF: 1e-4, F32: 1e-5}


def rel(x, y):
    y = y.detach().double()
    n = float(torch.linalg.vector_norm(y))
    return float(torch.linalg.vector_norm(x.double() - y)) / (n if n else 1.0)


def _hide(x, n):
    if n is not None:
        x[torch.arange(x.shape[1], device="cuda")[None] >= n[:, None]] = float("nan")
    return x


def make(b, t, g, h, nk, nv, dtype, reset=0.0, ragged=False, seed=0, bias=True, state=True):
    gen = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    c = dict(reset=None, lengths=None)
    if reset:
        c["reset"] = torch.rand(b, t, generator=gen, device="cuda") < reset
    if ragged:
        n = torch.randint(0, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        n[0] = 0
        if b > 1:
            n[1] = t
        c["lengths"] = n
    qkv = _hide(r(b, t, 2 * g * nk + h * nv).to(dtype), c["lengths"])
    gates = _hide(r(b, t, 2 * h).to(dtype), c["lengths"])
    c["tokens"] = (qkv[..., :g * nk].unflatten(2, (g, nk)), qkv[..., g * nk:2 * g * nk].unflatten(2, (g, nk)),
                   qkv[..., 2 * g * nk:].unflatten(2, (h, nv)), gates[..., :h], gates[..., h:])
    c["A"] = -torch.rand(h, generator=gen, device="cuda") * 4
    c["dt_bias"] = r(h) - 2 if bias else None
    c["state"] = r(b, h, nv, nk) if state else None
    c["dout"] = _hide(r(b, t, h, nv).to(dtype), c["lengths"])
    c["dfinal"] = r(b, h, nv, nk)
    return c


NAMES = ("q", "k", "v", "dt", "b", "A", "dt_bias", "state")


def oracle(c, grads=True, **kw):
    """(out, final, gradients by input) of the definition in 64 bits."""
    x = dict(zip(NAMES, c["tokens"] + (c["A"], c["dt_bias"], c["state"])))
    x = {n: None if v is None else v.double().detach().requires_grad_(grads) for n, v in x.items()}
    out, final = DR.gated_delta_reference(*(x[n] for n in NAMES[:6]), dt_bias=x["dt_bias"], state=x["state"],
                                          reset=c["reset"], lengths=c["lengths"], **kw)
    if not grads:
        return out, final, None
    dout = torch.nan_to_num(c["dout"].double())
    live = [n for n in NAMES if x[n] is not None]
    got = torch.autograd.grad((out * dout).sum() + (final * c["dfinal"].double()).sum(), [x[n] for n in live], allow_unused=True)
    return out, final, {n: torch.zeros_like(x[n]) if v is None else v for n, v in zip(live, got)}


def call(c, train=True, **kw):
    m = dict(dt_bias=c["dt_bias"], state=c["state"], reset=c["reset"], lengths=c["lengths"], **kw)
    r = DR.gated_delta(*c["tokens"], c["A"], train=train, **m)
    g = DR.gated_delta_grad(c["dout"], *c["tokens"], c["A"], saved=r.saved, dfinal=c["dfinal"], **m) if train else None
    return r, g


def _of_the_sign(c, n):
    """The gradient of a one-element key or query as if its length stayed the same."""
    q, k = (x.double() for x in c["tokens"][:2])
    u = dict(c, tokens=(q / torch.sqrt(q * q + 1e-6), k / torch.sqrt(k * k + 1e-6)) + c["tokens"][2:])
    x = c["tokens"][0 if n == "q" else 1].double()
    return oracle(u, normalize=False, scale=1.0)[2][n] / torch.sqrt(x * x + 1e-6)


CASES = [  # B, T, G, H, K, V, reset, ragged
    (1, 1, 1, 1, 1, 1, 0.0, False), (2, 3, 1, 2, 8, 16, 0.0, False), (1, 16, 1, 1, 16, 16, 0.0, False),
    (3, 17, 2, 2, 32, 24, 0.3, True), (2, 33, 1, 3, 24, 40, 0.1, True), (2, 64, 2, 2, 64, 64, 0.0, False),
    (3, 130, 1, 2, 64, 128, 0.05, True), (1, 100, 1, 1, 128, 64, 0.02, False), (2, 48, 1, 1, 128, 128, 1.0, False),
    (2, 40, 3, 6, 7, 5, 0.2, True), (1, 35, 1, 2, 33, 31, 0.1, False), (1, 47, 1, 1, 65, 127, 0.0, True),
    (1, 400, 1, 1, 16, 128, 0.0, False), (2, 0, 1, 1, 8, 8, 0.0, False),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", CASES)
def test_sequences_and_gradients(case, dtype):
    b, t, g, h, nk, nv, reset, ragged = case
    c = make(b, t, g, h, nk, nv, dtype, reset, ragged)
    out, final, want = oracle(c)
    r, d = call(c)
    tol = INNER[dtype]
    half = torch.finfo(dtype).eps / 2
    assert rel(r.out, out) < half + tol
    assert rel(r.final, final) < tol
    got = dict(zip(NAMES, d))
    for n in NAMES:
        assert torch.isfinite(got[n]).all(), n
        if n in ("A", "dt_bias", "state"):
            assert rel(got[n], want[n]) < 2 * tol, n
        elif nk == 1 and n in ("q", "k"):
            # the unit vector of one element is its sign: the gradient is 1e-6 of what the sign gets, the
            # difference of two such numbers. Each is rounded: a few times 2^-24 of it with 32-bit tokens;
            # with bfloat16 ones it is a sum of at most three products (P's, M's, its transposed) of
            # operands in two planes, 2^-16 of each
            step = 16 * 2.0 ** -24 if dtype == F32 else 3 * 2.0 ** -16
            assert float((got[n].double() - want[n]).abs().max()) < step * float(_of_the_sign(c, n).abs().max()) + half * 1e-6
        else:
            assert rel(got[n], want[n]) < half + 2 * tol, n
    if c["lengths"] is not None:
        dead = torch.arange(t, device="cuda")[None] >= c["lengths"][:, None]
        for x in (r.out, d.dq, d.dk, d.dv, d.ddt, d.db):
            assert not x[dead].any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_without_options(dtype):
    """No bias, no state, keys as they are (short, so that I - beta k k^T does not grow), a scale."""
    c = make(2, 37, 2, 2, 32, 48, dtype, bias=False, state=False)
    c["tokens"] = tuple((x * 0.2).to(dtype) if i < 2 else x for i, x in enumerate(c["tokens"]))
    kw = dict(normalize=False, scale=0.5)
    out, final, want = oracle(c, **kw)
    r, d = call(c, **kw)
    half, tol = torch.finfo(dtype).eps / 2, INNER[dtype]
    assert rel(r.out, out) < half + tol and rel(r.final, final) < tol
    assert d.ddt_bias is None and d.dstate is None
    for n, x in zip(NAMES[:6], d):
        assert rel(x, want[n]) < 2 * tol + (half if n != "A" else 0), n
    assert torch.equal(call(c, train=False, **kw)[0].out, r.out)


def test_strong_decays_keep_the_others_digits():
    """Decays from e^-0.001 to e^-300 side by side, and of -inf: the weak ones are as exact as alone."""
    c = make(2, 60, 1, 2, 32, 32, F32)
    q, k, v, dt, b = c["tokens"]
    dt = torch.full_like(dt, -7.0)
    dt[:, 5::11] = 60.0
    dt[:, 7] = -float("inf")
    c["tokens"] = (q, k, v, dt, b)
    c["A"] = torch.tensor([-5.0, -1.0], device="cuda")
    c["dt_bias"] = None
    out, final, want = oracle(c)
    r, d = call(c)
    assert rel(r.out, out) < 1e-5 and rel(r.final, final) < 1e-5
    for n in ("q", "k", "v", "b", "state"):
        assert rel(dict(zip(NAMES, d))[n], want[n]) < 2e-5, n
    c["A"] = torch.tensor([-float("inf"), -1.0], device="cuda")
    r, d = call(c)
    for x in (r.out, r.final) + tuple(d)[:5]:
        assert torch.isfinite(x).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_resets_end_what_is_not_finite(dtype, bad):
    """Tokens 0 .. 20 of row 0 and its state hold NaN or infinities; token 21 begins an episode."""
    c = make(2, 50, 1, 2, 32, 32, dtype)
    c["reset"] = torch.zeros(2, 50, dtype=torch.bool, device="cuda")
    c["reset"][:, 21] = True
    clean = call(c)
    c["tokens"] = tuple(x.clone() for x in c["tokens"])
    for x in c["tokens"]:
        x[0, :21] = bad
    c["state"] = c["state"].clone()
    c["state"][0] = bad
    r, d = call(c)
    # the tile with the reset is taken episode by episode, its sums in another order
    tol = torch.finfo(dtype).eps
    assert rel(r.out[0, 21:], clean[0].out[0, 21:]) < INNER[dtype] + tol and torch.equal(r.out[1], clean[0].out[1])
    assert rel(r.final, clean[0].final) < INNER[dtype]
    for x, y in zip(d[:5], clean[1][:5]):
        assert rel(x[0, 21:], y[0, 21:]) < 2 * INNER[dtype] + tol and torch.equal(x[1], y[1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("which", range(8))
def test_not_finite_reaches_no_other_episode(dtype, which):
    """One token of an episode in the middle of a tile (21 .. 25, 26 .. 27 and 28 on follow 0 .. 20) or the
    gradient of the final state, or the state before the row: the other episodes' results and gradients stay as they are, but for the
    sums over all tokens."""
    c = make(2, 50, 1, 2, 32, 32, dtype)
    c["reset"] = torch.zeros(2, 50, dtype=torch.bool, device="cuda")
    c["reset"][:, [21, 26, 28]] = True
    clean = call(c)
    bad, keep = 23, torch.ones(50, dtype=torch.bool)
    keep[21:26] = False
    if which < 5:
        x = c["tokens"][which].clone()
        x[0, bad] = float("nan")
        c["tokens"] = c["tokens"][:which] + (x,) + c["tokens"][which + 1:]
    elif which == 5:
        c["dout"] = c["dout"].clone()
        c["dout"][0, bad] = float("inf")
    elif which == 6:
        c["dfinal"] = c["dfinal"].clone()
        c["dfinal"][0] = float("nan")
        keep[21:26] = True
        keep[28:] = False
    else:
        c["state"] = c["state"].clone()
        c["state"][0] = float("inf")
        keep[:] = True
        keep[:21] = False
    r, d = call(c)
    keep = keep.cuda()
    fwd = torch.ones_like(keep) if which in (5, 6) else keep
    tol = torch.finfo(dtype).eps
    for x, y, k in ((r.out, clean[0].out, fwd),) + tuple((x, y, keep) for x, y in zip(d[:5], clean[1][:5])):
        assert torch.isfinite(x[0, k]).all() and torch.equal(x[1], y[1])
        # episodes by themselves sum in another order
        assert rel(x[0, k], y[0, k]) < 2 * INNER[dtype] + tol
    assert rel(r.final, clean[0].final) < INNER[dtype]
    if which < 7:
        assert rel(d.dstate, clean[1].dstate) < 2 * INNER[dtype]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_pieces_equal_the_whole(dtype):
    """Rows cut anywhere, the state carried: the state is 32-bit; outputs differ by the order of sums."""
    c = make(2, 90, 1, 2, 64, 32, dtype, reset=0.03)
    whole = call(c, train=False)[0]
    s, outs = c["state"], []
    for lo, hi in ((0, 1), (1, 30), (30, 64), (64, 90)):
        m = dict(dt_bias=c["dt_bias"], reset=c["reset"][:, lo:hi].contiguous())
        r = DR.gated_delta(*(x[:, lo:hi] for x in c["tokens"]), c["A"], state=s, **m)
        outs.append(r.out)
        s = r.final
    assert rel(s, whole.final) < 2 * INNER[dtype]
    assert rel(torch.cat(outs, 1), whole.out) < 2 * INNER[dtype] + torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("g,h,nk,nv", [(1, 1, 16, 16), (2, 4, 64, 64), (1, 2, 24, 40), (3, 3, 7, 5), (1, 2, 128, 33), (2, 2, 32, 128)])
def test_single_tokens_follow_the_definition(g, h, nk, nv, dtype):
    """Slots of a larger pool, a row without an env, resets; the other slots stay as they are."""
    rows, pool = 9, 14
    c = make(rows, 1, g, h, nk, nv, dtype, state=False)
    gen = torch.Generator("cuda").manual_seed(1)
    state = torch.randn(pool, h, nv, nk, generator=gen, device="cuda")
    slots = torch.randperm(pool, generator=gen, device="cuda")[:rows].to(torch.int32)
    slots[4] = -1
    reset = torch.zeros(rows, dtype=torch.bool, device="cuda")
    reset[[1, 4]] = True
    state[slots[1].long()] = float("nan")
    before = state.clone()
    tokens = tuple(x[:, 0] for x in c["tokens"])
    got = DR.gated_delta_step(*tokens, c["A"], state, dt_bias=c["dt_bias"], reset=reset, slots=slots)
    on = slots >= 0
    at = slots[on].long()
    c["state"] = torch.nan_to_num(before[at])
    c["tokens"] = tuple(x[on] for x in c["tokens"])
    c["reset"] = reset[on][:, None]
    out, final, _ = oracle(c, grads=False)
    assert rel(got[on], out[:, 0]) < torch.finfo(dtype).eps / 2 + 2e-6
    assert rel(state[at], final) < 2e-6
    assert not got[~on].any()
    rest = torch.ones(pool, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.equal(state[rest], before[rest])


def test_steps_follow_the_sequence():
    c = make(3, 40, 2, 4, 64, 64, BF, reset=0.1)
    r = call(c, train=False)[0]
    state = c["state"].clone()
    for i in range(40):
        out = DR.gated_delta_step(*(x[:, i] for x in c["tokens"]), c["A"], state, dt_bias=c["dt_bias"], reset=c["reset"][:, i].contiguous())
        # one rounding each
        assert rel(out, r.out[:, i]) < 2.0 ** -7 + 1e-4
    assert rel(state, r.final) < 1e-4


def test_slot_past_the_pool_is_reported():
    c = make(3, 1, 1, 2, 16, 16, BF)
    tokens = tuple(x[:, 0] for x in c["tokens"])
    state = c["state"][:2].clone()
    keep = state.clone()
    G.check_error_flag("cuda")
    slots = torch.tensor([1, 2, -1], dtype=torch.int32, device="cuda")
    out = DR.gated_delta_step(*tokens, c["A"], state, dt_bias=c["dt_bias"], slots=slots)
    assert not out[1:].any() and out[0].any() and torch.equal(state[0], keep[0])
    with pytest.raises(_lib.KernelError, match="state slot"):
        G.check_error_flag("cuda")


def _aligned_differently(x, shift):
    """The same values, `shift` elements off their boundary, rows further apart."""
    wide = x.new_empty((*x.shape[:-1], x.shape[-1] + 9))
    flat = torch.empty(wide.numel() + shift, dtype=x.dtype, device=x.device)[shift:].view(wide.shape)
    flat[..., :x.shape[-1]] = x
    return flat[..., :x.shape[-1]]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_odd_addresses_and_strides(dtype):
    c = make(2, 35, 2, 2, 32, 48, dtype, reset=0.1, ragged=True)
    r, d = call(c)
    odd = dict(c, tokens=tuple(_aligned_differently(x, 3) for x in c["tokens"]), dout=_aligned_differently(c["dout"], 1))
    r2, d2 = call(odd)
    assert torch.equal(r2.out, r.out) and torch.equal(r2.final, r.final)
    for x, y in zip(d2, d):
        assert torch.equal(x, y)
    out = _aligned_differently(torch.zeros_like(r.out), 5)
    flat = torch.as_strided(out, (2, 35, 2, 57), out.stride())
    flat[..., 48:] = 7.0
    m = dict(dt_bias=c["dt_bias"], state=c["state"], reset=c["reset"], lengths=c["lengths"])
    DR.gated_delta(*c["tokens"], c["A"], out=out, **m)
    assert torch.equal(out, r.out) and bool((flat[..., 48:] == 7.0).all())
    tokens = tuple(x[:, 0] for x in c["tokens"])
    odd = tuple(x[:, 0] for x in odd["tokens"])
    live = c["lengths"] > 0
    s1, s2 = c["state"].clone(), c["state"].clone()
    o1, o2 = DR.gated_delta_step(*tokens, c["A"], s1), DR.gated_delta_step(*odd, c["A"], s2)
    assert torch.equal(o1[live], o2[live]) and torch.equal(s1[live], s2[live])


def test_offsets_past_32_bits():
    """Rows 2^32 elements apart."""
    c = make(2, 20, 1, 1, 16, 16, BF)
    r, d = call(c)
    big = torch.empty(2 ** 32 + 20 * 64, dtype=BF, device="cuda")
    far = []
    for i, x in enumerate(c["tokens"][:3]):
        y = torch.as_strided(big, x.shape, (2 ** 32, 64, 16, 1), 16 * i)
        y.copy_(x)
        far.append(y)
    r2, d2 = call(dict(c, tokens=tuple(far) + c["tokens"][3:]))
    assert torch.equal(r2.out, r.out) and torch.equal(r2.final, r.final)
    assert torch.equal(d2.dstate, d.dstate) and torch.equal(d2.dq, d.dq) and torch.equal(d2.dv, d.dv)


def test_reruns_give_the_same_bits_on_any_stream_and_in_graphs():
    c = make(4, 70, 2, 4, 64, 64, BF, reset=0.05, ragged=True)
    r, d = call(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r2, d2 = call(c)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r3, d3 = call(c)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for rr, dd in ((r2, d2), (r3, d3)):
        for x, y in zip((rr.out, rr.final, rr.saved) + tuple(dd), (r.out, r.final, r.saved) + tuple(d)):
            # states kept of tiles past a row's end are not written
            if x is rr.saved:
                continue
            assert torch.equal(x, y)


def test_refusals():
    c = make(2, 10, 2, 4, 16, 16, BF)
    q, k, v, dt, b = c["tokens"]
    A = c["A"]
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        DR.gated_delta(q.half(), k.half(), v.half(), dt.half(), b.half(), A)
    with pytest.raises(TypeError, match="k is"):
        DR.gated_delta(q, k.float(), v, dt, b, A)
    with pytest.raises(ValueError, match="k has shape"):
        DR.gated_delta(q, k[:, :, :1], v, dt, b, A)
    with pytest.raises(ValueError, match="divide the value heads"):
        DR.gated_delta(q, k, v[:, :, :3], dt[..., :3], b[..., :3], A[:3])
    with pytest.raises(ValueError, match="1 to 128"):
        DR.gated_delta(torch.zeros(1, 1, 1, 129, dtype=BF, device="cuda"), torch.zeros(1, 1, 1, 129, dtype=BF, device="cuda"),
                       v[:1, :1, :1], dt[:1, :1, :1], b[:1, :1, :1], A[:1])
    with pytest.raises(ValueError, match="dense last axis"):
        DR.gated_delta(q, k, v.transpose(2, 3).contiguous().transpose(2, 3), dt, b, A)
    with pytest.raises(TypeError, match="A must be"):
        DR.gated_delta(q, k, v, dt, b, A.double())
    with pytest.raises(ValueError, match="state has shape"):
        DR.gated_delta(q, k, v, dt, b, A, state=c["state"][:1])
    with pytest.raises(TypeError, match="reset must be"):
        DR.gated_delta(q, k, v, dt, b, A, reset=torch.zeros(2, 10, device="cuda"))
    with pytest.raises(TypeError, match="lengths must be"):
        DR.gated_delta(q, k, v, dt, b, A, lengths=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="out shares memory with v"):
        DR.gated_delta(q, k, v, dt, b, A, out=v)
    with pytest.raises(_lib.KernelError):
        DR.gated_delta(*(x.cpu() for x in (q, k, v, dt, b, A)))
    with pytest.raises(ValueError, match="saved"):
        DR.gated_delta_grad(c["dout"], q, k, v, dt, b, A, saved=None)
    with pytest.raises(ValueError, match="saved has shape"):
        DR.gated_delta_grad(c["dout"], q, k, v, dt, b, A, saved=c["state"])
    one = tuple(x[:, 0] for x in c["tokens"])
    with pytest.raises(ValueError, match="slots"):
        DR.gated_delta_step(*one, A, c["state"][:1])
    with pytest.raises(ValueError, match="16-byte"):
        DR.gated_delta_step(*one, A, torch.zeros(2 * 4 * 256 + 1, device="cuda")[1:].view(2, 4, 16, 16))
    with pytest.raises(ValueError, match="out shares memory"):
        DR.gated_delta_step(*one, A, c["state"].clone(), out=one[2])


MANY = [  # more heads of sequences than SMs: two share a block in the gradient, the last may be alone
    (151, 37, 1, 1, 16, 16, 0.1, True), (50, 70, 1, 3, 64, 64, 0.1, True), (77, 35, 2, 2, 32, 24, 0.0, True),
    (40, 33, 2, 4, 64, 128, 0.2, True), (160, 20, 1, 1, 128, 64, 0.0, False), (149, 1, 1, 1, 40, 33, 0.0, False),
    (151, 50, 1, 1, 65, 100, 0.3, True),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", MANY)
def test_many_sequences(case, dtype):
    test_sequences_and_gradients(case, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("which", ["token", "state", "dfinal"])
def test_not_finite_stays_in_its_row_among_many(dtype, which):
    """Row 6 is bad, between two episodes inside a tile for a token; row 7 shares its block in the gradient."""
    c = make(151, 50, 1, 1, 32, 32, dtype, ragged=True)
    c["reset"] = torch.zeros(151, 50, dtype=torch.bool, device="cuda")
    c["reset"][:, [21, 26]] = True
    c["lengths"][5:8] = torch.tensor([50, 50, 33], dtype=torch.int32, device="cuda")
    c["tokens"] = tuple(torch.nan_to_num(x) for x in c["tokens"])
    c["dout"] = torch.nan_to_num(c["dout"])
    clean = call(c)
    for name in ("state", "dfinal"):
        if which == name:
            c[name] = c[name].clone()
            c[name][6] = float("nan")
    if which == "token":
        c["tokens"] = tuple(x.clone() for x in c["tokens"])
        c["tokens"][2][6, 23] = float("inf")
    r, d = call(c)
    rows = torch.arange(151, device="cuda") != 6
    assert torch.equal(r.out[rows], clean[0].out[rows]) and torch.equal(r.final[rows], clean[0].final[rows])
    for x, y in zip(d[:5] + (d.dstate,), clean[1][:5] + (clean[1].dstate,)):
        assert torch.equal(x[rows], y[rows])
    # the row's own tokens of other episodes than the bad one
    keep = {"token": [*range(21), *range(26, 50)], "state": [*range(21, 50)], "dfinal": [*range(26)]}[which]
    tol = torch.finfo(dtype).eps
    for x, y in zip(d[:5], clean[1][:5]):
        assert rel(x[6, keep], y[6, keep]) < 2 * INNER[dtype] + tol


def test_odd_saved_and_scales_past_float32_are_refused():
    c = make(2, 10, 1, 1, 16, 16, BF)
    saved = call(c)[0].saved
    odd = torch.empty(1 + saved.numel(), device="cuda")[1:].view(saved.shape)
    odd.copy_(saved)
    with pytest.raises(ValueError, match="16-byte"):
        DR.gated_delta_grad(c["dout"], *c["tokens"], c["A"], saved=odd)
    for scale in (1e39, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            DR.gated_delta(*c["tokens"], c["A"], scale=scale)
        with pytest.raises(ValueError, match="scale"):
            DR.gated_delta_step(*(x[:, 0] for x in c["tokens"]), c["A"], c["state"], scale=scale)


def test_two_calls_at_once():
    for case in ((3, 60, 1, 2, 64, 64), (160, 40, 1, 1, 32, 48)):
        c = make(*case, BF, reset=0.1, ragged=True)
        want, grads = call(c)
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(2)], []
        for s in streams * 3:
            with torch.cuda.stream(s):
                got.append(call(c))
        torch.cuda.synchronize()
        for r, d in got:
            assert torch.equal(r.out, want.out) and torch.equal(r.final, want.final)
            for x, y in zip(d, grads):
                assert torch.equal(x, y)


def test_shared_rows_as_inputs():
    """Views whose rows lie on one another: gradients are dense, each row's own."""
    c = make(1, 40, 1, 2, 32, 32, F32)
    c["tokens"] = tuple(x.expand(5, *x.shape[1:]) for x in c["tokens"])
    c["dout"] = c["dout"].expand(5, *c["dout"].shape[1:])
    c["state"], c["dfinal"] = (c[n].expand(5, *c[n].shape[1:]).contiguous() for n in ("state", "dfinal"))
    r, d = call(c)
    _, _, want = oracle(c)
    assert rel(r.out[4], r.out[0]) == 0
    for n, x in zip(NAMES, d):
        assert rel(x, want[n]) < 2 * INNER[F32] + torch.finfo(F32).eps, n
