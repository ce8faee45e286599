"""Causal convolution and selective scan kernels against their token-by-token
definition in 64 bits: sequences, gradients (autograd of the definition, and
differences), single tokens; masks, strides, odd sizes, refusals.

Tolerances. bfloat16 results are one rounding (2^-9 relative) of a 32-bit value: the
norm of the difference stays under 2^-8 of the result's. 32-bit results: a decay
exp(delta A) carries a relative error of up to 2^-22 (hardware exponential) plus
2^-23 |delta A| (its argument); the error of a state is the sum of its factors',
at most `memory` tokens back, where memory = 1 / (1 - largest decay) is about 100 here
(delta >= 0.01, A <= -1): 100 * 2^-22 = 2.4e-5 if all of them erred one way; the
norms are held to that. Convolutions sum at most 4 products: 1e-6 covers 16 roundings
of 2^-24; gradients summed over n tokens add at most n roundings, held to 1e-5 in norm.
"""
import pytest
import torch

from surfb200.ops import _lib, ssm
from surfb200.ops import gemm as G

pytestmark = pytest.mark.gpu
TOL = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.4e-5}


def rel(x, y):
    y = y.detach().double()
    n = float(torch.linalg.vector_norm(y))
    return float(torch.linalg.vector_norm(x.double() - y)) / (n if n else 1.0)


def _masks(b, t, gen, reset, ragged):
    r = torch.rand(b, t, generator=gen, device="cuda") < 0.1 if reset else None
    n = None
    if ragged:
        n = torch.randint(0, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        n[0] = 0
        if b > 1:
            n[1] = t
    return r, n


def _hide(x, n):
    if n is not None:
        x[torch.arange(x.shape[1], device="cuda")[None] >= n[:, None]] = float("nan")
    return x


CONV = [  # B, T, D, W, reset, ragged
    (1, 1, 1, 2, False, False), (2, 3, 8, 4, True, False), (3, 17, 36, 3, True, True), (2, 130, 33, 4, True, True),
    (4, 64, 256, 4, False, True), (1, 1000, 12, 4, True, False), (5, 16, 132, 2, True, True), (2, 0, 16, 4, False, False),
]


def _conv_case(b, t, d, w, reset, ragged, dtype, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    flags, n = _masks(b, t, gen, reset, ragged)
    xz = _hide(r(b, t, 2 * d).to(dtype), n)
    return dict(x=xz[..., d:], weight=r(d, w) / 2, bias=r(d), state=r(b, w - 1, d).to(dtype), reset=flags, lengths=n,
                dy=_hide(r(b, t, d).to(dtype), n), dfinal=r(b, w - 1, d).to(dtype))


def _conv_exact(c, silu=True, grad=True):
    f = {k: c[k].double().requires_grad_() for k in ("x", "weight", "bias", "state")}
    y, final = ssm.causal_conv_reference(f["x"], f["weight"], f["bias"], state=f["state"], reset=c["reset"],
                                         lengths=c["lengths"], silu=silu)
    if not grad:
        return y, final
    dy = torch.nan_to_num(c["dy"].double())
    loss = (y * dy).sum() + (final * c["dfinal"].double()).sum()
    return y, final, torch.autograd.grad(loss, [f[k] for k in ("x", "weight", "bias", "state")], allow_unused=True,
                                         materialize_grads=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", CONV, ids=str)
def test_conv_and_gradient(case, dtype):
    c = _conv_case(*case, dtype)
    kw = dict(state=c["state"], reset=c["reset"], lengths=c["lengths"])
    y, final = ssm.causal_conv(c["x"], c["weight"], c["bias"], **kw)
    g = ssm.causal_conv_grad(c["dy"], c["x"], c["weight"], c["bias"], dfinal=c["dfinal"], **kw)
    ey, ef, eg = _conv_exact(c)
    one = 2.0 ** -8 if dtype == torch.bfloat16 else 1e-6
    assert rel(y, ey) <= one
    assert torch.equal(final.double(), ef.detach())          # moved, never computed
    assert rel(g.dx, eg[0]) <= one and rel(g.dstate, eg[3]) <= one
    assert rel(g.dweight, eg[1]) <= 1e-5 and rel(g.dbias, eg[2]) <= 1e-5
    again = ssm.causal_conv_grad(c["dy"], c["x"], c["weight"], c["bias"], dfinal=c["dfinal"], **kw)
    assert all(torch.equal(p, q) for p, q in zip(g, again))


@pytest.mark.parametrize("t", [128, 129])
def test_conv_over_the_longest_stretches(t):
    """As many rows as fill the GPU without cutting: stretches of 128 tokens, one more behind."""
    assert ssm._stretches(304, t, 128)[0] == 128
    c = _conv_case(304, t, 512, 4, True, True, torch.float32)
    kw = dict(state=c["state"], reset=c["reset"], lengths=c["lengths"])
    y, final = ssm.causal_conv(c["x"], c["weight"], c["bias"], **kw)
    g = ssm.causal_conv_grad(c["dy"], c["x"], c["weight"], c["bias"], dfinal=c["dfinal"], **kw)
    ey, ef, eg = _conv_exact(c)
    assert rel(y, ey) <= 1e-6 and torch.equal(final.double(), ef.detach())
    assert rel(g.dx, eg[0]) <= 1e-6 and rel(g.dstate, eg[3]) <= 1e-6
    assert rel(g.dweight, eg[1]) <= 1e-5 and rel(g.dbias, eg[2]) <= 1e-5


def test_conv_without_state_bias_or_silu():
    c = _conv_case(2, 37, 20, 3, True, False, torch.float32)
    y, final = ssm.causal_conv(c["x"], c["weight"], reset=c["reset"], silu=False)
    ey, ef = ssm.causal_conv_reference(c["x"].double(), c["weight"].double(), reset=c["reset"], silu=False)
    assert rel(y, ey) <= 1e-6 and torch.equal(final.double(), ef)
    g = ssm.causal_conv_grad(c["dy"], c["x"], c["weight"], reset=c["reset"], silu=False)
    x = c["x"].double().requires_grad_()
    yy, _ = ssm.causal_conv_reference(x, c["weight"].double(), reset=c["reset"], silu=False)
    assert rel(g.dx, torch.autograd.grad((yy * c["dy"].double()).sum(), x)[0]) <= 1e-6
    assert g.dbias is None and g.dstate is None


def test_conv_in_pieces_equals_whole():
    c = _conv_case(2, 50, 24, 4, True, False, torch.bfloat16)
    y, final = ssm.causal_conv(c["x"], c["weight"], c["bias"], state=c["state"], reset=c["reset"])
    st, out = c["state"], []
    for lo, hi in ((0, 1), (1, 18), (18, 50)):
        o, st = ssm.causal_conv(c["x"][:, lo:hi], c["weight"], c["bias"], state=st, reset=c["reset"][:, lo:hi].contiguous())
        out.append(o)
    assert torch.equal(torch.cat(out, 1), y) and torch.equal(st, final)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 33])
def test_conv_step_equals_sequence(d, dtype):
    c = _conv_case(3, 9, d, 4, True, False, dtype)
    y, final = ssm.causal_conv(c["x"], c["weight"], c["bias"], state=c["state"], reset=c["reset"])
    pool = torch.full((7, 3, d), 5.0, device="cuda", dtype=dtype)
    slots = torch.tensor([6, -1, 2], dtype=torch.int32, device="cuda")
    pool[6], pool[2] = c["state"][0], c["state"][2]
    for i in range(9):
        o = ssm.causal_conv_step(c["x"][:, i], c["weight"], c["bias"], pool, reset=c["reset"][:, i].contiguous(), slots=slots)
        assert torch.equal(o[0], y[0, i]) and torch.equal(o[2], y[2, i]) and not o[1].any()
    assert torch.equal(pool[6], final[0]) and torch.equal(pool[2], final[2])
    assert (pool[[0, 1, 3, 4, 5]] == 5).all()


SCAN = [  # B, T, D, N, groups, reset, ragged
    (1, 1, 1, 1, 1, False, False), (2, 7, 6, 3, 2, True, False), (3, 33, 36, 8, 2, True, True),
    (2, 40, 130, 16, 1, True, True), (1, 700, 48, 16, 1, True, False), (2, 513, 16, 4, 1, False, True),
    (2, 100, 24, 24, 3, True, True), (1, 300, 20, 64, 1, False, False), (2, 0, 16, 16, 1, False, False),
    (3, 129, 64, 32, 2, True, True), (1, 2100, 128, 16, 2, True, True),
]


def _scan_case(b, t, d, n, g, reset, ragged, dtype, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    flags, lens = _masks(b, t, gen, reset, ragged)
    xz = _hide(r(b, t, 2 * d).to(dtype), lens)
    bc = _hide(r(b, t, 2 * g * n).to(dtype), lens)
    delta = 0.01 + 0.1 * torch.rand(d, generator=gen, device="cuda")
    return dict(x=xz[..., :d], z=xz[..., d:], dt=_hide((0.3 * r(b, t, d)).to(dtype), lens),
                A=-(1 + 4 * torch.rand(d, n, generator=gen, device="cuda")), B=bc[..., :g * n].unflatten(2, (g, n)),
                C=bc[..., g * n:].unflatten(2, (g, n)), D=r(d), dt_bias=torch.log(torch.expm1(delta)), state=r(b, d, n),
                reset=flags, lengths=lens, dout=_hide(r(b, t, d).to(dtype), lens), dfinal=r(b, d, n))


KEYS = ("x", "dt", "z", "B", "C", "A", "D", "dt_bias", "state")


def _scan_exact(c, keys=KEYS, softplus=True):
    f = {k: c[k].double().requires_grad_() if k in keys else None for k in KEYS}
    out, final = ssm.selective_scan_reference(f["x"], f["dt"], f["A"], f["B"], f["C"], D=f["D"], z=f["z"],
                                              dt_bias=f["dt_bias"], state=f["state"], reset=c["reset"],
                                              lengths=c["lengths"], softplus=softplus)
    loss = (out * torch.nan_to_num(c["dout"].double())).sum() + (final * c["dfinal"].double()).sum()
    return out, final, dict(zip(keys, torch.autograd.grad(loss, [f[k] for k in keys], allow_unused=True,
                                                          materialize_grads=True)))


def _scan_run(c, keys=KEYS, softplus=True):
    args = [c[k] for k in ("x", "dt", "A", "B", "C")]
    kw = {k: c[k] if k in keys else None for k in ("D", "z", "dt_bias", "state")}
    kw.update(reset=c["reset"], lengths=c["lengths"], softplus=softplus)
    r = ssm.selective_scan(*args, train=True, **kw)
    g = ssm.selective_scan_grad(c["dout"], *args, saved=r.saved, dfinal=c["dfinal"], **kw)
    return r, g


def _named(g):
    return dict(x=g.dx, dt=g.ddt, z=g.dz, B=g.dB, C=g.dC, A=g.dA, D=g.dD, dt_bias=g.ddt_bias, state=g.dstate)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", SCAN, ids=str)
def test_scan_and_gradient(case, dtype):
    c = _scan_case(*case, dtype)
    r, g = _scan_run(c)
    out, final, grads = _scan_exact(c)
    assert rel(r.out, out) <= TOL[dtype]
    assert rel(r.final, final) <= TOL[torch.float32]
    for k, v in _named(g).items():
        assert rel(v, grads[k]) <= TOL[v.dtype], k
    again = ssm.selective_scan_grad(c["dout"], *[c[k] for k in ("x", "dt", "A", "B", "C")], saved=r.saved, D=c["D"],
                                    z=c["z"], dt_bias=c["dt_bias"], state=c["state"], reset=c["reset"],
                                    lengths=c["lengths"], dfinal=c["dfinal"])
    assert all(torch.equal(p, q) for p, q in zip(g, again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,chunks", [(2, 127, 1), (2, 128, 8), (2, 129, 9), (2, 145, 10), (19, 200, None)])
def test_scan_about_the_rule_that_cuts(b, t, chunks, dtype):
    """Lengths where rows begin to be cut, a last chunk of one token, few and many chunks."""
    d = 64 if b == 2 else 1000
    got = ssm._chunks(b, t, d, 16, 1)[1]
    assert got == chunks if chunks else got != 2
    c = _scan_case(b, t, d, 16, 1, True, True, dtype)
    r, g = _scan_run(c)
    out, final, grads = _scan_exact(c)
    assert rel(r.out, out) <= TOL[dtype] and rel(r.final, final) <= TOL[torch.float32]
    for k, v in _named(g).items():
        assert rel(v, grads[k]) <= TOL[v.dtype], k


@pytest.mark.parametrize("softplus", [True, False])
def test_scan_bare(softplus):
    """No gate, skip, bias or start; delta as given."""
    c = _scan_case(2, 45, 32, 16, 1, True, False, torch.float32)
    if not softplus:
        c["dt"] = c["dt"].abs()
    keys = ("x", "dt", "B", "C", "A")
    r, g = _scan_run(c, keys, softplus)
    out, final, grads = _scan_exact(c, keys, softplus)
    assert rel(r.out, out) <= TOL[torch.float32] and rel(r.final, final) <= TOL[torch.float32]
    got = _named(g)
    assert all(rel(got[k], grads[k]) <= TOL[torch.float32] for k in keys)
    assert g.dz is None and g.dD is None and g.ddt_bias is None and g.dstate is None


def test_scan_gradient_by_differences():
    """The gradients against differences of the 64-bit definition along random directions:
    (f(p + e v) - f(p - e v)) / 2 e is off by e^2 f''' / 6, nothing at e = 1e-4 next to the
    32-bit error."""
    c = _scan_case(2, 60, 24, 16, 2, True, True, torch.float32, seed=3)
    _, g = _scan_run(c)
    gen = torch.Generator("cuda").manual_seed(9)

    def value(over):
        f = {k: torch.nan_to_num(c[k].double()) for k in KEYS}
        f.update(over)
        o, h = ssm.selective_scan_reference(f["x"], f["dt"], f["A"], f["B"], f["C"], D=f["D"], z=f["z"],
                                            dt_bias=f["dt_bias"], state=f["state"], reset=c["reset"], lengths=c["lengths"])
        return float((o * torch.nan_to_num(c["dout"].double())).sum() + (h * c["dfinal"].double()).sum())

    for k, v in _named(g).items():
        p = torch.nan_to_num(c[k].double())
        way = torch.randn(p.shape, generator=gen, device="cuda", dtype=torch.float64)
        e = 1e-4
        num = (value({k: p + e * way}) - value({k: p - e * way})) / (2 * e)
        scale = float(torch.linalg.vector_norm(v.double()) * torch.linalg.vector_norm(way))
        assert abs(num - float((v.double() * way).sum())) <= TOL[torch.float32] * scale, k


def test_scan_in_pieces_equals_whole():
    c = _scan_case(2, 90, 32, 16, 1, True, False, torch.float32)
    kw = dict(D=c["D"], dt_bias=c["dt_bias"])
    whole = ssm.selective_scan(c["x"], c["dt"], c["A"], c["B"], c["C"], z=c["z"], state=c["state"], reset=c["reset"], **kw)
    st, out = c["state"], []
    for lo, hi in ((0, 1), (1, 40), (40, 90)):
        cut = [c[k][:, lo:hi] for k in ("x", "dt", "B", "C", "z")]
        r = ssm.selective_scan(cut[0], cut[1], c["A"], cut[2], cut[3], z=cut[4], state=st,
                               reset=c["reset"][:, lo:hi].contiguous(), **kw)
        out.append(r.out)
        st = r.final
    assert rel(torch.cat(out, 1), whole.out) <= 1e-6 and rel(st, whole.final) <= 1e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,n,g", [(64, 16, 1), (33, 5, 3), (24, 64, 2), (8, 1, 1)])
def test_scan_step_follows_the_definition(d, n, g, dtype):
    c = _scan_case(3, 9, d, n, g, True, False, dtype)
    out, final, _ = _scan_exact(c)
    pool = torch.full((7, d, n), 5.0, device="cuda")
    slots = torch.tensor([6, -1, 2], dtype=torch.int32, device="cuda")
    pool[6], pool[2] = c["state"][0], c["state"][2]
    for i in range(9):
        o = ssm.selective_scan_step(c["x"][:, i], c["dt"][:, i], c["A"], c["B"][:, i], c["C"][:, i], pool, D=c["D"],
                                    z=c["z"][:, i], dt_bias=c["dt_bias"], reset=c["reset"][:, i].contiguous(), slots=slots)
        assert rel(o[[0, 2]], out[[0, 2], i]) <= TOL[dtype] and not o[1].any()
    assert rel(pool[[6, 2]], final[[0, 2]]) <= TOL[torch.float32]
    assert (pool[[0, 1, 3, 4, 5]] == 5).all()


def test_slot_out_of_range_is_reported():
    G.check_error_flag("cuda")
    c = _conv_case(2, 1, 8, 4, False, False, torch.float32)
    pool = torch.ones(2, 3, 8, device="cuda")
    slots = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    y = ssm.causal_conv_step(c["x"][:, 0], c["weight"], c["bias"], pool, slots=slots)
    torch.cuda.synchronize()
    assert not y[1].any() and (pool[1] == 1).all()
    with pytest.raises(_lib.KernelError, match="state slot"):
        G.check_error_flag("cuda")


def test_extreme_steps():
    """A step of -inf leaves the state alone, one past softplus' linear range is taken as
    it is, and a decay that underflows forgets."""
    d, n = 16, 16
    x = torch.ones(1, 3, d, device="cuda")
    dt = torch.tensor([float("-inf"), 50.0, 2000.0], device="cuda")[None, :, None].expand(1, 3, d).contiguous()
    A = torch.full((d, n), -1.0, device="cuda")
    B = torch.ones(1, 3, 1, n, device="cuda")
    st = torch.full((1, d, n), 3.0, device="cuda")
    r = ssm.selective_scan(x, dt, A, B, B, state=st)
    assert torch.allclose(r.out[0, :, 0], torch.tensor([3.0 * n, 50.0 * n, 2000.0 * n], device="cuda"), rtol=1e-6)


def test_other_stream():
    c = _scan_case(2, 200, 64, 16, 1, True, False, torch.bfloat16)
    r, g = _scan_run(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r2, g2 = _scan_run(c)
    s.synchronize()
    assert torch.equal(r.out, r2.out) and all(torch.equal(p, q) for p, q in zip(g, g2))


def test_graph_replay():
    c = _scan_case(4, 1, 64, 16, 1, False, False, torch.bfloat16)
    pool = c["state"].clone()
    step = lambda: ssm.selective_scan_step(c["x"][:, 0], c["dt"][:, 0], c["A"], c["B"][:, 0], c["C"][:, 0], pool)  # noqa: E731
    step()
    pool.copy_(c["state"])
    want = [step().clone() for _ in range(3)]
    pool.copy_(c["state"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    pool.copy_(c["state"])
    for w in want:
        graph.replay()
        assert torch.equal(out, w)


def _shifted(t, by):
    """The same values in a view that starts ``by`` elements into its storage."""
    flat = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
    flat[by:] = t.reshape(-1)
    return flat[by:].view(t.shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("by", [1, 2])
def test_operands_on_odd_addresses(by, dtype):
    """Views that start off the 16-byte boundaries, every operand: the same numbers."""
    c = _conv_case(2, 30, 24, 4, True, False, dtype)
    k = {n: _shifted(v, by) if isinstance(v, torch.Tensor) and n != "x" else v for n, v in c.items()}
    k["x"] = _shifted(c["x"].contiguous(), by)
    kw = lambda q: dict(state=q["state"], reset=q["reset"])  # noqa: E731
    one = 2.0 ** -8 if dtype == torch.bfloat16 else 1e-6
    want, got = (ssm.causal_conv(q["x"], q["weight"], q["bias"], **kw(q)) for q in (c, k))
    assert rel(got[0], want[0]) <= one and torch.equal(got[1], want[1])
    want, got = (ssm.causal_conv_grad(q["dy"], q["x"], q["weight"], q["bias"], dfinal=q["dfinal"], **kw(q)) for q in (c, k))
    assert all(rel(p, q) <= one for p, q in zip(got, want))
    c = _scan_case(2, 60, 40, 16, 1, True, False, dtype)
    k = {n: _shifted(v.contiguous(), by) if isinstance(v, torch.Tensor) else v for n, v in c.items()}
    (r, g), (r2, g2) = _scan_run(c), _scan_run(k)
    assert rel(r2.out, r.out) <= TOL[dtype] and rel(r2.final, r.final) <= 1e-6
    assert all(rel(p, q) <= TOL[p.dtype] for p, q in zip(g2, g))
    with pytest.raises(ValueError, match="16-byte"):
        ssm.selective_scan_step(c["x"][:, 0], c["dt"][:, 0], c["A"], c["B"][:, 0], c["C"][:, 0], k["state"])


def test_offsets_past_32_bits():
    """Rows 2^31 elements apart, in one allocation: the same as packed together."""
    far = (1 << 31) + 8
    buf = torch.zeros(far + 64 * 64, dtype=torch.bfloat16, device="cuda")
    c = _scan_case(2, 40, 32, 16, 1, True, False, torch.bfloat16)
    xz = buf.as_strided((2, 40, 64), (far, 64, 1))
    xz[..., :32], xz[..., 32:] = c["x"], c["z"]
    k = dict(c, x=xz[..., :32], z=xz[..., 32:])
    (r, g), (r2, g2) = _scan_run(c), _scan_run(k)
    assert torch.equal(r.out, r2.out) and all(torch.equal(p, q) for p, q in zip(g, g2))
    w = torch.randn(32, 4, device="cuda")
    y, f = ssm.causal_conv(c["x"], w)
    y2, f2 = ssm.causal_conv(k["x"], w)
    assert torch.equal(y, y2) and torch.equal(f, f2)
    a, b = (ssm.causal_conv_grad(c["dout"], q["x"], w) for q in (c, k))
    assert torch.equal(a.dx, b.dx) and torch.equal(a.dweight, b.dweight)


def test_a_reset_forgets_what_is_not_finite():
    """An episode that ended in infinities and NaN leaves nothing to the next one."""
    c = _scan_case(1, 24, 16, 16, 1, False, False, torch.float32)
    c["reset"] = torch.zeros(1, 24, dtype=torch.bool, device="cuda")
    c["reset"][0, 11] = True
    bad = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    bad["x"][0, 7] = float("inf")
    bad["x"][0, 8] = float("nan")
    (r, g), (r2, g2) = _scan_run(c), _scan_run(bad)
    assert torch.equal(r.out[0, 11:], r2.out[0, 11:]) and torch.equal(r.final, r2.final)
    for name in ("dx", "ddt", "dz", "dB", "dC"):
        assert torch.equal(getattr(g, name)[0, 11:], getattr(g2, name)[0, 11:]), name
    k = _conv_case(1, 24, 16, 4, False, False, torch.float32)
    k["x"] = k["x"].clone()
    y, _ = ssm.causal_conv(k["x"], k["weight"], reset=c["reset"])
    k["x"][0, 9:11] = float("nan")
    y2, _ = ssm.causal_conv(k["x"], k["weight"], reset=c["reset"])
    assert torch.equal(y[0, 11:], y2[0, 11:])


def test_refusals():
    c = _scan_case(2, 8, 16, 16, 1, False, False, torch.float32)
    a = [c[k] for k in ("x", "dt", "A", "B", "C")]
    with pytest.raises(_lib.KernelError):
        ssm.selective_scan(*[v.cpu() for v in a])
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        ssm.selective_scan(a[0].half(), *a[1:])
    with pytest.raises(TypeError, match="dt is"):
        ssm.selective_scan(a[0], a[1].bfloat16(), *a[2:])
    with pytest.raises(ValueError, match="dt has shape"):
        ssm.selective_scan(a[0], a[1][:, :4], *a[2:])
    with pytest.raises(ValueError, match="states"):
        ssm.selective_scan(a[0], a[1], torch.ones(16, 65, device="cuda"), *a[3:])
    with pytest.raises(ValueError, match="groups"):
        ssm.selective_scan(*a[:3], torch.ones(2, 8, 3, 16, device="cuda"), a[4])
    with pytest.raises(ValueError, match="dense last axis"):
        ssm.selective_scan(a[0].transpose(1, 2).contiguous().transpose(1, 2), *a[1:])
    with pytest.raises(TypeError, match="reset"):
        ssm.selective_scan(*a, reset=torch.zeros(2, 8, device="cuda"))
    with pytest.raises(TypeError, match="lengths"):
        ssm.selective_scan(*a, lengths=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="saved"):
        ssm.selective_scan_grad(c["dout"], *a, saved=None)
    with pytest.raises(ValueError, match="slots"):
        ssm.selective_scan_step(a[0][:, 0], a[1][:, 0], a[2], a[3][:, 0], a[4][:, 0], torch.zeros(1, 16, 16, device="cuda"))
    k = _conv_case(2, 8, 16, 4, False, False, torch.float32)
    with pytest.raises(ValueError, match="width"):
        ssm.causal_conv(k["x"], torch.ones(16, 5, device="cuda"))
    with pytest.raises(ValueError, match="state has shape"):
        ssm.causal_conv(k["x"], k["weight"], state=k["state"][:, :2])
    with pytest.raises(TypeError, match="weight"):
        ssm.causal_conv(k["x"], k["weight"].bfloat16())
    with pytest.raises(ValueError, match="slots"):
        ssm.causal_conv_step(k["x"][:, 0], k["weight"], None, torch.zeros(1, 3, 16, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_outputs_apart_from_inputs(dtype):
    """An output over an input is refused where other threads still read it; beside the input in
    the same buffer, or in the place of an input that only its writer reads, it is taken."""
    c = _conv_case(3, 70, 24, 4, True, True, dtype)
    kw = dict(state=c["state"], reset=c["reset"], lengths=c["lengths"])
    want, _ = ssm.causal_conv(c["x"], c["weight"], c["bias"], **kw)
    buf = torch.zeros(3, 70, 48, device="cuda", dtype=dtype)
    x = buf[..., 24:]
    x.copy_(c["x"])
    for out in (x, buf[..., 23:47], buf[..., 1:25], c["state"].new_zeros(1, 70, 24).expand(3, 70, 24)):
        with pytest.raises(ValueError, match="share"):
            ssm.causal_conv(x, c["weight"], c["bias"], out=out, **kw)
    assert torch.equal(ssm.causal_conv(x, c["weight"], c["bias"], out=buf[..., :24], **kw)[0], want)
    pool = torch.zeros(3, 3, 24, device="cuda", dtype=dtype)
    with pytest.raises(ValueError, match="memory with state"):
        ssm.causal_conv_step(c["x"][:, 0], c["weight"], c["bias"], pool, out=pool[:, 0])
    row = torch.nan_to_num(c["x"][:, 0])
    want = ssm.causal_conv_step(row, c["weight"], c["bias"], pool.clone())
    assert torch.equal(ssm.causal_conv_step(row, c["weight"], c["bias"], pool, out=row), want)

    for t in (70, 300):                                     # whole and cut
        c = _scan_case(2, t, 40, 16, 1, True, True, dtype)
        a = {k: c[k].contiguous() for k in ("x", "dt", "A", "B", "C", "z")}
        kw = dict(D=c["D"], dt_bias=c["dt_bias"], state=c["state"], reset=c["reset"], lengths=c["lengths"])
        want = ssm.selective_scan(*[a[k] for k in ("x", "dt", "A", "B", "C")], z=a["z"], **kw).out
        for place in ("x", "dt", "z"):
            q = {k: v.clone() for k, v in a.items()}
            got = ssm.selective_scan(*[q[k] for k in ("x", "dt", "A", "B", "C")], z=q["z"], out=q[place], **kw).out
            assert got is q[place] and torch.equal(got, want)
            q = {k: v[:, 0].clone() if k != "A" else v for k, v in a.items()}
            q = {k: torch.nan_to_num(v) for k, v in q.items()}
            step = lambda pool, **o: ssm.selective_scan_step(*[q[k] for k in ("x", "dt", "A", "B", "C")], pool, z=q["z"], **o)  # noqa: E731
            first = step(c["state"].clone())
            assert torch.equal(step(c["state"].clone(), out=q[place]), first)
        wide = torch.zeros(2, t, 60, device="cuda", dtype=dtype)
        wide[..., :40] = torch.nan_to_num(a["x"])
        with pytest.raises(ValueError, match="memory with x"):
            ssm.selective_scan(wide[..., :40], *[a[k] for k in ("dt", "A", "B", "C")], out=wide[..., 20:])


def _state_error(c):
    """The largest relative error of a 32-bit state of this case, from its own steps: a decay is
    off by 2^-22 (hardware exponential) and 2^-23 |delta A| (its argument), its product and sum by
    2^-24 each; a state sums these over min(T, 1 / (1 - largest decay)) tokens. What a gradient
    multiplies, a state and an adjoint, is off by twice that."""
    t = c["x"].shape[1]
    real = ssm._real(c["lengths"], c["x"].shape[0], t, "cuda")
    v = torch.nn.functional.softplus((c["dt"].double() + c["dt_bias"].double())[real])
    rate = c["A"].double().abs()
    rate = rate[rate.isfinite()]
    memory = min(t, 1 / (1 - float(torch.exp(-v.min() * rate.min()))))
    return memory * (2.0 ** -22 + 2.0 ** -23 * float(v.max() * rate.max()) + 2.0 ** -23)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [4, 8, 16, 24, 64])
@pytest.mark.parametrize("t", [5, 16, 23, 300])
def test_missing_tokens_leave_alone_what_forgets_at_once(t, n, dtype):
    """States with a rate of -inf hold the last token only. The tokens that fill up a row's last
    tile, and a chunk behind its end, are steps of zero: 0 * -inf must not reach the states nor the
    adjoints."""
    c = _scan_case(3, t, 40, n, 1, False, False, dtype, seed=t)
    c["lengths"] = torch.tensor([t, max(1, t // 3), 0], dtype=torch.int32, device="cuda")
    for k in ("x", "z", "dt", "B", "C", "dout"):
        c[k] = _hide(c[k].contiguous(), c["lengths"])
    c["A"][:, ::2] = float("-inf")
    r, g = _scan_run(c)
    out, final, grads = _scan_exact(c)
    tol = {torch.bfloat16: TOL[torch.bfloat16], torch.float32: _state_error(c)}
    assert rel(r.out, out) <= tol[dtype] and rel(r.final, final) <= tol[torch.float32]
    got = _named(g)
    for k in ("x", "z", "B", "C", "A", "D", "state"):               # ddelta = q A is 0 * -inf by the formula
        assert rel(got[k], grads[k]) <= 2 * tol[got[k].dtype], k


def test_steps_of_zero_leave_the_state_to_the_bit():
    """exp(0 A) is exactly 1: after any number of steps of zero the state, and the adjoint on the
    way back, are the same bits."""
    for n in (4, 8, 16, 32, 64):
        st = torch.randn(2, 48, n, device="cuda")
        A = -(1 + 9 * torch.rand(48, n, device="cuda"))
        x = torch.zeros(2, 37, 48, device="cuda")
        dt = torch.full((2, 37, 48), float("-inf"), device="cuda")
        B = torch.randn(2, 37, 1, n, device="cuda")
        r = ssm.selective_scan(x, dt, A, B, B, state=st, train=True)
        g = ssm.selective_scan_grad(x, x, dt, A, B, B, saved=r.saved, state=st, dfinal=st)
        assert torch.equal(r.final, st) and torch.equal(g.dstate, st)
        pool = st.clone()
        ssm.selective_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], B[:, 0], pool)
        assert torch.equal(pool, st)


@pytest.mark.parametrize("n,g", [(16, 1), (5, 2), (64, 1)])
def test_scan_slot_out_of_range_is_reported(n, g):
    """The row's output is zero, its neighbours' states are where they were, the rows beside it
    are answered, and the error is there to be raised."""
    G.check_error_flag("cuda")
    c = _scan_case(3, 1, 24, n, g, False, False, torch.float32)
    pool = torch.full((4, 24, n), 2.0, device="cuda")
    slots = torch.tensor([1, 3, 0], dtype=torch.int32, device="cuda")
    args = [c[k][:, 0] if k != "A" else c[k] for k in ("x", "dt", "A", "B", "C")]
    y = ssm.selective_scan_step(*args, pool[:3], z=c["z"][:, 0], slots=slots)
    torch.cuda.synchronize()
    assert not y[1].any() and y[0].any() and y[2].any()
    assert (pool[2:] == 2).all() and (pool[:2] != 2).any()
    with pytest.raises(_lib.KernelError, match="state slot"):
        G.check_error_flag("cuda")
    G.check_error_flag("cuda")


# B, T, D, N, groups, reset, ragged, rows in chunks: channels of a group on both sides of what
# makes a block ordinary (129, 65, 33, 17 for 1..4, 5..16, 17..32, 33..64 states) or narrow, for
# every count of lanes, in 16-byte and 4-byte pieces and element by element, whole and cut
BLOCKS = [
    (2, 37, 304, 4, 1, True, True, False), (3, 50, 258, 3, 2, True, True, False), (2, 23, 128, 4, 1, True, True, False),
    (1, 300, 320, 4, 1, True, False, True), (2, 260, 24, 2, 1, True, True, True),
    (2, 70, 200, 8, 1, True, True, False), (3, 45, 133, 7, 1, True, True, False), (2, 19, 128, 8, 2, False, True, False),
    (2, 300, 256, 8, 1, True, True, True), (1, 200, 12, 8, 1, False, False, True),
    (2, 41, 136, 16, 1, True, True, False), (2, 33, 65, 13, 1, True, True, False),
    (2, 41, 104, 32, 1, True, True, False), (3, 35, 74, 20, 2, True, True, False), (1, 39, 32, 24, 1, True, False, False),
    (2, 200, 80, 24, 1, True, True, True), (1, 260, 16, 32, 2, True, False, True),
    (2, 33, 32, 64, 2, True, True, False), (3, 40, 10, 40, 1, True, True, False), (2, 29, 72, 64, 1, True, True, False),
    (2, 200, 16, 48, 1, True, True, True), (1, 260, 51, 64, 1, True, False, True),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", BLOCKS, ids=str)
def test_scan_in_every_kind_of_block(case, dtype):
    b, t, d, n, g = case[:5]
    assert (ssm._chunks(b, t, d, n, g)[1] > 2) == case[7]
    c = _scan_case(*case[:7], dtype, seed=11)
    r, gr = _scan_run(c)
    out, final, grads = _scan_exact(c)
    tol = {torch.bfloat16: TOL[torch.bfloat16], torch.float32: _state_error(c)}
    assert rel(r.out, out) <= tol[dtype] and rel(r.final, final) <= tol[torch.float32]
    for k, v in _named(gr).items():
        assert rel(v, grads[k]) <= 2 * tol[v.dtype], k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_in_three_chunks(dtype):
    """The fewest chunks that a row is cut into, and never two."""
    assert ssm._chunks(19, 200, 1000, 16, 1) == (80, 3)
    for b in range(1, 80):
        for t in (127, 128, 129, 200, 1000):
            assert ssm._chunks(b, t, 1000, 16, 1)[1] != 2
    c = _scan_case(19, 200, 1000, 16, 1, True, True, dtype)
    r, g = _scan_run(c)
    out, final, grads = _scan_exact(c)
    tol = {torch.bfloat16: TOL[torch.bfloat16], torch.float32: _state_error(c)}
    assert rel(r.out, out) <= tol[dtype] and rel(r.final, final) <= tol[torch.float32]
    for k, v in _named(g).items():
        assert rel(v, grads[k]) <= 2 * tol[v.dtype], k
