"""Group norm with an activation against its definition in 64 bits, with gradients by autograd.

Tolerances, of norms: a bfloat16 result is one rounding (half a step, 2^-8 of the value). 32-bit
results: mean and variance are sums of n terms in parts, at most 64 roundings of 2^-24 one after
the other in any of them, and xh takes a handful more: 80 * 2^-24 = 5e-6 one way. The sigmoid's
hardware functions add 2^-21. Gradients of the channels sum over samples in the same way: 1e-5.
"""
import pytest
import torch

from surfb200.ops import _lib, norm as N

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def rel(x, y):
    y = y.detach().double()
    n = float(torch.linalg.vector_norm(y))
    return float(torch.linalg.vector_norm(x.double() - y)) / (n if n else 1.0)


def make(shape, dtype, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    c = shape[-1]
    return (r(*shape) * 2 + 3 * r(c)).to(dtype), 1 + 0.3 * r(c), 0.3 * r(c), r(*shape).to(dtype)


def check(x, w, b, dy, groups, activation, **kw):
    dtype = x.dtype
    half = torch.finfo(dtype).eps / 2 if dtype == BF else 0.0
    xd, wd, bd = (None if t is None else t.double().requires_grad_() for t in (x, w, b))
    want = N.group_norm_reference(xd, groups, wd, bd, activation=activation)
    live = [t for t in (xd, wd, bd) if t is not None]
    grads = dict(zip([n for n, t in zip("xwb", (xd, wd, bd)) if t is not None], torch.autograd.grad((want * dy.double()).sum(), live)))
    r = N.group_norm(x, groups, w, b, activation=activation, train=True, **kw)
    d = N.group_norm_grad(dy, x, groups, w, b, stats=r.stats, activation=activation)
    assert rel(r.out, want) < half + 5e-6
    assert rel(d.dx, grads["x"]) < half + 1e-5
    for name, got in (("w", d.dweight), ("b", d.dbias)):
        assert (got is None) == (name not in grads)
        if got is not None:
            assert rel(got, grads[name]) < 1e-5, name
    return r, d


SHAPES = [  # shape, groups
    ((5, 16), 1), ((1, 4, 8), 2), ((33, 512), 8), ((7, 3, 24), 3), ((2, 5, 7, 40), 5), ((3, 16, 32, 64), 8), ((1, 1, 1, 32), 2),
    ((300, 96), 4), ((2, 1000, 33), 3), ((1, 40000, 8), 1), ((2, 70, 1500), 2), ((4, 9, 257), 1), ((1, 3000, 120), 6),
    ((70, 2000, 16), 2), ((2, 4, 4096), 1), ((600, 2, 64), 32), ((3, 33, 130), 13),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("activation", ["none", "silu"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_against_the_definition(shape, groups, activation, dtype):
    check(*make(shape, dtype), groups, activation)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape,groups", [((40, 64), 4), ((3, 100, 48), 3), ((1, 9000, 64), 2)])
def test_relu(shape, groups, dtype):
    """Its gradient jumps at 0: values whose 64-bit pre-activation is within 1e-4 of it get none of dy."""
    x, w, b, dy = make(shape, dtype)
    pre = N.group_norm_reference(x.double(), groups, w.double(), b.double())
    check(x, w, b, torch.where(pre.abs() < 1e-4, torch.zeros_like(dy), dy), groups, "relu")


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("shape,groups", [((40, 64), 4), ((3, 100, 48), 3), ((1, 9000, 64), 2)])
def test_without_weights(shape, groups, weight, bias):
    x, w, b, dy = make(shape, F32)
    check(x, w if weight else None, b if bias else None, dy, groups, "silu")


def test_a_large_mean_costs_no_variance():
    """Values about 1000 with a spread of 1: the mean's own rounding, 1000 * 2^-24, shifts all alike."""
    for shape in ((20, 64), (3, 400, 64), (1, 30000, 64)):
        x, w, b, _ = make(shape, F32)
        x = x - x.mean() + 1000.0
        got = N.group_norm(x, 4, w, b).out
        assert rel(got, N.group_norm_reference(x.double(), 4, w.double(), b.double())) < 2e-4


def test_equal_values_give_the_bias():
    for shape in ((5, 32), (2, 300, 32), (1, 40000, 32)):
        b = torch.randn(32, device="cuda")
        got = N.group_norm(torch.full(shape, 3.0, device="cuda"), 4, None, b).out
        assert torch.equal(got, b.expand(shape))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_not_finite_stays_in_its_group(dtype):
    for shape in ((6, 64), (3, 300, 64), (2, 20000, 64)):
        x, w, b, _ = make(shape, dtype)
        want = N.group_norm(x, 4, w, b).out
        x[1].view(-1, 64)[0, 20] = float("nan")
        got = N.group_norm(x, 4, w, b).out
        assert got[1][..., 16:32].isnan().all()
        got[1][..., 16:32] = want[1][..., 16:32]
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_addresses_and_in_place(dtype):
    for shape, groups in (((9, 48), 3), ((2, 6, 7, 48), 3), ((2, 3000, 48), 3)):
        x, w, b, dy = make(shape, dtype)
        r, d = check(x, w, b, dy, groups, "silu")
        wide = torch.empty((*shape[:-1], 100), dtype=dtype, device="cuda")
        wide[..., 11:59], wide[..., 59] = x, 7.0
        v = wide[..., 11:59]
        # an odd address takes narrower pieces, and sums in another order
        half = torch.finfo(dtype).eps / 2 if dtype == BF else 0.0
        got = N.group_norm(v, groups, w, b, activation="silu", train=True)
        assert rel(got.out, r.out) < half + 1e-6 and rel(got.stats, r.stats) < 1e-6
        g = N.group_norm_grad(dy, v, groups, w, b, stats=r.stats, activation="silu")
        assert rel(g.dx, d.dx) < half + 1e-6 and rel(g.dweight, d.dweight) < 1e-6
        assert N.group_norm(v, groups, w, b, activation="silu", out=v).out is v
        assert torch.equal(v, got.out) and bool((wide[..., 59] == 7.0).all())


def test_offsets_past_32_bits():
    x, w, b, dy = make((2, 50, 32), BF)
    r, d = check(x, w, b, dy, 4, "none")
    big = torch.empty(2 ** 32 + 50 * 32, dtype=BF, device="cuda")
    far = torch.as_strided(big, x.shape, (2 ** 32, 32, 1))
    far.copy_(x)
    assert torch.equal(N.group_norm(far, 4, w, b).out, r.out)
    assert torch.equal(N.group_norm_grad(dy, far, 4, w, b, stats=r.stats).dx, d.dx)


def test_empty_streams_and_graphs():
    x, w, b, dy = make((0, 5, 16), BF)
    r = N.group_norm(x, 2, w, b, train=True)
    d = N.group_norm_grad(dy, x, 2, w, b, stats=r.stats)
    assert r.out.shape == x.shape and not d.dweight.any() and not d.dbias.any()
    for shape in ((40, 64), (3, 300, 64), (1, 30000, 64)):
        x, w, b, dy = make(shape, BF)

        def both():
            r = N.group_norm(x, 4, w, b, activation="silu", train=True)
            return (r.out, r.stats) + tuple(N.group_norm_grad(dy, x, 4, w, b, stats=r.stats, activation="silu"))
        want = both()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = both()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            replayed = both()
        graph.replay()
        torch.cuda.synchronize()
        for p, q, s in zip(want, other, replayed):
            assert torch.equal(p, q) and torch.equal(p, s)


def test_refusals():
    x, w, b, dy = make((4, 6, 32), BF)
    with pytest.raises(ValueError, match="divide the channels"):
        N.group_norm(x, 5)
    with pytest.raises(ValueError, match="activation"):
        N.group_norm(x, 4, activation="gelu")
    with pytest.raises(ValueError, match="eps"):
        N.group_norm(x, 4, eps=0.0)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        N.group_norm(x.half(), 4)
    with pytest.raises(TypeError, match="weight must be"):
        N.group_norm(x, 4, w.bfloat16())
    with pytest.raises(ValueError, match="bias has shape"):
        N.group_norm(x, 4, w, b[:8])
    with pytest.raises(ValueError, match="dense last axis"):
        N.group_norm(x.transpose(1, 2).contiguous().transpose(1, 2), 4)
    with pytest.raises(ValueError, match="constant stride"):
        N.group_norm(torch.zeros(2, 4, 9, 32, dtype=BF, device="cuda")[:, :, :5], 4)
    with pytest.raises(ValueError, match="out shares memory"):
        N.group_norm(x[:2], 4, out=x[1:3])
    with pytest.raises(ValueError, match="x must be"):
        N.group_norm(x[0, 0], 4)
    with pytest.raises(_lib.KernelError):
        N.group_norm(x.cpu(), 4)
    with pytest.raises(ValueError, match="statistics"):
        N.group_norm_grad(dy, x, 4, stats=None)
    with pytest.raises(ValueError, match="stats has shape"):
        N.group_norm_grad(dy, x, 4, stats=torch.zeros(4, 2, 2, device="cuda"))


def test_numbers_past_float32_and_odd_statistics_are_refused():
    x = torch.randn(4, 6, 32, device="cuda")
    for eps in (1e39, 1e-39, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            N.group_norm(x, 4, eps=eps)
    stats = N.group_norm(x, 4, train=True).stats
    odd = torch.empty(1 + stats.numel(), device="cuda")[1:].view(stats.shape)
    odd.copy_(stats)
    with pytest.raises(ValueError, match="8-byte"):
        N.group_norm_grad(x, x, 4, stats=odd)


@pytest.mark.parametrize("shape,groups", [((40, 96), 3), ((300, 200, 32), 4), ((1, 5000, 24), 3)])
def test_weights_at_odd_addresses_and_two_calls_at_once(shape, groups):
    gen = torch.Generator("cuda").manual_seed(5)
    c = shape[-1]
    x, dy = (torch.randn(*shape, generator=gen, device="cuda") for _ in range(2))
    flat = torch.randn(2 * c + 1, generator=gen, device="cuda")
    w, b = flat[1:c + 1], flat[c + 1:]
    whole = N.group_norm(x, groups, w.clone(), b.clone(), activation="silu", train=True)
    grads = N.group_norm_grad(dy, x, groups, w.clone(), b.clone(), stats=whole.stats, activation="silu")
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams * 3:
        with torch.cuda.stream(s):
            y = N.group_norm(x, groups, w, b, activation="silu", train=True)
            got.append((y, N.group_norm_grad(dy, x, groups, w, b, stats=y.stats, activation="silu")))
    torch.cuda.synchronize()
    for y, g in got:
        assert torch.equal(y.out, whole.out) and torch.equal(y.stats, whole.stats)
        for a, e in zip(g, grads):
            assert torch.equal(a, e)
